// Quantisation of rows to microscaled 4-bit floating point.
//
// E2M1 has the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6. Per block of B columns:
//   MXFP4 (B = 32): scale d = 2^(floor(log2 amax) - 2), an E8M0 byte.
//   NVFP4 (B = 16): scale d = s * r with s = RNE_e4m3(amax / (6 r)) and r the
//       smallest power of two (>= 2^-100) with amax_row / 6 <= 448 r, one per
//       row, so that s never saturates and needs no calibration pass.
//   code = RNE_e2m1(x / d), saturating (MXFP4's largest element lies in [4, 8)).
// r is a power of two, so d is exact; x / d is correctly rounded (Markstein:
// from y = RN(1/d) and q = RN(x y), q + (x - q d) y rounds to RN(x / d)). d
// has four significant bits, so RN(x / d) meets a rounding border of E2M1 only
// where x / d does: the codes are those of the real quotient, ties to even.
//
// One pass over the row, held in registers between the maximum and the codes:
// a lane has 8 columns (16 or 32 bytes of input, 4 bytes of codes), LANES
// lanes a row, 2 or 4 lanes a block.
#include "fp4.cuh"

namespace gatb {

namespace {

struct QuantArgs {
    uint64_t n;
    int width;
    int chunks;      // 8-column pieces of a row that are visited (whole scale tiles)
    int code_chunks; // of those, the ones inside the code row
    const void* x;
    int ldx;
    uint8_t* codes;
    int ldc;
    uint8_t* scales;
    int tiles;
    float* row_scale;
    void* values;
    int ldv;
    int v_bf16;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Memory is touched in fours: 4 elements at an address that is a multiple of
// their size. LOOSE: rows may begin and end inside a four, and a lane's 8
// columns then lie in up to three of them. A four with elements outside the
// row is taken apart. 58,798 x 3782 BF16 to NVFP4 took 540 us element by
// element and takes 275, 100,000 x 501 FP32 to MXFP4 133 and 78.

// The four at p, whose first element is column `col` of the row.
template <bool BF16, bool LOOSE>
__device__ __forceinline__ void load4(const void* p, int col, int width, uint32_t* u) {
    constexpr int kWords = BF16 ? 2 : 4;
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = 0u;
    if (LOOSE ? col >= 0 && col + 4 <= width : col < width) {
        if constexpr (BF16) {
            const uint2 t = __ldg(static_cast<const uint2*>(p));
            u[0] = t.x; u[1] = t.y;
        } else {
            const uint4 t = __ldg(static_cast<const uint4*>(p));
            u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w;
        }
    } else if (LOOSE && col > -4 && col < width) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i >= 0 && col + i < width) {
                if constexpr (BF16)
                    u[i / 2] |= uint32_t(__ldg(static_cast<const uint16_t*>(p) + i)) << (i % 2 * 16);
                else
                    u[i] = __ldg(static_cast<const uint32_t*>(p) + i);
            }
    }
}
// Its columns from `first` to the width.
template <bool BF16, bool LOOSE>
__device__ __forceinline__ void store4(void* p, int col, int first, int width, const uint32_t* u) {
    if (LOOSE ? col >= first && col + 4 <= width : col < width) {
        if constexpr (BF16)
            *static_cast<uint2*>(p) = make_uint2(u[0], u[1]);
        else
            *static_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else if (LOOSE && col > first - 4 && col < width) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i >= first && col + i < width) {
                if constexpr (BF16)
                    static_cast<uint16_t*>(p)[i] = uint16_t(u[i / 2] >> (i % 2 * 16));
                else
                    static_cast<uint32_t*>(p)[i] = u[i];
            }
    }
}

// Columns [col, col + 8) of the row at element offset `off`; zeros past the width.
template <bool BF16, bool LOOSE>
__device__ __forceinline__ void load8(const void* x, uint64_t off, int col, int width, float* v) {
    constexpr int kWords = BF16 ? 2 : 4, kSize = BF16 ? 2 : 4;  // words of a four, bytes of an element
    const char* p = static_cast<const char*>(x) + (off + uint64_t(col)) * kSize;
    uint32_t u[3 * kWords];
    if constexpr (LOOSE) {
        const int s = int(reinterpret_cast<uintptr_t>(p) / kSize & 3);
        p -= s * kSize;
        load4<BF16, true>(p, col - s, width, u);
        load4<BF16, true>(p + 4 * kSize, col - s + 4, width, u + kWords);
        load4<BF16, true>(p + 8 * kSize, col - s + 8, s ? width : 0, u + 2 * kWords);
        if constexpr (BF16) {
#pragma unroll
            for (int i = 0; i < 5; ++i) u[i] = s & 2 ? u[i + 1] : u[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __funnelshift_r(u[i], u[i + 1], s & 1 ? 16 : 0);
        } else {
#pragma unroll
            for (int i = 0; i < 9; ++i) u[i] = s & 2 ? u[i + 2] : u[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = s & 1 ? u[i + 1] : u[i];
        }
    } else {
        load4<BF16, false>(p, col, width, u);
        load4<BF16, false>(p + 4 * kSize, col + 4, width, u + kWords);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (BF16)
            v[i] = i % 2 ? bf16hi(u[i / 2]) : bf16lo(u[i / 2]);
        else
            v[i] = __uint_as_float(u[i]);
    }
}

// y to columns [col, col + 8) of the row at element offset `off`, up to the
// width. LOOSE: the whole warp calls it, `group` neighbouring lanes with
// neighbouring columns of a row. A lane stores the two fours that end in its
// columns, with up to three elements of the lane before it in the first; the
// group's last lane stores the elements behind them too.
template <bool BF16, bool LOOSE>
__device__ __forceinline__ void store8(void* out, uint64_t off, int col, int width, const float* y, int group) {
    constexpr int kWords = BF16 ? 2 : 4, kSize = BF16 ? 2 : 4;
    char* p = static_cast<char*>(out) + (off + uint64_t(col)) * kSize;
    uint32_t u[3 * kWords];  // columns [col - 4, col + 8)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (!BF16)
            u[kWords + i] = __float_as_uint(y[i]);
        else if (i % 2 == 0)
            u[kWords + i / 2] = pack_bf16x2(y[i], y[i + 1]);  // exact: at most six significant bits
    }
    if constexpr (LOOSE) {
        const int s = int(reinterpret_cast<uintptr_t>(p) / kSize & 3), at = threadIdx.x % group;
#pragma unroll
        for (int i = 0; i < kWords; ++i) u[i] = __shfl_up_sync(0xffffffffu, u[2 * kWords + i], 1);
        if (at == group - 1) {
#pragma unroll
            for (int i = 5; i < 8; ++i)
                if (i >= 8 - s && col + i < width) {
                    if constexpr (BF16)
                        reinterpret_cast<uint16_t*>(p)[i] = uint16_t(u[kWords + i / 2] >> (i % 2 * 16));
                    else
                        reinterpret_cast<uint32_t*>(p)[i] = u[kWords + i];
                }
        }
        if constexpr (BF16) {  // to columns [col - s, col - s + 8) from the second four on
#pragma unroll
            for (int i = 5; i >= 1; --i) u[i] = s & 2 ? u[i - 1] : u[i];
#pragma unroll
            for (int i = 5; i >= 2; --i) u[i] = __funnelshift_l(u[i - 1], u[i], s & 1 ? 16 : 0);
        } else {
#pragma unroll
            for (int i = 11; i >= 3; --i) u[i] = s & 2 ? u[i - 2] : u[i];
#pragma unroll
            for (int i = 11; i >= 4; --i) u[i] = s & 1 ? u[i - 1] : u[i];
        }
        p -= s * kSize;
        const int first = at == 0 ? col : 0;
        store4<BF16, true>(p, col - s, first, width, u + kWords);
        store4<BF16, true>(p + 4 * kSize, col - s + 4, first, width, u + 2 * kWords);
    } else {
        store4<BF16, false>(p, col, 0, width, u + kWords);
        store4<BF16, false>(p + 4 * kSize, col + 4, 0, width, u + 2 * kWords);
    }
}

// Eight floats to E2M1 (round to nearest even, saturating), element i at bits 4 i.
__device__ __forceinline__ uint32_t e2m1x8(const float* q) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return r;
}
// The values of eight codes.
__device__ __forceinline__ void from_e2m1x8(uint32_t c, float* v) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(v[2 * i]), "=f"(v[2 * i + 1])
            : "r"(h[i]));
}
__device__ __forceinline__ uint32_t to_e4m3(float x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
    return r & 0xffu;
}
__device__ __forceinline__ float from_e4m3(uint32_t b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(b)));
    float f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(h));
    return f;
}
// Power-of-two row scale of NVFP4 from the row's largest magnitude.
__device__ __forceinline__ float row_power(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u >= 0x7f800000u) return __uint_as_float(0x7fc00000u);  // Inf or NaN in the row
    if (u == 0) return 1.f;
    // amax <= 2688 * 2^j, 2688 = 1.3125 * 2^11; subnormal rows take the smallest r
    int j = int(u >> 23) - 127 - 11 + ((u & 0x7fffffu) > 0x280000u ? 1 : 0);
    j = j < -100 ? -100 : j;
    return __uint_as_float(uint32_t(j + 127) << 23);
}

// RN(1 / s) of an E4M3 number s > 0: one Newton step from an approximation
// within an ulp or so; s has four significant bits, so no 1 / s lies near the
// middle between two FP32 numbers.
__device__ __forceinline__ float reciprocal_e4m3(float s) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
    return fmaf(y, fmaf(-s, y, 1.f), y);
}

// LANES lanes per row (4 to 32: part of a warp; 256: the CTA), CHUNKS pieces
// of 8 columns a lane kept in registers. REREAD: rows longer than LANES *
// CHUNKS * 8 columns are read a second time for the codes. LOOSE: width, rows of
// x or rows of the values are not all whole, aligned fours of elements.
// Issue slots bind it as much as memory does, hence packed FP32 pairs and no
// branches on alignment inside: 2,449,029 x 100 FP32 to NVFP4 with BF16 values
// took 389 us with scalar arithmetic and such branches and takes 318 us
// (5.1 TB/s); 169,343 x 128 FP32 to MXFP4 26.5 us (5.3 TB/s).
template <int FORMAT, bool BF16, bool LOOSE, int LANES, int CHUNKS, bool REREAD>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const QuantArgs a) {
    constexpr bool kNv = FORMAT == GAT_B200_NVFP4;
    constexpr int kBlockLanes = fp4_block(FORMAT) / 8;  // lanes of one block
    const int lane = threadIdx.x % LANES;
    const uint64_t row = LANES >= 256 ? uint64_t(blockIdx.x) : uint64_t(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const bool live = row < a.n;
    const int width = live ? a.width : 0;
    const uint64_t xoff = row * uint64_t(a.ldx);
    float v[CHUNKS][8];
    float mine[CHUNKS];

    auto fetch = [&](int c0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = ((c0 + c) * LANES + lane) * 8;
            if (LOOSE && (c0 + c) * LANES * 8 >= a.width) {  // the same for all lanes
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
            } else {
                load8<BF16, LOOSE>(a.x, xoff, col, width, v[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float m = max_nan(fabsf(v[c][0]), fabsf(v[c][1]), fabsf(v[c][2]));
            m = max_nan(m, fabsf(v[c][3]), fabsf(v[c][4]));
            m = max_nan(m, fabsf(v[c][5]), fabsf(v[c][6]));
            mine[c] = max_nan(m, fabsf(v[c][7]));
        }
    };

    float r = 1.f, rinv = 1.f;
    if constexpr (kNv) {
        float m = 0.f;
        const int steps = REREAD ? (a.chunks + LANES * CHUNKS - 1) / (LANES * CHUNKS) : 1;
        for (int s = 0; s < steps; ++s) {
            fetch(s * CHUNKS);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) m = max_nan(m, mine[c]);
        }
#pragma unroll
        for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        if constexpr (LANES >= 256) {
            __shared__ float part[8];
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
            __syncthreads();
            m = part[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = max_nan(m, part[i]);
        }
        r = row_power(m);
        rinv = __uint_as_float((254u << 23) - __float_as_uint(r));  // 1 / r of a power of two
        if (lane == 0 && live) a.row_scale[row] = r;
    }
    const bool row_nan = kNv && r != r;
    uint8_t* code_row = a.codes + row * uint64_t(a.ldc);
    uint8_t* scale_row = a.scales + (row >> 7) * uint64_t(a.tiles) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;

    const int steps = REREAD || !kNv ? (a.chunks + LANES * CHUNKS - 1) / (LANES * CHUNKS) : 1;
    for (int s = 0; s < steps; ++s) {
        if (!kNv || REREAD) fetch(s * CHUNKS);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            if ((s * CHUNKS + c) * LANES >= a.chunks) break;  // the same for all lanes of the row
            const int chunk = (s * CHUNKS + c) * LANES + lane;
            float m = mine[c];
#pragma unroll
            for (int o = 1; o < kBlockLanes; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            uint32_t byte;
            float d, inv;
            if constexpr (kNv) {
                // amax / (6 r), correctly rounded (see above); amax * rinv is exact
                const float t = m * rinv;
                float q = t * (1.f / 6.f);
                q = fmaf(fmaf(-6.f, q, t), 1.f / 6.f, q);
                byte = row_nan ? 0u : to_e4m3(q);
                const float sc = from_e4m3(byte);
                d = sc * r;
                inv = sc > 0.f ? reciprocal_e4m3(sc) * rinv : 0.f;
            } else {
                const uint32_t u = __float_as_uint(m);
                const int e = int(u >> 23) - 2;  // biased exponent of the scale
                byte = u >= 0x7f800000u ? 255u : uint32_t(max(e, 0));
                d = byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte ? byte << 23 : 0x400000u);
                inv = byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
            }
            float q[8];
            const f32x2 inv2 = pack2(inv, inv), nd2 = pack2(-d, -d);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const f32x2 x2 = pack2(v[c][i], v[c][i + 1]);
                f32x2 q2 = mul2(x2, inv2);
                if constexpr (kNv) q2 = fma2(fma2(q2, nd2, x2), inv2, q2);
                unpack2(q2, q[i], q[i + 1]);
            }
            const uint32_t code = inv == 0.f ? 0u : e2m1x8(q);
            if (live && chunk < a.chunks) {
                if (chunk < a.code_chunks) *reinterpret_cast<uint32_t*>(code_row + uint32_t(chunk) * 4) = code;
                if (lane % kBlockLanes == 0) {
                    const uint32_t block = uint32_t(chunk) / kBlockLanes;
                    scale_row[uint64_t(block >> 2) * 512 + (block & 3)] = uint8_t(byte);
                }
            }
            if (a.values && (!LOOSE || (s * CHUNKS + c) * LANES * 8 < a.width)) {
                float y[8];
                from_e2m1x8(code, y);
                const f32x2 d2 = pack2(d, d);
#pragma unroll
                for (int i = 0; i < 8; i += 2) unpack2(mul2(pack2(y[i], y[i + 1]), d2), y[i], y[i + 1]);
                constexpr int kGroup = LANES < 32 ? LANES : 32;
                const uint64_t off = row * uint64_t(a.ldv);
                if (a.v_bf16)
                    store8<true, LOOSE>(a.values, off, chunk * 8, width, y, kGroup);
                else
                    store8<false, LOOSE>(a.values, off, chunk * 8, width, y, kGroup);
            }
        }
    }
}

// Alignment in bytes (at most 16) of base and of every row at `pitch` bytes.
int row_align(const void* base, uint64_t pitch) {
    const uint64_t u = uint64_t(reinterpret_cast<uintptr_t>(base)) | pitch | 16;
    return int(u & (~u + 1));
}

template <int FORMAT, bool BF16, bool LOOSE>
int launch_quantize(const QuantArgs& a, cudaStream_t st) {
    // As many lanes a row as its pieces take, up to a warp; one warp up to 1024
    // columns, the CTA for longer ones; above 8192 columns NVFP4 reads twice.
    // Up to 32 columns 4 lanes, as most of a scale tile is empty (305,316 x 32
    // FP32 to MXFP4: 25 us, 16 lanes 35; to NVFP4 18 us, 16 lanes 22).
    constexpr int kFew = FORMAT == GAT_B200_MXFP4 ? 4 : 2;  // pieces a lane of a scale tile
    const unsigned per64 = unsigned((a.n + 63) / 64), per32 = unsigned((a.n + 31) / 32);
    const unsigned per16 = unsigned((a.n + 15) / 16), per8 = unsigned((a.n + 7) / 8), n = unsigned(a.n);
    if (a.width <= 32)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 4, kFew, false><<<per64, 256, 0, st>>>(a);
    else if (FORMAT == GAT_B200_NVFP4 && a.chunks <= 8)
        fp4_quantize_kernel<GAT_B200_NVFP4, BF16, LOOSE, 8, 1, false><<<per32, 256, 0, st>>>(a);
    else if (a.chunks <= 16)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 16, 1, false><<<per16, 256, 0, st>>>(a);
    else if (a.chunks <= 32)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 32, 1, false><<<per8, 256, 0, st>>>(a);
    else if (a.chunks <= 64)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 32, 2, false><<<per8, 256, 0, st>>>(a);
    else if (a.chunks <= 128)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 32, 4, false><<<per8, 256, 0, st>>>(a);
    else if (a.chunks <= 256)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 256, 1, false><<<n, 256, 0, st>>>(a);
    else if (a.chunks <= 512)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 256, 2, false><<<n, 256, 0, st>>>(a);
    else if (a.chunks <= 1024)
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 256, 4, false><<<n, 256, 0, st>>>(a);
    else
        fp4_quantize_kernel<FORMAT, BF16, LOOSE, 256, 4, true><<<n, 256, 0, st>>>(a);
    GATB_LAUNCH("fp4_quantize kernel");
    return 0;
}
template <int FORMAT>
int launch_quantize(const QuantArgs& a, bool bf16, bool loose, cudaStream_t st) {
    if (bf16) return loose ? launch_quantize<FORMAT, true, true>(a, st) : launch_quantize<FORMAT, true, false>(a, st);
    return loose ? launch_quantize<FORMAT, false, true>(a, st) : launch_quantize<FORMAT, false, false>(a, st);
}

}  // namespace

int fp4_check_format(const char* what, int format) {
    if (format != GAT_B200_MXFP4 && format != GAT_B200_NVFP4) return fail(std::string(what) + ": bad format");
    return 0;
}

int fp4_quantize_launch(int format, uint64_t n, int width, const void* x, int x_dtype, int ldx, void* codes, int ldc,
                        void* scales, float* row_scale, void* values, int v_dtype, int ldv, cudaStream_t st) {
    if (int rc = fp4_check_format("fp4_quantize", format)) return rc;
    if (x_dtype != GAT_B200_F32 && x_dtype != GAT_B200_BF16) return fail("fp4_quantize: bad input dtype");
    if (width <= 0 || width > (1 << 24)) return fail("fp4_quantize: bad width");
    if (n > uint64_t(INT32_MAX)) return fail("fp4_quantize: too many rows");
    if (ldx < width) return fail("fp4_quantize: X row stride smaller than the width");
    if (ldc < fp4_row_bytes(width) || ldc % 16) return fail("fp4_quantize: code rows must be 16-byte aligned and hold the width");
    if (values && v_dtype != GAT_B200_F32 && v_dtype != GAT_B200_BF16) return fail("fp4_quantize: bad values dtype");
    if (values && ldv < width) return fail("fp4_quantize: values row stride smaller than the width");
    if (n == 0) return 0;
    if (!x || !codes || !scales) return fail("fp4_quantize: null argument");
    if (format == GAT_B200_NVFP4 && !row_scale) return fail("fp4_quantize: NVFP4 needs the row scales");
    const int xs = x_dtype == GAT_B200_F32 ? 4 : 2, vs = v_dtype == GAT_B200_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % xs || (values && reinterpret_cast<uintptr_t>(values) % vs) ||
        reinterpret_cast<uintptr_t>(row_scale) % 4)
        return fail("fp4_quantize: misaligned pointer");
    if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15)
        return fail("fp4_quantize: codes and scales must be 16-byte aligned");
    if (int rc = check_device_pointers("fp4_quantize", {x, codes, scales, row_scale, values})) return rc;
    QuantArgs a{};
    a.n = n;
    a.width = width;
    a.tiles = fp4_tiles(format, width);
    a.chunks = a.tiles * fp4_block(format) / 2;
    a.code_chunks = fp4_row_bytes(width) / 4;
    a.x = x;
    a.ldx = ldx;
    a.codes = static_cast<uint8_t*>(codes);
    a.ldc = ldc;
    a.scales = static_cast<uint8_t*>(scales);
    a.row_scale = row_scale;
    a.values = values;
    a.ldv = ldv;
    a.v_bf16 = v_dtype == GAT_B200_BF16;
    const bool loose = !(width % 4 == 0 && row_align(x, uint64_t(ldx) * xs) >= 4 * xs &&
                         (!values || row_align(values, uint64_t(ldv) * vs) >= 4 * vs));
    const bool bf16 = x_dtype == GAT_B200_BF16;
    return format == GAT_B200_MXFP4 ? launch_quantize<GAT_B200_MXFP4>(a, bf16, loose, st)
                                    : launch_quantize<GAT_B200_NVFP4>(a, bf16, loose, st);
}

}  // namespace gatb
