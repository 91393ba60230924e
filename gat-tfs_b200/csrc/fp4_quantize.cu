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
    int x_align;     // bytes to which every 8-column piece of x is aligned (at most 16)
    uint8_t* codes;
    int ldc;
    uint8_t* scales;
    int tiles;
    float* row_scale;
    void* values;
    int ldv;
    int v_align;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 8 columns from element offset `off`, of which `valid` exist (zeros behind).
template <bool BF16>
__device__ __forceinline__ void load8(const QuantArgs& a, uint64_t off, int valid, float* v) {
    if constexpr (BF16) {
        const uint16_t* p = static_cast<const uint16_t*>(a.x) + off;
        uint32_t u[4];
        if (valid == 8 && a.x_align >= 4) {
            if (a.x_align >= 16) {
                const uint4 t = ldg_nc_v4(p);
                u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w;
            } else if (a.x_align >= 8) {
                const uint2 t0 = __ldg(reinterpret_cast<const uint2*>(p)), t1 = __ldg(reinterpret_cast<const uint2*>(p) + 1);
                u[0] = t0.x; u[1] = t0.y; u[2] = t1.x; u[3] = t1.y;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = 2 * i < valid ? __ldg(p + 2 * i) : 0u;
                const uint32_t hi = 2 * i + 1 < valid ? __ldg(p + 2 * i + 1) : 0u;
                u[i] = lo | (hi << 16);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16lo(u[i]);
            v[2 * i + 1] = bf16hi(u[i]);
        }
    } else {
        const float* p = static_cast<const float*>(a.x) + off;
        if (valid == 8 && a.x_align >= 16) {
            const float4 t0 = __ldg(reinterpret_cast<const float4*>(p)), t1 = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = t0.x; v[1] = t0.y; v[2] = t0.z; v[3] = t0.w;
            v[4] = t1.x; v[5] = t1.y; v[6] = t1.z; v[7] = t1.w;
        } else if (valid == 4 && a.x_align >= 16) {
            const float4 t0 = __ldg(reinterpret_cast<const float4*>(p));
            v[0] = t0.x; v[1] = t0.y; v[2] = t0.z; v[3] = t0.w;
            v[4] = v[5] = v[6] = v[7] = 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < valid ? __ldg(p + i) : 0.f;
        }
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

// LANES lanes per row (16 or 32: part of a warp; 256: the CTA), CHUNKS pieces
// of 8 columns a lane kept in registers. REREAD: rows longer than LANES *
// CHUNKS * 8 columns are read a second time for the codes.
template <int FORMAT, bool BF16, int LANES, int CHUNKS, bool REREAD>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const QuantArgs a) {
    constexpr bool kNv = FORMAT == GAT_B200_NVFP4;
    constexpr int kBlockLanes = fp4_block(FORMAT) / 8;  // lanes of one block
    constexpr int kWordLanes = 4 * kBlockLanes;          // lanes of one scale word
    const int lane = threadIdx.x % LANES;
    const uint64_t row = LANES >= 256 ? uint64_t(blockIdx.x) : uint64_t(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const bool live = row < a.n;
    const uint64_t xoff = row * uint64_t(a.ldx);
    float v[CHUNKS][8];
    float mine[CHUNKS];

    auto fetch = [&](int c0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = ((c0 + c) * LANES + lane) * 8;
            const int valid = live ? min(8, a.width - col) : 0;
            if (valid > 0) {
                load8<BF16>(a, xoff + uint64_t(col), valid, v[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
            }
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float m = fabsf(v[c][0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[c][i]));
            mine[c] = m;
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

    const int steps = REREAD || !kNv ? (a.chunks + LANES * CHUNKS - 1) / (LANES * CHUNKS) : 1;
    for (int s = 0; s < steps; ++s) {
        if (!kNv || REREAD) fetch(s * CHUNKS);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int chunk = (s * CHUNKS + c) * LANES + lane;
            if ((s * CHUNKS + c) * LANES >= a.chunks) break;  // the same for all lanes of the row
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
                inv = sc > 0.f ? __frcp_rn(sc) * rinv : 0.f;
            } else {
                const uint32_t u = __float_as_uint(m);
                const int e = int(u >> 23) - 2;  // biased exponent of the scale
                byte = u >= 0x7f800000u ? 255u : (e > 0 ? uint32_t(e) : 0u);
                d = byte == 255u ? __uint_as_float(0x7fc00000u)
                                 : (byte ? __uint_as_float(byte << 23) : __uint_as_float(0x400000u));
                inv = byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
            }
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = v[c][i] * inv;
                if constexpr (kNv) q[i] = fmaf(fmaf(-q[i], d, v[c][i]), inv, q[i]);
            }
            uint32_t code = e2m1x8(q);
            if (inv == 0.f) code = 0;
            // the four scale bytes of a word, in the lane of its first block
            uint32_t word = byte;
            word |= __shfl_down_sync(0xffffffffu, byte, kBlockLanes) << 8;
            word |= __shfl_down_sync(0xffffffffu, byte, 2 * kBlockLanes) << 16;
            word |= __shfl_down_sync(0xffffffffu, byte, 3 * kBlockLanes) << 24;
            if (!live || chunk >= a.chunks) continue;
            if (chunk < a.code_chunks)
                *reinterpret_cast<uint32_t*>(a.codes + row * uint64_t(a.ldc) + uint64_t(chunk) * 4) = code;
            if (chunk % kWordLanes == 0)
                *reinterpret_cast<uint32_t*>(a.scales + ((row >> 7) * uint64_t(a.tiles) + chunk / kWordLanes) * 512 +
                                             (row & 31) * 16 + ((row >> 5) & 3) * 4) = word;
            const int valid = min(8, a.width - chunk * 8);
            if (a.values && valid > 0) {
                float y[8];
                from_e2m1x8(code, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= d;
                const uint64_t off = row * uint64_t(a.ldv) + uint64_t(chunk) * 8;
                if (a.v_align < 0) {  // FP32 values
                    float* p = static_cast<float*>(a.values) + off;
                    if (valid == 8 && a.v_align <= -16) {
                        reinterpret_cast<float4*>(p)[0] = make_float4(y[0], y[1], y[2], y[3]);
                        reinterpret_cast<float4*>(p)[1] = make_float4(y[4], y[5], y[6], y[7]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < valid) p[i] = y[i];
                    }
                } else {  // BF16: the values have at most six significant bits
                    uint16_t* p = static_cast<uint16_t*>(a.values) + off;
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
                    if (valid == 8 && a.v_align >= 16) {
                        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else if (a.v_align >= 8 && (valid & 3) == 0) {
                        reinterpret_cast<uint2*>(p)[0] = make_uint2(w[0], w[1]);
                        if (valid == 8) reinterpret_cast<uint2*>(p)[1] = make_uint2(w[2], w[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < valid) p[i] = uint16_t(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
                    }
                }
            }
        }
    }
}

// Alignment in bytes (at most 16) of base and of every row at `pitch` bytes.
int row_align(const void* base, uint64_t pitch) {
    const uint64_t u = uint64_t(reinterpret_cast<uintptr_t>(base)) | pitch | 16;
    return int(u & (~u + 1));
}

template <int FORMAT, bool BF16>
int launch_quantize(const QuantArgs& a, cudaStream_t st) {
    // 16 or 32 lanes a row while a row fits them once, one warp up to 1024
    // columns, the CTA for longer ones; above 16384 columns NVFP4 reads twice.
    const uint64_t per16 = (a.n + 15) / 16, per8 = (a.n + 7) / 8;
    if (a.chunks <= 16)
        fp4_quantize_kernel<FORMAT, BF16, 16, 1, false><<<unsigned(per16), 256, 0, st>>>(a);
    else if (a.chunks <= 32)
        fp4_quantize_kernel<FORMAT, BF16, 32, 1, false><<<unsigned(per8), 256, 0, st>>>(a);
    else if (a.chunks <= 64)
        fp4_quantize_kernel<FORMAT, BF16, 32, 2, false><<<unsigned(per8), 256, 0, st>>>(a);
    else if (a.chunks <= 128)
        fp4_quantize_kernel<FORMAT, BF16, 32, 4, false><<<unsigned(per8), 256, 0, st>>>(a);
    else if (a.chunks <= 256)
        fp4_quantize_kernel<FORMAT, BF16, 256, 1, false><<<unsigned(a.n), 256, 0, st>>>(a);
    else if (a.chunks <= 512)
        fp4_quantize_kernel<FORMAT, BF16, 256, 2, false><<<unsigned(a.n), 256, 0, st>>>(a);
    else if (a.chunks <= 1024)
        fp4_quantize_kernel<FORMAT, BF16, 256, 4, false><<<unsigned(a.n), 256, 0, st>>>(a);
    else
        fp4_quantize_kernel<FORMAT, BF16, 256, 4, true><<<unsigned(a.n), 256, 0, st>>>(a);
    GATB_LAUNCH("fp4_quantize kernel");
    return 0;
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
    a.x_align = row_align(x, uint64_t(ldx) * xs);
    a.codes = static_cast<uint8_t*>(codes);
    a.ldc = ldc;
    a.scales = static_cast<uint8_t*>(scales);
    a.row_scale = row_scale;
    a.values = values;
    a.ldv = ldv;
    a.v_align = values ? row_align(values, uint64_t(ldv) * vs) * (v_dtype == GAT_B200_F32 ? -1 : 1) : 0;
    if (format == GAT_B200_MXFP4)
        return x_dtype == GAT_B200_BF16 ? launch_quantize<GAT_B200_MXFP4, true>(a, st)
                                        : launch_quantize<GAT_B200_MXFP4, false>(a, st);
    return x_dtype == GAT_B200_BF16 ? launch_quantize<GAT_B200_NVFP4, true>(a, st)
                                    : launch_quantize<GAT_B200_NVFP4, false>(a, st);
}

}  // namespace gatb
