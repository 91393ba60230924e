// Product of two 4-bit microscaled tables on the tensor cores:
//   out[i][j] = ra[i] rb[j] sum_k (sa qa)[i][k] (sb qb)[j][k], FP32 accumulators.
// tcgen05.mma kind::mxf4 / mxf4nvf4 multiplies the block scales in the
// tensor core, out of tensor memory, where tcgen05.cp brings them from shared
// memory in the tables' own tile order (fp4.cuh).
//
// Persistent kernel, one CTA per SM, 6 warps:
//   warp 0  TMA producer: stages of 256 columns (128 bytes a row, 128-byte
//           swizzle) of 128 rows of a and of b with their scale tiles.
//   warp 1  scale copies and MMAs into one of two TMEM accumulators.
//   warps 2-5 epilogue: TMEM -> row scales -> rounding -> global.
// Every wait is bounded (GAT_B200_ETIMEOUT through gat_b200_check_device).
#include <cuda.h>

#include "fp4.cuh"
#include "tc.cuh"

namespace gatb {

__device__ unsigned g_fp4_error = 0;

int make_tiled_map(CUtensorMap* m, int type, int rank, const void* base, const uint64_t* dims, const uint64_t* strides,
                   const uint32_t* box, bool swizzle);
int fp4_check_format(const char* what, int format);

namespace {

using namespace tc;

constexpr int kBM = 128, kBN = 128;
constexpr int kStages = 5;
constexpr int kThreads = 192;

struct ProductArgs {
    uint64_t m;
    int n;
    int stages_k;   // 256-column stages of the reduction
    int last_mmas;  // 64-column MMAs of the last stage
    int tiles;      // scale tiles along a row
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    const float* a_row;
    const float* b_row;
    void* out;
    int ldo;
    int out_bf16;
    uint32_t grid_m, grid_n;
};

template <int FORMAT>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ ProductArgs g) {
    constexpr bool kMx = FORMAT == GAT_B200_MXFP4;
    constexpr int kTileMmas = kMx ? 2 : 1;           // MMAs served by one scale tile
    constexpr int kSfTiles = 4 / kTileMmas;          // scale tiles of a stage
    constexpr int kABytes = kBM * 128, kBBytes = kBN * 128, kSfBytes = kSfTiles * 512;
    constexpr int kStageBytes = kABytes + kBBytes + 2 * kSfBytes;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sf_s = smem + size_t(kStages) * (kABytes + kBBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + size_t(kStages) * kStageBytes);
    uint64_t* full = bars;
    uint64_t* empty = bars + kStages;
    uint64_t* acc_full = bars + 2 * kStages;  // [2]
    uint64_t* acc_empty = acc_full + 2;       // [2]
    uint64_t* mma_done = acc_empty + 2;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ntiles = g.grid_m * g.grid_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + b, 1);
            mbar_init(acc_empty + b, 4);
        }
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t kc = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
                const uint32_t tm = t % g.grid_m, tn = t / g.grid_m;
                for (int k = 0; k < g.stages_k; ++k, ++kc) {
                    const int s = int(kc % kStages);
                    if (!mbar_wait(empty + s, ((kc / kStages) & 1u) ^ 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                    const int sft = min(kSfTiles, g.tiles - k * kSfTiles);
                    mbar_expect_tx(full + s, kABytes + kBBytes + 2 * 512 * sft);
                    uint8_t* a_s = smem + size_t(s) * (kABytes + kBBytes);
                    tma_load_2d(a_s, &tm_a, full + s, k * 128, int(tm * kBM));
                    tma_load_2d(a_s + kABytes, &tm_b, full + s, k * 128, int(tn * kBN));
                    uint8_t* sf = sf_s + size_t(s) * 2 * kSfBytes;
                    bulk_load(sf, g.a_scales + (uint64_t(tm) * g.tiles + k * kSfTiles) * 512, 512 * sft, full + s);
                    bulk_load(sf + kSfBytes, g.b_scales + (uint64_t(tn) * g.tiles + k * kSfTiles) * 512, 512 * sft, full + s);
                }
            }
            for (int s = 0; s < kStages; ++s)
                if (kc > uint32_t(s)) {
                    const uint32_t last = kc - 1 - ((kc - 1 - s) % kStages);
                    mbar_wait(full + s, (last / kStages) & 1u, abort_flag, &g_fp4_error);
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t kc = 0, tl = 0;
            bool ok = true;
            const uint32_t sf_t = tmem + 256;
            for (uint32_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ++tl) {
                const uint32_t buf = tl & 1u;
                if (!mbar_wait(acc_empty + buf, ((tl >> 1) & 1u) ^ 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                fence_after();
                const uint32_t d = tmem + buf * 128;
                for (int k = 0; k < g.stages_k; ++k, ++kc) {
                    const int s = int(kc % kStages);
                    if (!mbar_wait(full + s, (kc / kStages) & 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                    fence_after();
                    const uint32_t a_addr = smem_u32(smem + size_t(s) * (kABytes + kBBytes));
                    const uint32_t b_addr = a_addr + kABytes;
                    const uint32_t sfa_s = smem_u32(sf_s + size_t(s) * 2 * kSfBytes), sfb_s = sfa_s + kSfBytes;
                    const int mmas = k + 1 == g.stages_k ? g.last_mmas : 4;
                    const uint32_t sfa = sf_t + (kc & 1u) * (8 * kSfTiles), sfb = sfa + 4 * kSfTiles;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j >= mmas) break;
                        const int st = j / kTileMmas;
                        if (j % kTileMmas == 0) {
                            tmem_cp_scales<1>(sfa + st * 4, desc_scales(sfa_s + st * 512));
                            tmem_cp_scales<1>(sfb + st * 4, desc_scales(sfb_s + st * 512));
                        }
                        mma_fp4<kMx, 1>(d, desc_sw128(a_addr + j * 32, 16, 1024), desc_sw128(b_addr + j * 32, 16, 1024),
                                        idesc_fp4(kBM, kBN, kMx, kMx ? 2 * (j & 1) : 0), sfa + st * 4, sfb + st * 4,
                                        (k | j) ? 1u : 0u);
                    }
                    mma_commit(empty + s);
                }
                if (!ok) break;
                mma_commit(acc_full + buf);
            }
            mma_commit(mma_done);
            mbar_wait(mma_done, 0, abort_flag, &g_fp4_error);
        }
    } else {
        const int q = warp & 3;
        uint32_t tl = 0;
        for (uint32_t t = blockIdx.x; t < ntiles; t += gridDim.x, ++tl) {
            const uint32_t tm = t % g.grid_m, tn = t / g.grid_m;
            const uint32_t buf = tl & 1u;
            if (!mbar_wait(acc_full + buf, (tl >> 1) & 1u, abort_flag, &g_fp4_error)) break;
            fence_after();
            const uint64_t row = uint64_t(tm) * kBM + q * 32 + lane;
            const float ra = g.a_row && row < g.m ? g.a_row[row] : 1.f;
#pragma unroll
            for (int c = 0; c < kBN; c += 32) {
                float v[32];
                tmem_ld32(tmem + buf * 128 + (uint32_t(q * 32) << 16) + c, v);
                const int col = int(tn) * kBN + c;
                if (row < g.m) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (col + j < g.n) {
                            const float y = g.b_row ? v[j] * ra * __ldg(g.b_row + col + j) : v[j] * ra;
                            const uint64_t off = row * uint64_t(g.ldo) + col + j;
                            if (g.out_bf16)
                                static_cast<uint16_t*>(g.out)[off] = uint16_t(pack_bf16x2(y, 0.f));
                            else
                                static_cast<float*>(g.out)[off] = y;
                        }
                }
                __syncwarp();
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + buf);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Codes as bytes: rows of `row_bytes`, boxes of 128 bytes x `box_rows` rows.
int codes_map(CUtensorMap* m, const void* base, uint64_t rows, int row_bytes, int ld, uint32_t box_rows) {
    const uint64_t dims[2] = {uint64_t(row_bytes), rows};
    const uint64_t strides[1] = {uint64_t(ld)};
    const uint32_t box[2] = {128, box_rows};
    return make_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, true);
}

template <int FORMAT>
int launch_product(const ProductArgs& g, const CUtensorMap& tm_a, const CUtensorMap& tm_b, int sms, cudaStream_t st) {
    constexpr int sf = FORMAT == GAT_B200_MXFP4 ? 1024 : 2048;
    const size_t smem = size_t(kStages) * (kBM * 128 + kBN * 128 + 2 * sf) + 256 + 1024;
    auto kern = fp4_product_kernel<FORMAT>;
    GATB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    const uint32_t ntiles = g.grid_m * g.grid_n;
    kern<<<ntiles < uint32_t(sms) ? ntiles : sms, kThreads, smem, st>>>(tm_a, tm_b, g);
    GATB_LAUNCH("fp4_product kernel");
    return 0;
}

}  // namespace

int fp4_product_launch(int format, uint64_t m, int n, int k, const void* a, int lda, const void* a_scales,
                       const float* a_row, const void* b, int ldb, const void* b_scales, const float* b_row, void* out,
                       int out_dtype, int ldo, cudaStream_t st) {
    if (int rc = fp4_check_format("fp4_product", format)) return rc;
    if (out_dtype != GAT_B200_F32 && out_dtype != GAT_B200_BF16) return fail("fp4_product: bad output dtype");
    if (n < 0 || k <= 0 || k > (1 << 24)) return fail("fp4_product: bad shape");
    if (m > uint64_t(INT32_MAX - 256) || n > INT32_MAX - 256) return fail("fp4_product: too many rows");
    const int kb = fp4_row_bytes(k);
    if (lda < kb || lda % 16 || ldb < kb || ldb % 16)
        return fail("fp4_product: code rows must be 16-byte aligned and hold the width");
    if (ldo < n) return fail("fp4_product: output row stride smaller than the width");
    if (m == 0 || n == 0) return 0;
    if (!a || !a_scales || !b || !b_scales || !out) return fail("fp4_product: null argument");
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b) |
         reinterpret_cast<uintptr_t>(b_scales)) & 15)
        return fail("fp4_product: codes and scales must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(out) % (out_dtype == GAT_B200_BF16 ? 2 : 4) ||
        (reinterpret_cast<uintptr_t>(a_row) | reinterpret_cast<uintptr_t>(b_row)) % 4)
        return fail("fp4_product: misaligned pointer");
    if (int rc = check_device_pointers("fp4_product", {a, a_scales, a_row, b, b_scales, b_row, out})) return rc;
    ProductArgs g{};
    g.m = m;
    g.n = n;
    g.stages_k = (kb + 127) / 128;
    g.last_mmas = (k - (g.stages_k - 1) * 256 + 63) / 64;
    g.tiles = fp4_tiles(format, k);
    g.a_scales = static_cast<const uint8_t*>(a_scales);
    g.b_scales = static_cast<const uint8_t*>(b_scales);
    g.a_row = a_row;
    g.b_row = b_row;
    g.out = out;
    g.ldo = ldo;
    g.out_bf16 = out_dtype == GAT_B200_BF16;
    g.grid_m = uint32_t((m + kBM - 1) / kBM);
    g.grid_n = uint32_t((n + kBN - 1) / kBN);
    if (uint64_t(g.grid_m) * g.grid_n > uint64_t(INT32_MAX)) return fail("fp4_product: output too large");
    int dev = 0, sms = 0;
    GATB_CUDA(cudaGetDevice(&dev));
    GATB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    CUtensorMap tm_a, tm_b;
    if (int rc = codes_map(&tm_a, a, m, kb, lda, kBM)) return rc;
    if (int rc = codes_map(&tm_b, b, uint64_t(n), kb, ldb, kBN)) return rc;
    return format == GAT_B200_MXFP4 ? launch_product<GAT_B200_MXFP4>(g, tm_a, tm_b, sms, st)
                                    : launch_product<GAT_B200_NVFP4>(g, tm_a, tm_b, sms, st);
}

int fp4_check_error() {
    unsigned e = 0;
    GATB_CUDA(cudaMemcpyFromSymbol(&e, g_fp4_error, sizeof(e)));
    if (e) {
        unsigned z = 0;
        cudaMemcpyToSymbol(g_fp4_error, &z, sizeof(z));
        return fail_code(GAT_B200_ETIMEOUT, "fp4_product kernel: a bounded wait timed out");
    }
    return 0;
}

}  // namespace gatb
