// Product of two 4-bit microscaled tables on the tensor cores:
//   out[i][j] = ra[i] rb[j] sum_k (sa qa)[i][k] (sb qb)[j][k], FP32 accumulators.
// tcgen05.mma kind::mxf4 / mxf4nvf4 multiplies the block scales in the
// tensor core, out of tensor memory, where tcgen05.cp brings them from shared
// memory in the tables' own tile order (fp4.cuh).
//
// Two kernels; launch_product chooses between them.
//  pair_kernel  256 x 256 tiles of a CTA pair (cta_group::2), persistent.
//  rows_kernel  128 rows of b x BN rows of a, the reduction split over a cluster
//               and joined through distributed shared memory: few rows, small outputs.
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
    int tma_out;  // output rows are 16-byte aligned: tiles leave through TMA stores
    int n_whole;  // n columns are whole 16-byte pieces
    uint32_t grid_m, grid_n;
};

// MMAs served by one 4-block scale tile, scale tiles of a 256-column stage.
template <int FORMAT>
struct Scales {
    static constexpr bool kMx = FORMAT == GAT_B200_MXFP4;
    static constexpr int kTileMmas = kMx ? 2 : 1;
    static constexpr int kTiles = 4 / kTileMmas;
    static constexpr int kBytes = kTiles * 512;  // of 128 rows in a stage
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// Only tensor memory is handed over by it (tcgen05 fences order that), so it
// needs no release at cluster scope, which waits for every store: 1100 cycles.
__device__ __forceinline__ void mbar_arrive_rank(uint64_t* bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(smem_u32(bar), rank)) : "memory");
}
// Loads of a CTA pair count on the first CTA's barrier (bit 24 of a shared
// address holds the CTA's parity in the pair).
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar) & 0xfeffffffu), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
}

// A sum v times two row scales a and b may well be an FP32 number where a b is
// none (rows of huge or tiny elements). NVFP4's v is zero or at least 2^-20
// (products of block scales and elements), at most 2^23 k, so ((v first) b) rest
// with a = first * rest, rest a power of two, leaves FP32's range only where the
// result does. (MXFP4's block scales span FP32's range by themselves.)
__device__ __forceinline__ bool ordinary(float x) { return fabsf(x) >= 0x1p-50f && fabsf(x) <= 0x1p50f; }
__device__ __forceinline__ float split_scale(float a, float& rest) {
    const float m = fabsf(a);
    const bool huge = m > 0x1p80f, tiny = m < 0x1p-100f;
    rest = huge ? 0x1p40f : tiny ? 0x1p-50f : 1.f;
    return a * (huge ? 0x1p-40f : tiny ? 0x1p50f : 1.f);
}

// ------------------------------------------------------------ CTA pairs
// Roles of the 20 warps of each CTA of a pair (2 and 3 idle):
//   warp 0    TMA producer: this CTA's 128 rows of a, 128 of the tile's 256 rows
//             of b (the pair's MMA reads both halves) and their scales; the
//             scales of b's whole tile, which each CTA's tensor memory holds.
//   warp 1    first CTA only: scale copies and MMAs of the pair.
//   warps 4-19 epilogue: 32 rows x 64 columns of this CTA's 128 x 256
//             accumulators each, in registers at once, so the next tile's MMAs
//             start while this one is scaled, rounded and stored.
// Tensor memory: accumulators in columns 0-255, scales in 448-511 (two whole
// accumulators and the scales do not fit): a tile's MMAs wait until all epilogue
// warps have the one before it in registers.
constexpr int kEpiWarps = 16;
constexpr int kPairThreads = 128 + 32 * kEpiWarps;
constexpr int kPairStages = 4;
constexpr int kScaleCols = 448;

template <int FORMAT>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb,
                const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ ProductArgs g) {
    using S = Scales<FORMAT>;
    constexpr int kHalf = 128 * 128;  // codes of 128 rows in a stage
    constexpr int kStage = 2 * kHalf + 3 * S::kBytes;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* st_s = smem + kPairStages * 2 * kHalf;               // 4 KB per epilogue warp
    uint8_t* sf_s = st_s + kEpiWarps * 4096;                       // stages x 3 scale pieces
    float* rb_s = reinterpret_cast<float*>(sf_s + kPairStages * 3 * S::kBytes);  // 64 per epilogue warp
    uint64_t* bars = reinterpret_cast<uint64_t*>(rb_s + kEpiWarps * 64);
    uint64_t* full = bars;
    uint64_t* empty = full + kPairStages;
    uint64_t* acc_full = empty + kPairStages;
    uint64_t* drained = acc_full + 1;
    uint64_t* mma_done = drained + 1;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t ntiles = g.grid_m * g.grid_n;
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    // 8 row tiles by all column tiles at a time, so that the tiles in flight share rows and columns in L2
    auto tile_at = [&](uint32_t t, uint32_t& tm, uint32_t& tn) {
        const uint32_t per = 8 * g.grid_n, grp = t / per, in = t % per;
        const uint32_t rows = min(8u, g.grid_m - grp * 8);
        tm = grp * 8 + in % rows;
        tn = in / rows;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drained, 2 * kEpiWarps);
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t kc = 0;
            bool ok = true;
            for (uint32_t t = pair; t < ntiles && ok; t += pairs) {
                uint32_t tm, tn;
                tile_at(t, tm, tn);
                const int arow = int(tm * 256 + rank * 128), brow = int(tn * 256 + rank * 128);
                for (int k = 0; k < g.stages_k; ++k, ++kc) {
                    const int s = int(kc % kPairStages);
                    if (!mbar_wait(empty + s, ((kc / kPairStages) & 1u) ^ 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(full + s, 2 * kStage);
                    uint8_t* c = smem + s * 2 * kHalf;
                    uint8_t* f = sf_s + s * 3 * S::kBytes;
                    pair_load_2d(c, &tm_a, full + s, k * 128, arow);
                    pair_load_2d(c + kHalf, &tm_b, full + s, k * 128, brow);
                    // boxes of a stage's scale tiles; past a row's last tile they hold what no MMA uses
                    pair_load_2d(f, &tm_sa, full + s, 0, int((tm * 2 + rank) * g.tiles) + k * S::kTiles);
                    pair_load_2d(f + S::kBytes, &tm_sb, full + s, 0, int(tn * 2 * g.tiles) + k * S::kTiles);
                    pair_load_2d(f + 2 * S::kBytes, &tm_sb, full + s, 0, int((tn * 2 + 1) * g.tiles) + k * S::kTiles);
                }
            }
            // every load has landed once its stage came back (or, at the first CTA, filled)
            for (uint32_t i = kc > kPairStages ? kc - kPairStages : 0; i < kc; ++i)
                mbar_wait(empty + i % kPairStages, (i / kPairStages) & 1u, abort_flag, &g_fp4_error);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t kc = 0, tl = 0;
            bool ok = true;
            const uint32_t sfa0 = tmem + kScaleCols, sfb0 = sfa0 + 4 * S::kTiles;
            for (uint32_t t = pair; t < ntiles && ok; t += pairs, ++tl) {
                if (tl && !mbar_wait_warp(drained, (tl - 1) & 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                fence_after();
                for (int k = 0; k < g.stages_k; ++k, ++kc) {
                    const int s = int(kc % kPairStages);
                    if (!mbar_wait_warp(full + s, (kc / kPairStages) & 1u, abort_flag, &g_fp4_error)) { ok = false; break; }
                    fence_after();
                    const uint32_t a_addr = smem_u32(smem + s * 2 * kHalf), b_addr = a_addr + kHalf;
                    const uint64_t adesc = desc_sw128(a_addr, 16, 1024), bdesc = desc_sw128(b_addr, 16, 1024);
                    const uint64_t fdesc = desc_scales(smem_u32(sf_s + s * 3 * S::kBytes));
                    const int mmas = k + 1 == g.stages_k ? g.last_mmas : 4;
                    if (elect_one()) {
                        // descriptors count in 16 bytes
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (j >= mmas) break;
                            const int st = j / S::kTileMmas;
                            const uint32_t sfa = sfa0 + st * 4, sfb = sfb0 + st * 8;
                            if (j % S::kTileMmas == 0) {
                                tmem_cp_scales<2>(sfa, fdesc + st * 32);
                                tmem_cp_scales<2>(sfb, fdesc + S::kBytes / 16 + st * 32);
                                tmem_cp_scales<2>(sfb + 4, fdesc + 2 * S::kBytes / 16 + st * 32);
                            }
                            mma_fp4<S::kMx, 2>(tmem, adesc + j * 2, bdesc + j * 2,
                                               idesc_fp4(256, 256, S::kMx, S::kMx ? 2 * (j & 1) : 0), sfa, sfb,
                                               (k | j) ? 1u : 0u);
                        }
                        pair_commit(empty + s);
                        if (k + 1 == g.stages_k) pair_commit(acc_full);
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) pair_commit(mma_done);
            mbar_wait_warp(mma_done, 0, abort_flag, &g_fp4_error);
        }
    } else if (warp >= 4) {
        const int q = warp & 3, ew = warp - 4, grp = ew >> 2;
        uint8_t* sb = st_s + ew * 4096;
        float* rb = rb_s + ew * 64;
        // the row scales of a tile, fetched while the one before it is worked on
        float ra = 1.f, rb0 = 1.f, rb1 = 1.f;
        uint32_t tm = 0, tn = 0;
        auto fetch = [&](uint32_t t) {
            tile_at(t, tm, tn);
            const uint64_t r = uint64_t(tm) * 256 + rank * 128 + q * 32 + lane;
            if (g.a_row && r < g.m) ra = g.a_row[r];
            const int c = int(tn) * 256 + grp * 64 + lane;
            if (g.b_row && c < g.n) rb0 = g.b_row[c];
            if (g.b_row && c + 32 < g.n) rb1 = g.b_row[c + 32];
        };
        if (pair < ntiles) fetch(pair);
        uint32_t tl = 0;
        for (uint32_t t = pair; t < ntiles; t += pairs, ++tl) {
            const uint64_t row0 = uint64_t(tm) * 256 + rank * 128 + q * 32;
            const int col = int(tn) * 256 + grp * 64;
            const float ra_t = ra;
            // outside the usual range of scales the tile takes them one after the other
            const bool wild = __any_sync(0xffffffffu, !ordinary(ra) || !ordinary(rb0) || !ordinary(rb1));
            __syncwarp();  // the last tile's reads of rb
            rb[lane] = rb0;
            rb[lane + 32] = rb1;
            __syncwarp();
            if (t + pairs < ntiles) fetch(t + pairs);
            if (!mbar_wait_warp(acc_full, tl & 1u, abort_flag, &g_fp4_error)) break;
            fence_after();
            float v[64];
            tmem_ld64(tmem + (uint32_t(q * 32) << 16) + grp * 64, v);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_rank(drained, 0);
            if (col >= g.n || row0 >= g.m) continue;
            if (wild && g.b_row) {
                float rest;
                const float first = split_scale(ra_t, rest);
#pragma unroll
                for (int c = 0; c < 64; ++c) v[c] = v[c] * first * rb[c] * rest;
            } else if (g.b_row) {
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const float4 b4 = *reinterpret_cast<const float4*>(rb + c);
                    v[c] *= ra_t * b4.x;
                    v[c + 1] *= ra_t * b4.y;
                    v[c + 2] *= ra_t * b4.z;
                    v[c + 3] *= ra_t * b4.w;
                }
            } else if (g.a_row) {
#pragma unroll
                for (int c = 0; c < 64; ++c) v[c] *= ra_t;
            }
            // 32 rows x 128 bytes at a time, 16-byte pieces swizzled as the TMA store expects
            auto stage = [&](int h, auto piece) {
                const int c0 = col + h * 32, width = g.out_bf16 ? 64 : 32;
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4*>(sb + lane * 128 + ((c ^ (lane & 7)) * 16)) = piece(c);
                // a TMA store writes whole 16-byte pieces: the last columns go out one by one unless n ends a piece
                if (g.tma_out && (g.n_whole || c0 + width <= g.n)) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_out, sb, c0, int(row0));
                        bulk_commit();
                    }
                } else {
                    // a lane takes 4 bytes of a row: two BF16 columns or an FP32 one
                    __syncwarp();
                    const int live = int(min(uint64_t(32), g.m - row0));
                    const int c = g.out_bf16 ? c0 + 2 * lane : c0 + lane;
                    const bool pair = g.ldo % 2 == 0 && reinterpret_cast<uintptr_t>(g.out) % 4 == 0;
                    uint8_t* o = static_cast<uint8_t*>(g.out) + (row0 * uint64_t(g.ldo) + c) * (g.out_bf16 ? 2 : 4);
                    const uint64_t pitch = uint64_t(g.ldo) * (g.out_bf16 ? 2 : 4);
#pragma unroll 8
                    for (int r = 0; r < 32; ++r) {
                        if (r >= live) break;
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(sb + r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4);
                        uint8_t* p = o + r * pitch;
                        if (!g.out_bf16) {
                            if (c < g.n) *reinterpret_cast<uint32_t*>(p) = w;
                        } else if (pair && c + 1 < g.n) {
                            *reinterpret_cast<uint32_t*>(p) = w;
                        } else {
                            if (c < g.n) *reinterpret_cast<uint16_t*>(p) = uint16_t(w);
                            if (c + 1 < g.n) *reinterpret_cast<uint16_t*>(p + 2) = uint16_t(w >> 16);
                        }
                    }
                    __syncwarp();
                }
            };
            if (g.out_bf16) {
                stage(0, [&](int c) {
                    return make_uint4(pack_bf16x2(v[8 * c], v[8 * c + 1]), pack_bf16x2(v[8 * c + 2], v[8 * c + 3]),
                                      pack_bf16x2(v[8 * c + 4], v[8 * c + 5]), pack_bf16x2(v[8 * c + 6], v[8 * c + 7]));
                });
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (col + 32 * h >= g.n) break;
                    stage(h, [&](int c) {
                        return make_uint4(__float_as_uint(v[32 * h + 4 * c]), __float_as_uint(v[32 * h + 4 * c + 1]),
                                          __float_as_uint(v[32 * h + 4 * c + 2]), __float_as_uint(v[32 * h + 4 * c + 3]));
                    });
                }
            }
        }
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ------------------------------------------------------------- few rows
// out^T: 128 rows of b (an MMA's M) x BN rows of a (its N). The SPLIT CTAs of a
// cluster take a part of the reduction each, leave their FP32 tile in shared
// memory, and each sums a share of the tile's columns over the cluster in rank
// order, so results do not depend on timing. 6 warps: producer, MMA, 4 epilogue.
constexpr int kRowsThreads = 192;

template <int BN>
struct RowsTile {
    static constexpr int kStages = BN <= 16 ? 5 : BN == 64 ? 3 : 4;  // so that kCtas fit an SM's shared memory
    static constexpr int kCols = BN <= 16 ? 32 : BN;  // accumulator columns, up to 32 of scales behind them
    static constexpr int kTmem = BN <= 32 ? 64 : (BN <= 64 ? 128 : 256);
    static constexpr int kCtas = BN <= 64 ? 2 : 1;  // an SM, by shared memory
};

template <int FORMAT, int BN>
__global__ void __launch_bounds__(kRowsThreads)
    rows_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ ProductArgs g, const int split) {
    using S = Scales<FORMAT>;
    constexpr int kSt = RowsTile<BN>::kStages, kTmem = RowsTile<BN>::kTmem;
    constexpr int kB = 128 * 128, kA = BN * 128;  // codes of a stage: b's rows, a's rows
    constexpr int kStage = kB + kA + 2 * S::kBytes;
    constexpr int kPitch = 128 + 4;               // floats of a column of out^T in the exchange buffer
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* a_s = smem + kSt * kB;
    uint8_t* sf_s = a_s + kSt * kA;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSt * kStage);
    uint64_t* full = bars;
    uint64_t* empty = full + kSt;
    uint64_t* acc_full = empty + kSt;
    float* rb_s = reinterpret_cast<float*>(bars + 16);  // [128] row scales of b, [BN] of a
    float* ra_s = rb_s + 128;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ra_s + BN);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    float* part = reinterpret_cast<float*>(smem);  // [BN][kPitch], over the stages once they are used up
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = split > 1 ? cluster_rank() : 0;
    const uint32_t tile = blockIdx.x / split;
    const uint32_t tn = tile % g.grid_n, tm = tile / g.grid_n;  // 128 rows of b, BN rows of a
    const int k0 = int(uint64_t(g.stages_k) * rank / split), k1 = int(uint64_t(g.stages_k) * (rank + 1) / split);
    const uint64_t arow = uint64_t(tm) * BN;
    auto load = [&](int k) {
        const int s = (k - k0) % kSt;
        const int sft = min(S::kTiles, g.tiles - k * S::kTiles);
        mbar_expect_tx(full + s, kB + kA + 2 * 512 * sft);
        tma_load_2d(smem + s * kB, &tm_b, full + s, k * 128, int(tn * 128));
        tma_load_2d(a_s + s * kA, &tm_a, full + s, k * 128, int(arow));
        uint8_t* f = sf_s + s * 2 * S::kBytes;
        bulk_load(f, g.b_scales + (uint64_t(tn) * g.tiles + k * S::kTiles) * 512, 512 * sft, full + s);
        bulk_load(f + S::kBytes, g.a_scales + ((arow >> 7) * uint64_t(g.tiles) + k * S::kTiles) * 512, 512 * sft, full + s);
    };

    const int q = warp & 3;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSt; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        mbar_init(acc_full, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
        // the first stages are on their way while the CTA sets itself up
        for (int k = k0; k < min(k1, k0 + kSt); ++k) load(k);
    } else if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"(kTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp >= 2) {
        const int i = threadIdx.x - 64, col = int(tn) * 128 + i;
        rb_s[i] = g.b_row && col < g.n ? g.b_row[col] : 1.f;
        for (int r = i; r < BN; r += 128) ra_s[r] = g.a_row && arow + r < g.m ? g.a_row[arow + r] : 1.f;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0) {
            int k = min(k1, k0 + kSt);
            for (; k < k1; ++k) {
                const int i = k - k0;
                if (!mbar_wait(empty + i % kSt, ((uint32_t(i) / kSt) & 1u) ^ 1u, abort_flag, &g_fp4_error)) break;
                load(k);
            }
            for (int i = max(0, k - k0 - kSt); i < k - k0; ++i)
                mbar_wait(full + i % kSt, (uint32_t(i) / kSt) & 1u, abort_flag, &g_fp4_error);
        }
    } else if (warp == 1) {
        // scales behind the accumulator; a's rows start a scale tile (below 128 rows there is one tile of them)
        const uint32_t sfb0 = tmem + RowsTile<BN>::kCols, sfa0 = sfb0 + 4 * S::kTiles;
        for (int k = k0; k < k1; ++k) {
            const int i = k - k0, s = i % kSt;
            if (!mbar_wait_warp(full + s, (uint32_t(i) / kSt) & 1u, abort_flag, &g_fp4_error)) break;
            fence_after();
            const uint64_t adesc = desc_sw128(smem_u32(a_s + s * kA), 16, 1024);
            const uint64_t bdesc = desc_sw128(smem_u32(smem + s * kB), 16, 1024);
            const uint64_t fdesc = desc_scales(smem_u32(sf_s + s * 2 * S::kBytes));
            const int mmas = k + 1 == g.stages_k ? g.last_mmas : 4;
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= mmas) break;
                    const int st = j / S::kTileMmas;
                    if (j % S::kTileMmas == 0) {
                        tmem_cp_scales<1>(sfb0 + st * 4, fdesc + st * 32);
                        tmem_cp_scales<1>(sfa0 + st * 4, fdesc + S::kBytes / 16 + st * 32);
                    }
                    mma_fp4<S::kMx, 1>(tmem, bdesc + j * 2, adesc + j * 2,
                                       idesc_fp4(128, BN, S::kMx, S::kMx ? 2 * (j & 1) : 0), sfb0 + st * 4, sfa0 + st * 4,
                                       (i | j) ? 1u : 0u);
                }
                mma_commit(empty + s);
            }
            __syncwarp();
        }
        if (elect_one()) mma_commit(acc_full);
        mbar_wait_warp(acc_full, 0, abort_flag, &g_fp4_error);
    }
    // the accumulator is complete; nobody reads the stages any more
    bool ok = k1 > k0;
    if (warp >= 2 && ok) ok = mbar_wait(acc_full, 0, abort_flag, &g_fp4_error);
    __syncthreads();
    const int rows = int(min(uint64_t(BN), g.m - arow));
    if (warp >= 2) {
        fence_after();
#pragma unroll 1
        for (int c = 0; c < rows; c += 16) {
            float v[16];
            tmem_ld16(tmem + (uint32_t(q * 32) << 16) + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) part[(c + i) * kPitch + q * 32 + lane] = ok ? v[i] : 0.f;
        }
        fence_before();
    }
    if (split > 1)
        cluster_sync();
    else
        __syncthreads();
    if (warp >= 2) {
        // rows rank, rank + split, ..: a thread takes four columns of a row from every CTA of the cluster
        const int mine = (rows - int(rank) + split - 1) / split;
        const int es = g.out_bf16 ? 2 : 4;
        const bool vec = g.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(g.out) % (4 * es) == 0;
#pragma unroll 2
        for (int it = threadIdx.x - 64; it < mine * 32; it += 128) {
            const int r = int(rank) + (it >> 5) * split, c = (it & 31) * 4, col = int(tn) * 128 + c;
            float y[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t at = smem_u32(part + r * kPitch + c);
            for (int i = 0; i < split; ++i) {
                float x[4];
                asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                    : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                    : "r"(split > 1 ? map_to_rank(at, uint32_t(i)) : at)
                    : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += x[e];
            }
            float rest;
            const float ra = split_scale(ra_s[r], rest);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = y[e] * ra * rb_s[c + e] * rest;
            const uint64_t off = (arow + r) * uint64_t(g.ldo) + col;
            if (g.out_bf16) {
                uint16_t* o = static_cast<uint16_t*>(g.out) + off;
                const uint32_t lo = pack_bf16x2(y[0], y[1]), hi = pack_bf16x2(y[2], y[3]);
                if (vec && col + 4 <= g.n) {
                    *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
                } else {
                    if (col < g.n) o[0] = uint16_t(lo);
                    if (col + 1 < g.n) o[1] = uint16_t(lo >> 16);
                    if (col + 2 < g.n) o[2] = uint16_t(hi);
                    if (col + 3 < g.n) o[3] = uint16_t(hi >> 16);
                }
            } else {
                float* o = static_cast<float*>(g.out) + off;
                if (vec && col + 4 <= g.n) {
                    *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < g.n) o[e] = y[e];
                }
            }
        }
    }
    if (split > 1)
        cluster_sync();  // the others have read this CTA's part
    else
        __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem));
    }
}

// ---- host side -------------------------------------------------------------
// Codes as bytes: rows of `row_bytes`, boxes of 128 bytes x `box_rows` rows.
int codes_map(CUtensorMap* m, const void* base, uint64_t rows, int row_bytes, int ld, uint32_t box_rows) {
    const uint64_t dims[2] = {uint64_t(row_bytes), rows};
    const uint64_t strides[1] = {uint64_t(ld)};
    const uint32_t box[2] = {128, box_rows};
    return make_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, true);
}
// Scale tiles as rows of 512 bytes, boxes of a stage's tiles.
int scales_map(CUtensorMap* m, const void* base, uint64_t rows, int tiles, uint32_t box_tiles) {
    const uint64_t dims[2] = {128, (rows + 127) / 128 * uint64_t(tiles)};
    const uint64_t strides[1] = {512};
    const uint32_t box[2] = {128, box_tiles};
    return make_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, base, dims, strides, box, false);
}

template <int FORMAT>
int launch_pair(ProductArgs g, const void* a, int lda, const void* b, int ldb, int kb, int sms, cudaStream_t st) {
    using S = Scales<FORMAT>;
    g.grid_m = uint32_t((g.m + 255) / 256);
    g.grid_n = uint32_t((g.n + 255) / 256);
    CUtensorMap tm_a, tm_b, tm_sa, tm_sb, tm_out;
    if (int rc = codes_map(&tm_a, a, g.m, kb, lda, 128)) return rc;
    if (int rc = codes_map(&tm_b, b, uint64_t(g.n), kb, ldb, 128)) return rc;
    if (int rc = scales_map(&tm_sa, g.a_scales, g.m, g.tiles, S::kTiles)) return rc;
    if (int rc = scales_map(&tm_sb, g.b_scales, uint64_t(g.n), g.tiles, S::kTiles)) return rc;
    const int es = g.out_bf16 ? 2 : 4;
    g.tma_out = (reinterpret_cast<uintptr_t>(g.out) | (uint64_t(g.ldo) * es)) % 16 == 0;
    g.n_whole = uint64_t(g.n) * es % 16 == 0;
    if (g.tma_out) {
        const uint64_t dims[2] = {uint64_t(g.n), g.m};
        const uint64_t strides[1] = {uint64_t(g.ldo) * es};
        const uint32_t box[2] = {uint32_t(128 / es), 32};
        if (int rc = make_tiled_map(&tm_out, g.out_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                                    2, g.out, dims, strides, box, true))
            return rc;
    } else {
        tm_out = tm_a;  // not used
    }
    constexpr int smem = kPairStages * (2 * 16384 + 3 * S::kBytes) + kEpiWarps * (4096 + 256) + 256 + 1024;
    auto kern = pair_kernel<FORMAT>;
    GATB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const uint64_t ntiles = uint64_t(g.grid_m) * g.grid_n;
    const unsigned pairs = unsigned(ntiles < uint64_t(sms / 2) ? ntiles : uint64_t(sms / 2));
    kern<<<2 * pairs, kPairThreads, smem, st>>>(tm_a, tm_b, tm_sa, tm_sb, tm_out, g);
    GATB_LAUNCH("fp4_product (pair) kernel");
    return 0;
}

// Parts that the rows kernel splits the reduction into: while all of them run at
// once and each keeps two stages.
int rows_split(uint64_t tiles, int stages_k, uint64_t slots) {
    int split = 1;
    while (split < 8 && tiles * split * 2 <= slots && stages_k >= 4 * split) split *= 2;
    return split;
}

template <int FORMAT, int BN>
int launch_rows(ProductArgs g, const void* a, int lda, const void* b, int ldb, int kb, int sms, cudaStream_t st) {
    using S = Scales<FORMAT>;
    g.grid_m = uint32_t((g.m + BN - 1) / BN);
    g.grid_n = uint32_t((g.n + 127) / 128);
    const uint64_t tiles = uint64_t(g.grid_m) * g.grid_n;
    const int split = rows_split(tiles, g.stages_k, uint64_t(sms) * RowsTile<BN>::kCtas);
    CUtensorMap tm_a, tm_b;
    if (int rc = codes_map(&tm_a, a, g.m, kb, lda, BN)) return rc;
    if (int rc = codes_map(&tm_b, b, uint64_t(g.n), kb, ldb, 128)) return rc;
    constexpr int stages = RowsTile<BN>::kStages * (128 * 128 + BN * 128 + 2 * S::kBytes);
    constexpr int part = BN * 132 * 4;
    static_assert(part <= stages, "the exchange buffer lies over the stages");
    constexpr int smem = stages + 256 + (128 + BN) * 4 + 1024;
    auto kern = rows_kernel<FORMAT, BN>;
    GATB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(tiles * split));
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(split);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    GATB_CUDA(cudaLaunchKernelEx(&cfg, kern, tm_a, tm_b, g, split));
    return 0;
}

template <int FORMAT>
int launch_product(const ProductArgs& g, const void* a, int lda, const void* b, int ldb, int kb, int sms,
                   cudaStream_t st) {
    // Up to 64 rows the rows kernel (64 x 8192 x 2048: both 8.4 us; 33 x 8192 x 8192: 10 us, pairs 16;
    // 48 x 20000 x 1024: 8.6 us, pairs 9.6). Above, whichever these times, fitted to both, give the lead:
    // a pair kernel takes 5.3 us and 0.35 us a stage and wave, a rows kernel 9 us and as much a stage of
    // its part (100 x 1000 x 8192: 9.6 us, pairs 16.3; 100 x 4096 x 1024: 9.3 us, pairs 7.5;
    // 2000 x 2000 x 8192: 47 us, pairs 18.6).
    if (g.m <= 16) return launch_rows<FORMAT, 16>(g, a, lda, b, ldb, kb, sms, st);
    if (g.m <= 32) return launch_rows<FORMAT, 32>(g, a, lda, b, ldb, kb, sms, st);
    if (g.m <= 64) return launch_rows<FORMAT, 64>(g, a, lda, b, ldb, kb, sms, st);
    const uint64_t pair_tiles = (g.m + 255) / 256 * ((uint64_t(g.n) + 255) / 256), pairs = uint64_t(sms) / 2;
    const uint64_t tiles = (g.m + 127) / 128 * ((uint64_t(g.n) + 127) / 128);
    const int split = rows_split(tiles, g.stages_k, uint64_t(sms));
    const double by_pairs = 5.3 + 0.35 * g.stages_k * double((pair_tiles + pairs - 1) / pairs);
    const double by_rows = (split == 1 ? 11.0 : 9.0) +
                           0.35 * ((g.stages_k + split - 1) / split) * double((tiles * split + sms - 1) / sms);
    return by_pairs <= by_rows ? launch_pair<FORMAT>(g, a, lda, b, ldb, kb, sms, st)
                               : launch_rows<FORMAT, 128>(g, a, lda, b, ldb, kb, sms, st);
}

}  // namespace

int fp4_product_launch(int format, uint64_t m, int n, int k, const void* a, int lda, const void* a_scales,
                       const float* a_row, const void* b, int ldb, const void* b_scales, const float* b_row, void* out,
                       int out_dtype, int ldo, cudaStream_t st) {
    if (int rc = fp4_check_format("fp4_product", format)) return rc;
    if (out_dtype != GAT_B200_F32 && out_dtype != GAT_B200_BF16) return fail("fp4_product: bad output dtype");
    if (n < 0 || k <= 0 || k > (1 << 24)) return fail("fp4_product: bad shape");
    if (m > uint64_t(INT32_MAX - 512) || n > INT32_MAX - 512) return fail("fp4_product: too many rows");
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
    ProductArgs g{};
    g.m = m;
    g.n = n;
    g.stages_k = (kb + 127) / 128;
    g.last_mmas = (k - (g.stages_k - 1) * 256 + 63) / 64;
    g.tiles = fp4_tiles(format, k);
    // scale tiles are counted in 32 bits (TMA rows), output tiles as a grid
    if (((m > uint64_t(n) ? m : uint64_t(n)) + 511) / 128 * uint64_t(g.tiles) > uint64_t(INT32_MAX) ||
        (m + 15) / 16 * ((uint64_t(n) + 127) / 128) * 8 > uint64_t(INT32_MAX))
        return fail("fp4_product: tables too large");
    if (int rc = check_device_pointers("fp4_product", {a, a_scales, a_row, b, b_scales, b_row, out})) return rc;
    g.a_scales = static_cast<const uint8_t*>(a_scales);
    g.b_scales = static_cast<const uint8_t*>(b_scales);
    g.a_row = a_row;
    g.b_row = b_row;
    g.out = out;
    g.ldo = ldo;
    g.out_bf16 = out_dtype == GAT_B200_BF16;
    int dev = 0, sms = 0;
    GATB_CUDA(cudaGetDevice(&dev));
    GATB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    return format == GAT_B200_MXFP4 ? launch_product<GAT_B200_MXFP4>(g, a, lda, b, ldb, kb, sms, st)
                                    : launch_product<GAT_B200_NVFP4>(g, a, lda, b, ldb, kb, sms, st);
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
