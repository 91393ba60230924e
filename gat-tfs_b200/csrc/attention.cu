// Masked softmax attention inside the segments of a packed batch (tcgen05/TMA).
//
//   z_ij = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - pos_j|
//   out_i = sum_j softmax_j(z_ij) v_j,   lse_i = log sum_j exp z_ij
// over the keys j of row i's segment that its mask shows. Every mask here
// (segment, causal, prefix) shows a row one interval [lo, hi) of packed keys,
// so a tile of 128 packed rows may span many segments: small graphs share tiles
// and a long document is one run of tiles.
//
// One CTA: TILES tiles of 128 rows of one head, all key blocks of 128 that one
// of their rows sees. Up to dim 64 a CTA has one tile and two CTAs share an SM;
// above, shared memory holds one CTA and it has two tiles. Either way one
// tile's softmax runs beside the other's MMAs. Warps:
//   0     TMA producer: Q once, K and V blocks through rings.
//   1     MMA issuer: S = Q K^T into TMEM; O += P V with P read from TMEM. With
//         one tile P has columns of its own and the next S is computed while
//         the softmax is at work; with two, P overlays S.
//   2-3   masked blocks only: take non-finite values of V out of shared memory
//         (a weight of zero times Inf or NaN is NaN) and note their keys; rows
//         that do see such a key add it themselves.
//   4 ..  softmax, a row per thread (no shuffles), four warps a tile; eight, two
//         threads a row, where the weights need no common maximum (see below).
// The running maximum is only moved when it grows by more than 24 (weights up
// to 2^24, far inside FP32 and BF16's range), so O is seldom rescaled.
// MMAs of a CTA run in order, so where P overlays S, S's barrier also says that
// the tile's last P V is done and O is at rest. P is rounded to BF16 (the tensor cores' input
// type); out is divided by the FP32 sum of the rounded weights, so a row is an
// average with its own weights, and lse takes the sum of the unrounded ones.
// The exponentials bound it (16 a clock and SM; a 128 x 128 block of dim 128
// takes the tensor cores as long as its exponentials): the cap's tanh is a
// polynomial on the FMA pipe wherever a block's scores stay below 0.6 cap. A
// row's largest capped score lies within +-cap (of the bias of its nearest key),
// so up to a cap of 55 the weights are taken relative to cap / 4 (and that bias)
// instead of the running maximum. The largest weight of a row is then 2^-100 ..
// 2^60, so that in the lowest of rows a key counts until it is 2^-26 of the
// largest one (what a bias pushes further down is flushed to zero at 2^-126, less
// than 2e-6 of the row's sum) and values from 2^-26 to 2^40 keep their products
// among FP32's ordinary numbers. No pass for the maximum, no rescaling, 32 columns
// at a time flow from S to P and two threads share a row. (With a maximum to agree on, two
// threads a row were slower than one: 8192 x 32 x 128 causal, 320 us and 359 us.)
#include <cuda.h>

#include "attention.cuh"
#include "tc.cuh"

namespace gatb {

__device__ unsigned g_attention_error = 0;

int make_tiled_map(CUtensorMap* m, int type, int rank, const void* base, const uint64_t* dims, const uint64_t* strides,
                   const uint32_t* box, bool swizzle);

namespace {

using namespace tc;

constexpr int kRows = 128;  // rows of a tile, keys of a block

struct AttnArgs {
    uint64_t n_q, n_k;
    int heads, group, dim, nseg, mask;
    const uint64_t* q_row;
    const uint64_t* k_row;
    const uint64_t* prefix;
    const float* slopes;
    const uint16_t* v;
    int ldv;
    float zscale;    // without a cap: scale * log2 e; with one: scale / cap
    float zcap;      // cap * log2 e
    float small;     // raw scores up to which the tanh's long polynomial holds (a third of it: the short one)
    float tanh[5];   // coefficients of s, s^3 .. in zcap tanh(scale / cap * s)
    float tanh3[3];
    uint16_t* out;
    int ldo;
    float* lse;
};

__device__ __forceinline__ void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc) {
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, 1;" ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc),
                 "r"(idesc)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// 32 lanes x 32 columns: the load, and the wait after which r may be read.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32_wait(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                   "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]),
                   "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]),
                   "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]),
                   "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Segments of the 32 consecutive rows first + lane (a converged warp): the
// first row's by a 32-way search, the others' from the row pointers behind it.
__device__ __forceinline__ int segment_of_lane(const uint64_t* row, int nseg, uint64_t first, int lane) {
    int a = 0, b = nseg;
    while (b - a > 1) {
        const int step = (b - a + 31) / 32, at = a + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, at < b && row[at] <= first);
        const int n = max(1, __popc(le));
        a += (n - 1) * step;
        b = min(b, a + step);
    }
    int s = a;
    for (int next = a + 1; next < nseg; next += 32) {
        // rows at and past o belong to segment next + lane or a later one
        const int at = next + lane;
        const int o = at < nseg ? int(min(uint64_t(32), row[at] > first ? row[at] - first : 0)) : 32;
        const unsigned live = __ballot_sync(0xffffffffu, o < 32);
        for (int l = 0; l < __popc(live); ++l)
            if (__shfl_sync(0xffffffffu, o, l) <= lane) ++s;
        if (live != 0xffffffffu) break;
    }
    return min(s, nseg - 1);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Sums of weights and of their BF16 roundings.
struct WeightSum {
    f32x2 w[2], r[2];
    __device__ __forceinline__ WeightSum() { w[0] = w[1] = r[0] = r[1] = pack2(0.f, 0.f); }
    __device__ __forceinline__ void add(int i, float p0, float p1, uint32_t rounded) {
        w[i & 1] = add2(w[i & 1], pack2(p0, p1));
        r[i & 1] = add2(r[i & 1], pack2(bf16lo(rounded), bf16hi(rounded)));
    }
    __device__ __forceinline__ void into(float& sum, float& sum_rounded) const {
        float a, b;
        unpack2(add2(w[0], w[1]), a, b);
        sum += a + b;
        unpack2(add2(r[0], r[1]), a, b);
        sum_rounded += a + b;
    }
};

// Bits of the columns [b, e) of 32.
__device__ __forceinline__ uint32_t visible(int b, int e) {
    b = min(max(b, 0), 32);
    e = min(max(e, 0), 32);
    return e > b ? (e == 32 ? 0u : (1u << e)) - (1u << b) : 0u;
}

// Growth of the maximum (log2) up to which the reference stays.
constexpr float kGrow = 24.f;
// Largest cap * log2 e whose weights are taken relative to a quarter of it.
constexpr float kFixedCap = 80.f;
// The polynomials' coefficients take scale / cap into themselves, in powers up
// to the ninth: used for scale / cap up to kTanhScale and products q.k whose
// powers stay FP32 numbers; other scores go one by one through capped_score().
constexpr double kTanhScale = 8192.0;
constexpr float kTanhProducts = 4915.f;

// DP: dim rounded up to 64 or 128. CAP / BIAS: scores go through the tanh / get the distance bias.
// FIXED: weights relative to a quarter of the cap (capped scores).
// TMEM, one tile: S at 0, P at 128, O at 192; two: S and P of tile t at 128 t, O at 256 + 128 t.
template <int DP, bool FIXED>
struct Shape {
    static constexpr int kTiles = DP == 64 ? 1 : 2;
    static constexpr int kHalves = FIXED ? 2 : 1;        // softmax threads a row
    static constexpr int kThreads = 128 + 128 * kTiles * kHalves;
    static constexpr int kCtas = DP == 64 ? 2 : 1;       // per SM
    // registers after setmaxnreg, inside the launch's kCtas * kThreads * (65536 / (kCtas * kThreads), whole eights)
    static constexpr int kRoleRegs = kTiles * kHalves == 1 || FIXED ? 56 : 72;
    static constexpr int kSoftmaxRegs = FIXED ? (DP == 64 ? 88 : 104) : (DP == 64 ? 200 : 216);
    static constexpr int kLaunchRegs = 65536 / (kCtas * kThreads) / 8 * 8;
    static_assert(128 * kRoleRegs + 128 * kTiles * kHalves * kSoftmaxRegs <= kThreads * kLaunchRegs, "register split");
    static constexpr int kTmem = DP == 64 ? 256 : 512;
    static constexpr int kTile = kRows * DP * 2;         // bytes of a Q tile, a K block, a V block
    static constexpr int kStages = 2;                    // K and V stages
    static constexpr int kSmem = (kTiles + 2 * kStages) * kTile + (FIXED ? kTiles * 4 * kRows * 4 : 0) + 1024 + 512;
};
template <int DP, bool CAP, bool BIAS, bool FIXED>
__global__ void __launch_bounds__(Shape<DP, FIXED>::kThreads, Shape<DP, FIXED>::kCtas)
    attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnArgs g) {
    constexpr int kTiles = Shape<DP, FIXED>::kTiles, kHalves = Shape<DP, FIXED>::kHalves, kTile = Shape<DP, FIXED>::kTile, kSt = Shape<DP, FIXED>::kStages;
    static_assert(!FIXED || CAP, "only capped scores are bounded");
    constexpr bool kOwnP = kTiles == 1;
    // P's columns for the block's keys 64 and up start kPHalf behind the others: where P overlays S, each
    // half of P lies in its own half of S
    constexpr uint32_t kP = kOwnP ? 128 : 0, kPHalf = kOwnP ? 32 : 64, kO = kOwnP ? 192 : 256;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;
    uint8_t* k_s = q_s + kTiles * kTile;
    uint8_t* v_s = k_s + kSt * kTile;
    float* sums = reinterpret_cast<float*>(v_s + kSt * kTile);  // FIXED: [kTiles][4][kRows]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sums + (FIXED ? kTiles * 4 * kRows : 0));
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;
    uint64_t* k_empty = k_full + kSt;
    uint64_t* v_full = k_empty + kSt;
    uint64_t* v_ready = v_full + kSt;
    uint64_t* v_empty = v_ready + kSt;
    uint64_t* s_full = v_empty + kSt;    // [kTiles]
    uint64_t* p_full = s_full + kTiles;  // [kTiles]
    uint64_t* o_full = p_full + kTiles;  // [kTiles]
    uint64_t* s_read = o_full + kTiles;  // own P: S is in registers
    uint64_t* pv_done = s_read + 1;      // own P: P and O are at rest
    uint64_t* pairs = pv_done + 1;       // FIXED: [kTiles][4], the two warps of the same rows
    uint32_t* bad = reinterpret_cast<uint32_t*>(pairs + 4 * kTiles);  // [kSt][4] keys of the block with non-finite values
    unsigned* range = bad + 4 * kSt;  // per tile: smallest lo, largest hi, largest lo, smallest hi
    uint32_t* tmem_holder = range + 4 * kTiles;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = int(blockIdx.x % unsigned(g.heads)), kv_head = head / g.group;
    // later rows see more keys under a causal mask: the longest tiles of all heads start first
    const uint64_t row0 = uint64_t((gridDim.x - 1 - blockIdx.x) / unsigned(g.heads)) * (kTiles * kRows);
    const int boxes = g.dim > 64 ? 2 : 1;
    const uint32_t bytes = uint32_t(boxes) * kRows * 128;  // of a tile or block as TMA counts them
    const int q_tiles = row0 + kRows < g.n_q ? kTiles : 1;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < kSt; ++s) {
            mbar_init(k_full + s, 1);
            mbar_init(k_empty + s, 1);
            mbar_init(v_full + s, 1);
            mbar_init(v_ready + s, 2);
            mbar_init(v_empty + s, 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            mbar_init(s_full + t, 1);
            mbar_init(p_full + t, 4 * kHalves);
            for (int i = 0; i < 4; ++i) mbar_init(pairs + 4 * t + i, 2);
            mbar_init(o_full + t, 1);
            range[4 * t] = 0xffffffffu;
            range[4 * t + 1] = 0;
            range[4 * t + 2] = 0;
            range[4 * t + 3] = 0xffffffffu;
        }
        mbar_init(s_read, 4 * kHalves);
        mbar_init(pv_done, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
        mbar_expect_tx(q_full, bytes * q_tiles);
        for (int t = 0; t < q_tiles; ++t)
            for (int b = 0; b < boxes; ++b)
                tma_load_3d(q_s + t * kTile + b * (kRows * 128), &tm_q, q_full, b * 64, head, int(row0) + t * kRows);
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"(Shape<DP, FIXED>::kTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }

    // The row's key interval (softmax threads), its position and the tile's ranges.
    const int half = kHalves == 2 ? ((warp - 4) >> 2) & 1 : 0;
    const int tile = kTiles == 2 && warp >= 4 + 4 * kHalves ? 1 : 0;
    const int r = (warp & 3) * 32 + lane;
    const uint64_t row = row0 + uint64_t(tile) * kRows + r;
    int lo = 0, hi = -1, pos = 0;  // hi -1: no row, or one outside the segments
    if (warp >= 4) {
        const int s = segment_of_lane(g.q_row, g.nseg, row - lane, lane);
        // row pointers are taken as given but kept inside the tables
        const uint64_t q0 = g.q_row[s], q1 = g.q_row[s + 1];
        if (row < g.n_q && row >= q0 && row < q1) {
            const uint64_t ks = min(g.k_row[s], g.n_k), ke = max(ks, min(g.k_row[s + 1], g.n_k));
            const int64_t at = int64_t(row - q0) + int64_t(ke - ks) - int64_t(q1 - q0);
            lo = int(ks);
            hi = int(ke);
            if (g.mask != GAT_B200_MASK_FULL) {
                int64_t seen = at + 1;
                if (g.mask == GAT_B200_MASK_PREFIX) seen = max(seen, int64_t(min(g.prefix[s], g.n_k)));
                seen = max(int64_t(0), min(seen, int64_t(ke - ks)));
                hi = lo + int(seen);
            }
            pos = int(max(int64_t(-INT32_MAX), min(at, int64_t(INT32_MAX))));
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_holder;
    if (warp >= 4) {
        const bool some = hi > lo;
        const unsigned min_lo = __reduce_min_sync(0xffffffffu, some ? unsigned(lo) : 0xffffffffu);
        const unsigned max_hi = __reduce_max_sync(0xffffffffu, some ? unsigned(hi) : 0u);
        const unsigned max_lo = __reduce_max_sync(0xffffffffu, some ? unsigned(lo) : 0u);
        const unsigned min_hi = __reduce_min_sync(0xffffffffu, some ? unsigned(hi) : 0xffffffffu);
        if (lane == 0) {
            atomicMin(range + 4 * tile, min_lo);
            atomicMax(range + 4 * tile + 1, max_hi);
            atomicMax(range + 4 * tile + 2, max_lo);
            atomicMin(range + 4 * tile + 3, min_hi);
        }
    }
    __syncthreads();
    // key blocks [from, to) that tile t works on; blocks inside [max_lo, min_hi)
    // are seen whole by every row that sees anything
    unsigned first_key = range[0], end_key = range[1], max_lo = range[2], min_hi = range[3];
    if constexpr (kTiles == 2) {
        first_key = min(first_key, range[4]);
        end_key = max(end_key, range[5]);
        max_lo = max(max_lo, range[6]);
        min_hi = min(min_hi, range[7]);
    }
    const int blocks = end_key > first_key ? int((end_key - first_key + kRows - 1) / kRows) : 0;
    int from[kTiles], to[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        const bool any = range[4 * t + 1] > range[4 * t];
        from[t] = any ? int((range[4 * t] - first_key) / kRows) : 0;
        to[t] = any ? int((range[4 * t + 1] - first_key + kRows - 1) / kRows) : 0;
    }
    const int last_tile = to[kTiles - 1] > 0 ? kTiles - 1 : 0;
    const int ksteps = (g.dim + 15) / 16;
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape<DP, FIXED>::kRoleRegs));
    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int j = 0;
            for (; j < blocks && ok; ++j) {
                const int s = j % kSt;
                const uint32_t ph = uint32_t(j / kSt) & 1u;
                const int key = int(first_key) + j * kRows;
                if (!mbar_wait(k_empty + s, ph ^ 1u, abort_flag, &g_attention_error)) { ok = false; break; }
                mbar_expect_tx(k_full + s, bytes);
                for (int b = 0; b < boxes; ++b)
                    tma_load_3d(k_s + s * kTile + b * (kRows * 128), &tm_k, k_full + s, b * 64, kv_head, key);
                if (!mbar_wait(v_empty + s, ph ^ 1u, abort_flag, &g_attention_error)) {
                    mbar_wait(k_full + s, ph, abort_flag, &g_attention_error);
                    ok = false;
                    break;
                }
                mbar_expect_tx(v_full + s, bytes);
                for (int b = 0; b < boxes; ++b)
                    tma_load_3d(v_s + s * kTile + b * (kRows * 128), &tm_v, v_full + s, b * 64, kv_head, key);
            }
            // the loads still in flight land before the CTA ends
            mbar_wait(q_full, 0, abort_flag, &g_attention_error);
            for (int i = j > kSt ? j - kSt : 0; i < j; ++i) {
                mbar_wait(k_full + i % kSt, uint32_t(i / kSt) & 1u, abort_flag, &g_attention_error);
                mbar_wait(v_full + i % kSt, uint32_t(i / kSt) & 1u, abort_flag, &g_attention_error);
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc_s = idesc_bf16(kRows, kRows, 0, 0);
        const uint32_t idesc_o = idesc_bf16(kRows, ksteps * 16, 0, 1);
        bool ok = mbar_wait_warp(q_full, 0, abort_flag, &g_attention_error);
        auto scores = [&](int t, int s) {
            const uint64_t qdesc = desc_sw128(smem_u32(q_s + t * kTile), 16, 1024);
            const uint64_t kdesc = desc_sw128(smem_u32(k_s + s * kTile), 16, 1024);
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                if (ks >= ksteps) break;
                const uint32_t off = (ks >> 2) * (kRows * 128 / 16) + (ks & 3) * 2;
                mma_bf16(tmem + 128 * t, qdesc + off, kdesc + off, idesc_s, ks > 0);
            }
            mma_commit(s_full + t);
        };
        auto values = [&](int t, int s) {
            const uint64_t vdesc = desc_sw128(smem_u32(v_s + s * kTile), kRows * 128, 1024);
#pragma unroll
            for (int ks = 0; ks < kRows / 16; ++ks)
                mma_bf16_ts(tmem + kO + DP * t, tmem + kP + 128 * t + (ks >> 2) * kPHalf + (ks & 3) * 8, vdesc + ks * 128, idesc_o);
        };
        if constexpr (kOwnP) {
            for (int j = -1; j < blocks && ok; ++j) {
                if (j + 1 < blocks) {
                    const int s = (j + 1) % kSt;
                    ok = mbar_wait_warp(k_full + s, uint32_t((j + 1) / kSt) & 1u, abort_flag, &g_attention_error) &&
                         (j < 0 || mbar_wait_warp(s_read, uint32_t(j) & 1u, abort_flag, &g_attention_error));
                    if (!ok) break;
                    fence_after();
                    if (elect_one()) {
                        scores(0, s);
                        mma_commit(k_empty + s);
                    }
                    __syncwarp();
                }
                if (j >= 0) {
                    const int s = j % kSt;
                    ok = mbar_wait_warp(v_ready + s, uint32_t(j / kSt) & 1u, abort_flag, &g_attention_error) &&
                         mbar_wait_warp(p_full, uint32_t(j) & 1u, abort_flag, &g_attention_error);
                    if (!ok) break;
                    fence_after();
                    if (elect_one()) {
                        values(0, s);
                        mma_commit(pv_done);
                        mma_commit(v_empty + s);
                        if (j + 1 == blocks) mma_commit(o_full);
                    }
                    __syncwarp();
                }
            }
        } else {
            uint32_t used[2] = {0, 0};  // blocks of tile t issued so far
            for (int j = -1; j < blocks && ok; ++j) {
                const int s = j % kSt, sn = (j + 1) % kSt;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (t > last_tile || !ok) break;
                    const bool now = j >= from[t] && j < to[t], next = j + 1 >= from[t] && j + 1 < to[t];
                    if (j >= 0) {
                        if (t == 0) ok = mbar_wait_warp(v_ready + s, uint32_t(j / kSt) & 1u, abort_flag, &g_attention_error);
                        if (ok && now) ok = mbar_wait_warp(p_full + t, used[t]++ & 1u, abort_flag, &g_attention_error);
                        if (!ok) break;
                        fence_after();
                        if (elect_one()) {
                            if (now) {
                                values(t, s);
                                if (j + 1 == to[t]) mma_commit(o_full + t);
                            }
                            if (t == last_tile) mma_commit(v_empty + s);
                        }
                        __syncwarp();
                    }
                    if (j + 1 < blocks) {
                        if (t == 0) ok = mbar_wait_warp(k_full + sn, uint32_t((j + 1) / kSt) & 1u, abort_flag, &g_attention_error);
                        if (!ok) break;
                        fence_after();
                        if (elect_one()) {
                            if (next) scores(t, sn);
                            if (t == last_tile) mma_commit(k_empty + sn);
                        }
                        __syncwarp();
                    }
                }
            }
        }
        // whatever was issued has finished before the CTA ends (v_empty of the last block)
        if (ok && blocks > 0)
            mbar_wait_warp(v_empty + (blocks - 1) % kSt, uint32_t((blocks - 1) / kSt) & 1u, abort_flag, &g_attention_error);
    } else if (warp < 4) {
        // ---- V of masked blocks: non-finite values out, their keys noted ----
        for (int j = 0; j < blocks; ++j) {
            const int s = j % kSt;
            if (!mbar_wait_warp(v_full + s, uint32_t(j / kSt) & 1u, abort_flag, &g_attention_error)) break;
            const unsigned key = first_key + unsigned(j) * kRows;
            if (key < max_lo || key + kRows > min_hi) {
                uint32_t* words = bad + 4 * s;
                const int half = warp - 2;  // 64 keys a warp
                if (lane < 2) words[2 * half + lane] = 0;
                __syncwarp();
                for (int b = 0; b < boxes; ++b) {
                    uint8_t* base = v_s + s * kTile + b * (kRows * 128) + half * 64 * 128;
#pragma unroll 2
                    for (int i = lane; i < 64 * 8; i += 32) {
                        uint4 w = *reinterpret_cast<const uint4*>(base + i * 16);
                        auto hit = [](uint32_t x) {
                            return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
                        };
                        if (hit(w.x) | hit(w.y) | hit(w.z) | hit(w.w)) {
                            auto clean = [](uint32_t x) {
                                if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
                                if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
                                return x;
                            };
                            *reinterpret_cast<uint4*>(base + i * 16) =
                                make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
                            const int k = half * 64 + (i >> 3);
                            atomicOr(words + (k >> 5), 1u << (k & 31));
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(v_ready + s);
        }
    }
    } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape<DP, FIXED>::kSoftmaxRegs));
    const int my_from = kTiles == 2 && tile ? from[kTiles - 1] : from[0], my_to = kTiles == 2 && tile ? to[kTiles - 1] : to[0];
    if (my_to > 0) {
        // ---- softmax of one tile: thread = row (FIXED: half the columns of a row, of S, P and O) ----
        constexpr int kOCols = DP / kHalves;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t s_t = tmem + lanes + 128 * tile, p_t = s_t + kP, o_t = tmem + lanes + kO + DP * tile + kOCols * half;
        const float nslope = BIAS ? -g.slopes[head] * kLog2e : 0.f;
        {
            uint32_t z[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
            for (int c = 0; c < kOCols; c += 32) tmem_st32(o_t + c, z);
            tmem_wait_st();
        }
        f32x2 tk[5] = {}, tk3[3] = {};  // the tanh's polynomials
        if constexpr (CAP) {
#pragma unroll
            for (int i = 0; i < 5; ++i) tk[i] = pack2(g.tanh[i], g.tanh[i]);
#pragma unroll
            for (int i = 0; i < 3; ++i) tk3[i] = FIXED ? pair_of(g.tanh3[i]) : 0;
        }
        // the reference maximum (log2 units), the sums of the weights and of the rounded weights
        float m = FIXED ? 0.25f * g.zcap : -INFINITY, l = 0.f, lr = 0.f;
        // FIXED with a bias: the distance of the row's nearest key (farthest with a negative slope), whose
        // bias the weights are relative to
        const int past = pos - (hi - lo - 1);  // behind the last key that it sees
        const float near = !FIXED || !BIAS ? 0.f
                           : nslope <= 0.f ? float(max(0, max(-pos, past)))
                                           : fmaxf(fabsf(float(pos)), fabsf(float(past)));
        // the intervals of the warp's rows that see anything: smallest and largest begin and end
        const bool some = hi > lo;
        const int lo_min = __reduce_min_sync(0xffffffffu, some ? lo : INT32_MAX);
        const int lo_max = __reduce_max_sync(0xffffffffu, some ? lo : 0);
        const int hi_min = __reduce_min_sync(0xffffffffu, some ? hi : INT32_MAX);
        const int hi_max = __reduce_max_sync(0xffffffffu, some ? hi : 0);
        uint32_t met = 0;
        // the other warp of the same rows has come as far, and its shared and tensor memory can be read
        auto meet_pair = [&] {
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pairs + 4 * tile + (warp & 3));
            const bool met_it = mbar_wait_warp(pairs + 4 * tile + (warp & 3), met++ & 1u, abort_flag, &g_attention_error);
            fence_after();
            return met_it;
        };
        bool ok = true;
        uint32_t use = 0;
        for (int j = my_from; j < my_to; ++j, ++use) {
            if (!mbar_wait_warp(s_full + tile, use & 1u, abort_flag, &g_attention_error)) { ok = false; break; }
            fence_after();
            const int key = int(first_key) + j * kRows;
            const int jl = lo - key, jh = hi - key;  // visible columns [jl, jh)
            // 32-column words of the block: 0 nobody sees, 1 seen in part, 2 seen whole
            auto seen = [&](int w) {
                const int a = key + 32 * w, b = a + 32;
                return b <= lo_min || a >= hi_max ? 0 : a >= lo_max && b <= hi_min ? 2 : 1;
            };
            // S may be overwritten once it is in registers; P and O may be touched once the last P V is done
            auto s_is_read = [&] {
                if constexpr (kOwnP) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_read);
                }
            };
            auto p_is_free = [&] {
                if (!kOwnP || use == 0) return true;
                const bool done = mbar_wait_warp(pv_done, (use - 1) & 1u, abort_flag, &g_attention_error);
                fence_after();
                return done;
            };
            if constexpr (FIXED) {
                WeightSum sum;
                if (!p_is_free()) { ok = false; break; }
                float x2[2][32];
                tmem_ld32_start(s_t + 64 * half, x2[0]);
                tmem_ld32_start(s_t + 64 * half + 32, x2[1]);
                tmem_ld32_wait(x2[0]);
                tmem_ld32_wait(x2[1]);
                s_is_read();
                float top = 0.f, top2 = 0.f;
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    top = max3(top, fabsf(x2[0][c]), fabsf(x2[0][c + 1]));
                    top2 = max3(top2, fabsf(x2[1][c]), fabsf(x2[1][c + 1]));
                }
                top = fmaxf(top, top2);
                const int degree = __all_sync(0xffffffffu, top <= g.small * (1.f / 3.f)) ? 3
                                   : __all_sync(0xffffffffu, top <= g.small)      ? 5
                                                                                  : 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int w = 2 * half + i;
                    float* x = x2[i];
                    uint32_t p[16];
                    const int sw = seen(w);
                    if (sw == 0) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) p[c] = 0;
                        tmem_st16(p_t + kPHalf * half + 16 * i, p);
                        continue;
                    }
                    const float rel = float(pos + jl - 32 * w);  // distance of column c: |rel - c|
                    // all columns before the rows: the last one's bias and, per column, what it has more (both
                    // of one sign, so that a near key does not carry the rounding of a far one's bias)
                    const bool before = BIAS && nslope <= 0.f && __all_sync(0xffffffffu, rel >= 31.f);
                    const float off = before ? fmaf(nslope, rel - 31.f - near, -m) : -m;
                    const f32x2 nref = pack2(off, off);
                    if (degree == 3) {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const f32x2 t = pack2(x[c], x[c + 1]), u = mul2(t, t);
                            const f32x2 k = fma2(fma2(tk3[2], u, tk3[1]), u, tk3[0]);
                            unpack2(fma2(k, t, nref), x[c], x[c + 1]);
                        }
                    } else if (degree == 5) {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const f32x2 t = pack2(x[c], x[c + 1]), u = mul2(t, t);
                            f32x2 k = fma2(tk[4], u, tk[3]);
                            k = fma2(k, u, tk[2]);
                            k = fma2(k, u, tk[1]);
                            k = fma2(k, u, tk[0]);
                            unpack2(fma2(k, t, nref), x[c], x[c + 1]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[c] = capped_score(x[c] * g.zscale, g.zcap) + off;
                    }
                    if (before) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[c] = fmaf(float(31 - c), nslope, x[c]);
                    } else if (BIAS) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[c] = fmaf(nslope, fabsf(rel - float(c)) - near, x[c]);
                    }
                    if (sw == 1) {
                        const uint32_t bits = visible(jl - 32 * w, jh - 32 * w);
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[c] = bits & (1u << c) ? x[c] : -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float p0 = ex2(x[c]), p1 = ex2(x[c + 1]);
                        p[c / 2] = pack_bf16x2(p0, p1);
                        sum.add(c >> 1, p0, p1, p[c / 2]);
                    }
                    tmem_st16(p_t + kPHalf * half + 16 * i, p);
                }
                sum.into(l, lr);
            } else {
            float z[kRows];
#pragma unroll
            for (int w = 0; w < 4; ++w) tmem_ld32_start(s_t + 32 * w, z + 32 * w);
#pragma unroll
            for (int w = 0; w < 4; ++w) tmem_ld32_wait(z + 32 * w);
            s_is_read();
            const bool whole = key >= lo_max && key + kRows <= hi_min;
            if constexpr (CAP) {
                float top = fabsf(z[0]);
#pragma unroll
                for (int c = 1; c + 1 < kRows; c += 2) top = max3(top, fabsf(z[c]), fabsf(z[c + 1]));
                top = fmaxf(top, fabsf(z[kRows - 1]));
                if (__all_sync(0xffffffffu, top <= g.small)) {
#pragma unroll
                    for (int c = 0; c < kRows; c += 2) {
                        const f32x2 t = pack2(z[c], z[c + 1]), u = mul2(t, t);
                        f32x2 p = fma2(tk[4], u, tk[3]);
                        p = fma2(p, u, tk[2]);
                        p = fma2(p, u, tk[1]);
                        p = fma2(p, u, tk[0]);
                        unpack2(mul2(p, t), z[c], z[c + 1]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kRows; ++c) z[c] = capped_score(z[c] * g.zscale, g.zcap);
                }
            }
            if constexpr (BIAS) {
                const float rel = float(pos + jl);  // distance of column c: |rel - c|
                // (with a cap as well there are no registers to spare for the shorter form)
                if (!CAP && __all_sync(0xffffffffu, rel >= float(kRows - 1))) {
                    // as above: the last column's bias and what the others have more
                    const float base = nslope * (rel - float(kRows - 1));
#pragma unroll
                    for (int c = 0; c < kRows; ++c) {
                        const float e = fmaf(float(kRows - 1 - c), nslope, base);
                        z[c] = fmaf(z[c], g.zscale, e);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kRows; ++c) {
                        if constexpr (!CAP) z[c] *= g.zscale;
                        z[c] = fmaf(nslope, fabsf(rel - float(c)), z[c]);
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t bits = visible(jl - 32 * w, jh - 32 * w);  // bit c: column 32 w + c is visible
#pragma unroll
                    for (int c = 0; c < 32; ++c) z[32 * w + c] = bits & (1u << c) ? z[32 * w + c] : -INFINITY;
                }
            }
            float mb = z[0], mb2 = z[1];
#pragma unroll
            for (int c = 2; c + 3 < kRows; c += 4) {
                mb = max3(mb, z[c], z[c + 1]);
                mb2 = max3(mb2, z[c + 2], z[c + 3]);
            }
            mb = max3(mb, z[kRows - 2], z[kRows - 1]);
            mb = fmaxf(mb, mb2);
            if constexpr (!CAP && !BIAS) mb *= g.zscale;
            if (!p_is_free()) { ok = false; break; }
            if (m == -INFINITY) m = mb;
            const bool grow = mb > m + kGrow;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2(m - mb) : 1.f;
                if (grow) m = mb;
                l *= f;
                lr *= f;
#pragma unroll 1
                for (int c = 0; c < DP; c += 32) {
                    float o[32];
                    tmem_ld32(o_t + c, o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f;
                    tmem_st32(o_t + c, reinterpret_cast<const uint32_t*>(o));
                }
                tmem_wait_st();
            }
            const float ref = m == -INFINITY ? 0.f : m;
            const f32x2 nref = pack2(-ref, -ref), zs = pack2(g.zscale, g.zscale);
            uint32_t p[kRows / 2];
            WeightSum sum;
#pragma unroll
            for (int c = 0; c < kRows; c += 2) {
                const f32x2 s2 = pack2(z[c], z[c + 1]);
                float p0, p1;
                unpack2(CAP || BIAS ? add2(s2, nref) : fma2(s2, zs, nref), p0, p1);
                p0 = ex2(p0);
                p1 = ex2(p1);
                p[c / 2] = pack_bf16x2(p0, p1);
                sum.add(c >> 1, p0, p1, p[c / 2]);
            }
            sum.into(l, lr);
            tmem_st32(p_t, p);
            tmem_st32(p_t + kPHalf, p + 32);
            }
            if (unsigned(key) < max_lo || unsigned(key) + kRows > min_hi) {
                // keys with non-finite values that this row sees: their weights times those values
                const int s = j % kSt;
                if (!mbar_wait_warp(v_ready + s, uint32_t(j / kSt) & 1u, abort_flag, &g_attention_error)) { ok = false; break; }
                const bool any_bad = bad[4 * s] | bad[4 * s + 1] | bad[4 * s + 2] | bad[4 * s + 3];
                if (any_bad) {  // the same for both warps of a row
                    tmem_wait_st();
                    if (kHalves == 2 && !meet_pair()) { ok = false; break; }  // both halves' weights are in P
                }
#pragma unroll 1
                for (int w = any_bad ? 0 : 4; w < 4; ++w) {
                    uint32_t bits = bad[4 * s + w];
                    while (bits) {  // the same for the whole warp
                        const int c = w * 32 + __ffs(bits) - 1;
                        bits &= bits - 1;
                        uint32_t pw;
                        asm volatile(
                            "tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
                            : "=r"(pw)
                            : "r"(p_t + (c >> 6) * kPHalf + (c & 63) / 2)
                            : "memory");
                        const float pc = (c & 1) ? bf16hi(pw) : bf16lo(pw);
                        const bool mine = c >= jl && c < jh;
                        const uint16_t* vr = g.v + (uint64_t(key) + c) * uint64_t(g.ldv) + uint64_t(kv_head) * g.dim;
#pragma unroll 1
                        for (int x = 0; x < kOCols; x += 8) {
                            float o[8];
                            tmem_ld8(o_t + x, o);
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (mine && kOCols * half + x + i < g.dim) {
                                    const uint32_t e = vr[kOCols * half + x + i];
                                    if ((e & 0x7f80u) == 0x7f80u) o[i] += pc * bf16lo(e);
                                }
                            const uint32_t* ou = reinterpret_cast<const uint32_t*>(o);
                            asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(
                                             o_t + x),
                                         "r"(ou[0]), "r"(ou[1]), "r"(ou[2]), "r"(ou[3]), "r"(ou[4]), "r"(ou[5]),
                                         "r"(ou[6]), "r"(ou[7])
                                         : "memory");
                        }
                        tmem_wait_st();  // the next such key reads the same columns
                    }
                }
            }
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + tile);
        }
        if (ok && mbar_wait_warp(o_full + tile, 0, abort_flag, &g_attention_error)) {
            fence_after();
            if constexpr (kHalves == 2) {
                float* s2 = sums + tile * 4 * kRows;
                s2[half * kRows + r] = l;
                s2[(2 + half) * kRows + r] = lr;
                meet_pair();
                l = s2[r] + s2[kRows + r];
                lr = s2[2 * kRows + r] + s2[3 * kRows + r];
            }
            const float inv = hi > lo ? 1.f / lr : 0.f;
            const bool live = hi >= 0;
            uint16_t* orow = g.out + row * uint64_t(g.ldo) + uint64_t(head) * g.dim + kOCols * half;
#pragma unroll 1
            for (int c = 0; c < kOCols; c += 32) {
                float o[32];
                tmem_ld32(o_t + c, o);
                if (live) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        if (kOCols * half + c + i >= g.dim) break;
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = hi > lo ? pack_bf16x2(o[i + 2 * e] * inv, o[i + 2 * e + 1] * inv) : 0u;
                        *reinterpret_cast<uint4*>(orow + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
            }
            if (live && g.lse && half == 0) g.lse[row * g.heads + head] = hi > lo ? ((FIXED && BIAS ? fmaf(nslope, near, m) : m) + log2f(l)) * kLn2 : -INFINITY;
        }
    }
    if (my_to == 0 && hi >= 0 && half == 0) {  // every row of the tile sees nothing
        uint16_t* orow = g.out + row * uint64_t(g.ldo) + uint64_t(head) * g.dim;
        for (int c = 0; c < g.dim; c += 8) *reinterpret_cast<uint4*>(orow + c) = make_uint4(0, 0, 0, 0);
        if (g.lse) g.lse[row * g.heads + head] = -INFINITY;
    }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape<DP, FIXED>::kTmem));
    }
}

int heads_map(CUtensorMap* m, const void* base, int dim, int heads, uint64_t rows, int ld) {
    const uint64_t dims[3] = {uint64_t(dim), uint64_t(heads), rows};
    const uint64_t strides[2] = {uint64_t(dim) * 2, uint64_t(ld) * 2};
    const uint32_t box[3] = {64, 1, kRows};
    return make_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, true);
}

template <int DP, bool CAP, bool BIAS, bool FIXED>
int launch(const AttnArgs& g, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
    constexpr int smem = Shape<DP, FIXED>::kSmem, rows = Shape<DP, FIXED>::kTiles * kRows;
    auto kern = attention_kernel<DP, CAP, BIAS, FIXED>;
    GATB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const uint64_t grid = (g.n_q + rows - 1) / rows * uint64_t(g.heads);
    if (grid > uint64_t(INT32_MAX)) return fail("masked_attention: too many rows times heads");
    kern<<<unsigned(grid), Shape<DP, FIXED>::kThreads, smem, st>>>(q, k, v, g);
    GATB_LAUNCH("masked_attention kernel");
    return 0;
}
template <int DP>
int launch(const AttnArgs& g, bool cap, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
           cudaStream_t st) {
    if (cap && g.zcap <= kFixedCap)
        return g.slopes ? launch<DP, true, true, true>(g, q, k, v, st) : launch<DP, true, false, true>(g, q, k, v, st);
    if (cap) return g.slopes ? launch<DP, true, true, false>(g, q, k, v, st) : launch<DP, true, false, false>(g, q, k, v, st);
    return g.slopes ? launch<DP, false, true, false>(g, q, k, v, st) : launch<DP, false, false, false>(g, q, k, v, st);
}

}  // namespace

int attention_check(const char* what, const AttentionShape& s, uint64_t n_q, uint64_t n_k, int nseg, const void* q,
                    int ldq, const void* k, int ldk, const void* v, int ldv, const void* out, int ldo) {
    const std::string w = std::string(what) + ": ";
    if (s.heads <= 0 || s.heads > 65535 || s.kv_heads <= 0 || s.heads % s.kv_heads)
        return fail(w + "heads must be a multiple of kv_heads");
    if (s.dim <= 0 || s.dim > 128 || s.dim % 8) return fail_code(GAT_B200_EUNSUPPORTED, w + "dim must be a multiple of 8, at most 128");
    if (n_q > uint64_t(INT32_MAX - 512) || n_k > uint64_t(INT32_MAX - 512)) return fail(w + "too many rows");
    if (nseg < 0) return fail(w + "bad segment count");
    if (nseg > INT32_MAX - 513) return fail(w + "too many segments");
    if (!(s.scale > 0.f) || s.scale > 1e30f) return fail(w + "scale must be positive, at most 1e30");
    if (!(s.cap >= 0.f) || s.cap > 1e30f) return fail(w + "cap must lie in 0 (none) .. 1e30");
    if (s.cap > 0.f && s.scale / s.cap > 1e30f) return fail(w + "cap too small for the scale");
    const int64_t hq = int64_t(s.heads) * s.dim, hk = int64_t(s.kv_heads) * s.dim;
    if (ldq < hq || ldk < hk || ldv < hk || ldo < hq) return fail(w + "row stride smaller than heads * dim");
    if ((ldq | ldk | ldv | ldo) % 8) return fail(w + "rows must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
         reinterpret_cast<uintptr_t>(out)) & 15)
        return fail(w + "rows must be 16-byte aligned");
    return 0;
}

int masked_attention_launch(const AttentionShape& s, int nseg, uint64_t n_q, uint64_t n_k, const uint64_t* q_row,
                            const uint64_t* k_row, int mask, const uint64_t* prefix, const void* q, int ldq,
                            const void* k, int ldk, const void* v, int ldv, void* out, int ldo, float* lse,
                            cudaStream_t st) {
    if (int rc = attention_check("masked_attention", s, n_q, n_k, nseg, q, ldq, k, ldk, v, ldv, out, ldo)) return rc;
    if (mask < GAT_B200_MASK_FULL || mask > GAT_B200_MASK_PREFIX) return fail("masked_attention: bad mask");
    if (mask == GAT_B200_MASK_PREFIX && !prefix) return fail("masked_attention: the prefix mask needs the prefix lengths");
    if (n_q == 0) return 0;
    if (nseg == 0) return fail("masked_attention: rows without segments");
    if (!q_row || !k_row || !q || !out || (n_k && (!k || !v))) return fail("masked_attention: null argument");
    if ((reinterpret_cast<uintptr_t>(q_row) | reinterpret_cast<uintptr_t>(k_row) | reinterpret_cast<uintptr_t>(prefix)) % 8 ||
        (reinterpret_cast<uintptr_t>(s.slopes) | reinterpret_cast<uintptr_t>(lse)) % 4)
        return fail("masked_attention: misaligned pointer");
    if (int rc = check_device_pointers("masked_attention", {q_row, k_row, prefix, q, k, v, s.slopes, out, lse})) return rc;
    AttnArgs g{};
    g.n_q = n_q;
    g.n_k = n_k;
    g.heads = s.heads;
    g.group = s.heads / s.kv_heads;
    g.dim = s.dim;
    g.nseg = nseg;
    g.mask = mask;
    g.q_row = q_row;
    g.k_row = k_row;
    g.prefix = mask == GAT_B200_MASK_PREFIX ? prefix : nullptr;
    g.slopes = s.slopes;
    g.v = static_cast<const uint16_t*>(v);
    g.ldv = ldv;
    g.zscale = s.cap > 0.f ? s.scale / s.cap : s.scale * kLog2e;
    g.zcap = s.cap * kLog2e;
    if (s.cap > 0.f) {
        const double t = double(s.scale) / s.cap;
        const bool fits = t <= kTanhScale;
        g.small = !fits ? -1.f : kTanhLimit / t < kTanhProducts ? float(kTanhLimit / t) : kTanhProducts;
        double power = t * s.cap * 1.4426950408889634;
        for (int i = 0; i < 5; ++i, power *= t * t) {
            g.tanh[i] = fits ? float(kTanh[i] * power) : 0.f;
            if (i < 3) g.tanh3[i] = fits ? float(kTanhShort[i] * power) : 0.f;
        }
    }
    g.out = static_cast<uint16_t*>(out);
    g.ldo = ldo;
    g.lse = lse;
    CUtensorMap tq, tk, tv;
    if (int rc = heads_map(&tq, q, s.dim, s.heads, n_q, ldq)) return rc;
    // without keys nothing is loaded: any valid map will do
    if (int rc = heads_map(&tk, n_k ? k : q, s.dim, n_k ? s.kv_heads : s.heads, n_k ? n_k : n_q, n_k ? ldk : ldq)) return rc;
    if (int rc = heads_map(&tv, n_k ? v : q, s.dim, n_k ? s.kv_heads : s.heads, n_k ? n_k : n_q, n_k ? ldv : ldq)) return rc;
    return s.dim <= 64 ? launch<64>(g, s.cap > 0.f, tq, tk, tv, st) : launch<128>(g, s.cap > 0.f, tq, tk, tv, st);
}

int attention_check_error() {
    unsigned e = 0;
    GATB_CUDA(cudaMemcpyFromSymbol(&e, g_attention_error, sizeof(e)));
    if (e) {
        unsigned z = 0;
        cudaMemcpyToSymbol(g_attention_error, &z, sizeof(z));
        return fail_code(GAT_B200_ETIMEOUT, "masked_attention kernel: a bounded wait timed out");
    }
    return 0;
}

}  // namespace gatb
