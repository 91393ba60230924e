// Masked attention of one new row per segment over its keys (single tokens).
//
// The bytes of K and V bound it: every key and value is read once, for all
// query heads of its key head together (up to eight a CTA). The keys of all
// segments, laid end to end, are cut into equal runs, one per CTA column, so
// neither one long segment nor many ragged ones leave SMs idle (each segment
// counts as kPieceCost keys more than it has: what starting a piece costs). A
// segment cut by a run's border leaves a partial state (maximum, sum, weighted
// values) per piece, and a second kernel, started ahead by programmatic launch,
// joins a segment's pieces in their order.
//
// A warp takes 32 keys at a time, straight from global memory into the
// fragments of mma.sync m16n8k16 (16-byte loads; which of the 16 reduction
// slots a column takes does not matter as long as q and k agree):
//   S^T [16 keys x 8 heads] = K Q^T;  P^T by movmatrix;  O^T [16 columns x 8 heads] += V^T P^T.
// mma.sync is ample: 16 keys are 16 MMAs for 8 KB of K and V.
//
// P is rounded to BF16 (the MMA's input type). A warp's weighted values are an
// average over its own rounded weights, scaled to the sum of the unrounded ones,
// with which states are joined and the log-sum-exp is made.
#include "attention.cuh"

namespace gatb {

namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 32;       // keys of a warp's step
constexpr int kHeadTile = 8;    // query heads of a CTA
constexpr uint64_t kPieceCost = kWarps * kKeys;

struct StepArgs {
    uint64_t n_k;
    int heads, kv_heads, group, dim, nseg, runs;
    const uint64_t* begin;
    const uint64_t* length;
    const float* slopes;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    int ldq, ldk, ldv;
    float zscale, zcap;
    uint16_t* out;
    int ldo;
    float* lse;
    float* part;  // [runs + nseg][heads][dim + 2]: weighted values, maximum, sum
};

// Key count of a segment, kept inside the table.
__device__ __forceinline__ uint64_t seg_len(const StepArgs& a, int s) {
    const uint64_t b = a.begin[s], l = a.length[s];
    return b >= a.n_k ? 0 : min(l, a.n_k - b);
}

// Places of a segment in the runs.
__device__ __forceinline__ uint64_t seg_places(uint64_t len) { return len ? len + kPieceCost : 0; }

// Places of all segments and places before segment `upto`; all threads of the CTA.
__device__ __forceinline__ void count_keys(const StepArgs& a, int upto, uint64_t& total, uint64_t& before) {
    __shared__ uint64_t part[2][32];
    uint64_t t = 0, b = 0;
    for (int s = threadIdx.x; s < a.nseg; s += blockDim.x) {
        const uint64_t l = seg_places(seg_len(a, s));
        t += l;
        if (s < upto) b += l;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        t += __shfl_xor_sync(0xffffffffu, t, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if ((threadIdx.x & 31) == 0) {
        part[0][threadIdx.x >> 5] = t;
        part[1][threadIdx.x >> 5] = b;
    }
    __syncthreads();
    total = before = 0;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) {
        total += part[0][w];
        before += part[1][w];
    }
    __syncthreads();
}
// Places of a run: the total in `runs` parts, whole steps of a CTA.
__device__ __forceinline__ uint64_t run_places(uint64_t total, int runs) {
    constexpr uint64_t unit = kWarps * kKeys;
    const uint64_t c = (total + runs - 1) / runs;
    return (c + unit - 1) / unit * unit;
}

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint4 load16(const uint16_t* p, bool ok) {
    return ok ? ldg_nc_v4(p) : make_uint4(0, 0, 0, 0);
}

// SETS: 64-column sets of the head dim. Grid: (runs, kv_heads, tiles of 8 query heads).
template <int SETS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kWarps * 32) attention_step_kernel(const StepArgs a) {
    constexpr int kTiles = 4 * SETS;  // 16-column tiles of O^T; also K's MMA steps of 16 columns
    __shared__ float o_s[kWarps][kHeadTile][64 * SETS + 4];
    __shared__ float m_s[kWarps][kHeadTile], l_s[kWarps][kHeadTile];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rr = lane >> 2, qq = lane & 3;  // fragment row and quad
    const int kvh = blockIdx.y, head0 = kvh * a.group + blockIdx.z * kHeadTile;
    const int live_heads = min(kHeadTile, a.group - int(blockIdx.z) * kHeadTile);

    asm volatile("griddepcontrol.launch_dependents;");
    if (a.runs == 1) {  // no second kernel: segments without keys are written here
        for (int s = 0; s < a.nseg; ++s) {
            if (seg_len(a, s)) continue;
            for (int e = threadIdx.x; e < live_heads * a.dim; e += kWarps * 32)
                a.out[uint64_t(s) * a.ldo + uint64_t(head0) * a.dim + e] = 0;
            if (a.lse && int(threadIdx.x) < live_heads) a.lse[uint64_t(s) * a.heads + head0 + threadIdx.x] = -INFINITY;
        }
    }
    // Where this run lies: a thread adds up the places of neighbouring segments, a
    // scan over the threads gives the total and the first segment of the run. Up
    // to kKept segments' keys stay in shared memory (300 segments of 40 keys,
    // 16/4 x 128: 29 us with two passes and reads in between, now 27).
    constexpr int kThreads = kWarps * 32, kKept = 512;
    __shared__ uint64_t sums[kWarps], len_s[kKept], begin_s[kKept];
    __shared__ int found;
    __shared__ uint64_t found_start;
    const bool kept = a.nseg <= kKept;
    const int each = (a.nseg + kThreads - 1) / kThreads;
    const int s0 = min(a.nseg, int(threadIdx.x) * each), s1 = min(a.nseg, s0 + each);
    uint64_t places = 0;
    for (int s = s0; s < s1; ++s) {
        const uint64_t len = seg_len(a, s);
        if (kept) {
            len_s[s] = len;
            begin_s[s] = a.begin[s];
        }
        places += seg_places(len);
    }
    uint64_t off = places;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, off, o);
        if (lane >= o) off += y;
    }
    if (lane == 31) sums[warp] = off;
    __syncthreads();
    off -= places;  // places before this thread's segments
    uint64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) off += sums[w];
        total += sums[w];
    }
    const uint64_t run = run_places(total, a.runs), v0 = run * blockIdx.x, v1 = min(total, v0 + run);
    if (v0 >= v1) return;  // the same for the whole CTA
    if (off <= v0 && v0 < off + places) {
        int s = s0;
        for (;; ++s) {
            const uint64_t l = seg_places(kept ? len_s[s] : seg_len(a, s));
            if (v0 < off + l) break;
            off += l;
        }
        found = s;
        found_start = off;
    }
    __syncthreads();
    int seg = found;
    uint64_t seg_start = found_start;  // places before it

    float slope[2] = {0.f, 0.f};
    if constexpr (BIAS) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * qq + i < live_heads) slope[i] = -a.slopes[head0 + 2 * qq + i] * kLog2e;
    }

    for (uint64_t at = v0; at < v1; ++seg) {
        const uint64_t len = kept ? len_s[seg] : seg_len(a, seg);
        if (len == 0) continue;
        const uint64_t j0 = at - seg_start, j1 = min(len, v1 - seg_start);
        const bool entire = j0 == 0 && j1 == len;
        at = seg_start + seg_places(len);
        if (j0 >= j1) {  // only the places behind its keys
            seg_start = at;
            continue;
        }
        const uint64_t kbase = kept ? begin_s[seg] : a.begin[seg];
        // Q as B fragments: head rr, the 8 columns 32 i + 8 qq of two reduction steps
        uint4 qf[2 * SETS];
#pragma unroll
        for (int i = 0; i < 2 * SETS; ++i) {
            const int col = 32 * i + 8 * qq;
            qf[i] = load16(a.q + uint64_t(seg) * a.ldq + uint64_t(head0 + rr) * a.dim + col, rr < live_heads && col < a.dim);
        }
        float o[kTiles][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, lr[2] = {0.f, 0.f};  // maximum, sums of weights and rounded weights

        for (uint64_t j = j0 + warp * kKeys; j < j1; j += kWarps * kKeys) {
            const uint16_t* kp = a.k + (kbase + j) * uint64_t(a.ldk) + uint64_t(kvh) * a.dim;
            const uint16_t* vp = a.v + (kbase + j) * uint64_t(a.ldv) + uint64_t(kvh) * a.dim;
            const int left = int(min(uint64_t(kKeys), j1 - j));
            uint4 kf[2][2][2 * SETS];  // 16-key tile, rows rr and rr + 8
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2 * SETS; ++i) {
                        const int key = 16 * t + 8 * h + rr, col = 32 * i + 8 * qq;
                        kf[t][h][i] = load16(kp + uint64_t(key) * a.ldk + col, key < left && col < a.dim);
                    }
            uint4 vf[2][4][SETS];  // keys 2 qq, 2 qq + 1, 2 qq + 8, 2 qq + 9; the 8 columns 64 s + 8 rr
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int s = 0; s < SETS; ++s) {
                        const int key = 16 * t + (h >> 1) * 8 + 2 * qq + (h & 1), col = 64 * s + 8 * rr;
                        vf[t][h][s] = load16(vp + uint64_t(key) * a.ldv + col, key < left && col < a.dim);
                    }
            float z[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * SETS; ++i) {
                    const uint4 k0 = kf[t][0][i], k1 = kf[t][1][i];
                    const uint32_t fa[4] = {k0.x, k1.x, k0.y, k1.y}, fb[4] = {k0.z, k1.z, k0.w, k1.w};
                    mma16816(z[t], fa, qf[i].x, qf[i].y);
                    mma16816(z[t], fb, qf[i].z, qf[i].w);
                }
            }
            // z[t][2 h + i]: key 16 t + 8 h + rr, head 2 qq + i
            float mb[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int key = 16 * t + 8 * h + rr;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float& x = z[t][2 * h + i];
                        x = CAP ? capped_score(x * a.zscale, a.zcap) : x * a.zscale;
                        if constexpr (BIAS) x = fmaf(slope[i], float(len - 1 - (j + key)), x);
                        if (key >= left) x = -INFINITY;
                        mb[i] = fmaxf(mb[i], x);
                    }
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) mb[i] = fmaxf(mb[i], __shfl_xor_sync(0xffffffffu, mb[i], s));
            }
            const float mn[2] = {fmaxf(m[0], mb[0]), fmaxf(m[1], mb[1])};
            if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
                const float f[2] = {ex2(m[0] - (mn[0] == -INFINITY ? 0.f : mn[0])),
                                    ex2(m[1] - (mn[1] == -INFINITY ? 0.f : mn[1]))};
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    o[t][0] *= f[0];
                    o[t][1] *= f[1];
                    o[t][2] *= f[0];
                    o[t][3] *= f[1];
                }
                l[0] *= f[0];
                l[1] *= f[1];
                lr[0] *= f[0];
                lr[1] *= f[1];
                m[0] = mn[0];
                m[1] = mn[1];
            }
            const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = ex2(z[t][e] - ref[e & 1]);
                    l[e & 1] += p[e];
                }
                const uint32_t r0 = pack_bf16x2(p[0], p[1]), r1 = pack_bf16x2(p[2], p[3]);
                lr[0] += bf16lo(r0) + bf16lo(r1);
                lr[1] += bf16hi(r0) + bf16hi(r1);
                const uint32_t b0 = transpose8x8(r0), b1 = transpose8x8(r1);
#pragma unroll
                for (int s = 0; s < SETS; ++s) {
                    const uint32_t* x0 = &vf[t][0][s].x;
                    const uint32_t* x1 = &vf[t][1][s].x;
                    const uint32_t* x2 = &vf[t][2][s].x;
                    const uint32_t* x3 = &vf[t][3][s].x;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        // columns 64 s + 8 rr + 2 w (fragment row rr) and + 1 (row rr + 8)
                        const uint32_t fa[4] = {__byte_perm(x0[w], x1[w], 0x5410), __byte_perm(x0[w], x1[w], 0x7632),
                                                __byte_perm(x2[w], x3[w], 0x5410), __byte_perm(x2[w], x3[w], 0x7632)};
                        mma16816(o[4 * s + w], fa, b0, b1);
                    }
                }
            }
        }

        // the four warps' states of this piece, joined in warp order
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], s);
                lr[i] += __shfl_xor_sync(0xffffffffu, lr[i], s);
            }
            const float own = lr[i] > 0.f ? l[i] / lr[i] : 1.f;  // no weights: zeros
            if (rr == 0) {
                m_s[warp][2 * qq + i] = m[i];
                l_s[warp][2 * qq + i] = l[i];
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int col = 64 * (t >> 2) + 8 * rr + 2 * (t & 3);
                o_s[warp][2 * qq + i][col] = o[t][i] * own;
                o_s[warp][2 * qq + i][col + 1] = o[t][2 + i] * own;
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < live_heads * a.dim; e += kWarps * 32) {
            const int h = e / a.dim, c = e % a.dim;
            float mm = m_s[0][h];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, m_s[w][h]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f, acc = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(m_s[w][h] - ref);  // a warp without keys adds zeros
                sum = fmaf(l_s[w][h], f, sum);
                acc = fmaf(o_s[w][h][c], f, acc);
            }
            const int head = head0 + h;
            if (entire) {
                a.out[uint64_t(seg) * a.ldo + uint64_t(head) * a.dim + c] = uint16_t(pack_bf16x2(acc / sum, 0.f));
                if (a.lse && c == 0) a.lse[uint64_t(seg) * a.heads + head] = (mm + log2f(sum)) * kLn2;
            } else {
                float* p = a.part + ((uint64_t(blockIdx.x) + seg) * a.heads + head) * (a.dim + 2);
                p[c] = acc;
                if (c == 0) {
                    p[a.dim] = mm;
                    p[a.dim + 1] = sum;
                }
            }
        }
        __syncthreads();
        seg_start = at;
    }
}

constexpr int kMostRuns = 512;  // runs are never more than this
constexpr int kJoinTeams = 4;   // teams of 128 threads, a column each

// Grid (segments, heads / HEADS): joins the pieces of a segment that runs cut,
// writes zeros for a segment without keys. HEADS 1: the teams share a head's
// pieces (few, long segments). HEADS 4: a head a team (many segments: fewer CTAs
// that find their segment uncut).
template <int HEADS>
__global__ void __launch_bounds__(kJoinTeams * 128) attention_join_kernel(const StepArgs a) {
    constexpr int kShare = kJoinTeams / HEADS;  // teams of one head
    constexpr int kWarpsHead = 4 * kShare;
    __shared__ float f_s[HEADS][kMostRuns], red[kJoinTeams * 4], acc_s[kJoinTeams][128];
    const int seg = blockIdx.x, c = threadIdx.x & 127, team = threadIdx.x >> 7;
    const int sub = HEADS == 1 ? 0 : team, share = HEADS == 1 ? team : 0;
    const int head = blockIdx.y * HEADS + sub;
    const bool live = head < a.heads;
    uint64_t total, start;
    count_keys(a, seg, total, start);
    const uint64_t len = seg_len(a, seg);
    uint16_t* out = a.out + uint64_t(seg) * a.ldo + uint64_t(head) * a.dim;
    const uint64_t run = run_places(total, a.runs);
    const uint64_t first = len ? start / run : 0, last = len ? (start + len - 1) / run : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the pieces are written
    if (len == 0) {
        if (live && share == 0 && c < a.dim) out[c] = 0;
        if (live && share == 0 && c == 0 && a.lse) a.lse[uint64_t(seg) * a.heads + head] = -INFINITY;
        return;
    }
    if (first == last) return;  // one piece: written already
    const uint64_t stride = uint64_t(a.heads) * (a.dim + 2);
    const float* p = a.part + ((first + seg) * a.heads + (live ? head : 0)) * uint64_t(a.dim + 2);
    const int n = int(last - first + 1);
    // the pieces' maxima and sums, a thread each
    float mm = -INFINITY;
    for (int i = share * 128 + c; i < n; i += kShare * 128) mm = fmaxf(mm, p[i * stride + a.dim]);
    mm = warp_max(mm);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarpsHead; ++w) mm = fmaxf(mm, red[sub * kWarpsHead + w]);
    __syncthreads();
    float part = 0.f;
    for (int i = share * 128 + c; i < n; i += kShare * 128) {
        const float f = ex2(p[i * stride + a.dim] - (mm == -INFINITY ? 0.f : mm));
        f_s[sub][i] = f;
        part = fmaf(p[i * stride + a.dim + 1], f, part);
    }
    part = warp_sum(part);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = part;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarpsHead; ++w) sum += red[sub * kWarpsHead + w];
    float acc = 0.f;
    if (c < a.dim) {
#pragma unroll 8
        for (int i = share; i < n; i += kShare) acc = fmaf(p[i * stride + c], f_s[sub][i], acc);
    }
    if constexpr (kShare > 1) {
        acc_s[team][c] = acc;
        __syncthreads();
        acc = acc_s[0][c];
#pragma unroll
        for (int t = 1; t < kShare; ++t) acc += acc_s[t][c];
    }
    if (!live || share) return;
    if (c < a.dim) out[c] = uint16_t(pack_bf16x2(acc / sum, 0.f));
    if (c == 0 && a.lse) a.lse[uint64_t(seg) * a.heads + head] = (mm + log2f(sum)) * kLn2;
}

// Runs the keys are cut into: all the CTAs that fit the SMs at once (three or
// two an SM by their registers), no more than there can be pieces for, also
// where segments share keys (119 segments of up to 9 keys took 55 us in as many
// runs as their keys fill, and take 9).
int step_runs(int kv_heads, int group, int dim, uint64_t n_k, int nseg, int sms) {
    const int columns = kv_heads * ((group + kHeadTile - 1) / kHeadTile);
    const uint64_t want = uint64_t((dim <= 64 ? 3 : 2) * sms / columns);
    const uint64_t most = (n_k + kWarps * kKeys - 1) / (kWarps * kKeys) * uint64_t(nseg);
    const uint64_t runs = want < most ? want : most;
    return runs < 1 ? 1 : runs > uint64_t(kMostRuns) ? kMostRuns : int(runs);
}

}  // namespace

uint64_t masked_attention_step_workspace(int heads, int dim, int nseg) {
    if (heads <= 0 || dim <= 0 || nseg < 0) return 0;
    return (uint64_t(kMostRuns) + nseg) * uint64_t(heads) * (uint64_t(dim) + 2) * 4;
}

int masked_attention_step_launch(const AttentionShape& s, int nseg, uint64_t n_k, const uint64_t* begin,
                                 const uint64_t* length, const void* q, int ldq, const void* k, int ldk, const void* v,
                                 int ldv, void* out, int ldo, float* lse, void* workspace, uint64_t workspace_bytes,
                                 cudaStream_t st) {
    if (int rc = attention_check("masked_attention_step", s, nseg > 0 ? uint64_t(nseg) : 0, n_k, nseg, q, ldq, k, ldk, v,
                                 ldv, out, ldo))
        return rc;
    if (nseg == 0) return 0;
    if (!begin || !length || !q || !out || (n_k && (!k || !v))) return fail("masked_attention_step: null argument");
    if ((reinterpret_cast<uintptr_t>(begin) | reinterpret_cast<uintptr_t>(length)) % 8 ||
        (reinterpret_cast<uintptr_t>(s.slopes) | reinterpret_cast<uintptr_t>(lse)) % 4 ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail("masked_attention_step: misaligned pointer");
    if (!workspace || workspace_bytes < masked_attention_step_workspace(s.heads, s.dim, nseg))
        return fail("masked_attention_step: workspace too small");
    if (s.kv_heads > 65535) return fail("masked_attention_step: too many heads");
    if (int rc = check_device_pointers("masked_attention_step",
                                       {begin, length, q, k, v, s.slopes, out, lse, workspace}))
        return rc;
    int dev = 0, sms = 0;
    GATB_CUDA(cudaGetDevice(&dev));
    GATB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    StepArgs a{};
    a.n_k = n_k;
    a.heads = s.heads;
    a.kv_heads = s.kv_heads;
    a.group = s.heads / s.kv_heads;
    a.dim = s.dim;
    a.nseg = nseg;
    a.runs = step_runs(a.kv_heads, a.group, a.dim, n_k, nseg, sms);
    a.begin = begin;
    a.length = length;
    a.slopes = s.slopes;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.zscale = s.cap > 0.f ? s.scale / s.cap : s.scale * kLog2e;
    a.zcap = s.cap * kLog2e;
    a.out = static_cast<uint16_t*>(out);
    a.ldo = ldo;
    a.lse = lse;
    a.part = static_cast<float*>(workspace);
    const dim3 grid(unsigned(a.runs), unsigned(a.kv_heads), unsigned((a.group + kHeadTile - 1) / kHeadTile));
    auto go = [&](auto kern) { kern<<<grid, kWarps * 32, 0, st>>>(a); };
    const bool cap = s.cap > 0.f, bias = s.slopes != nullptr;
    if (s.dim <= 64) {
        if (cap && bias) go(attention_step_kernel<1, true, true>);
        else if (cap) go(attention_step_kernel<1, true, false>);
        else if (bias) go(attention_step_kernel<1, false, true>);
        else go(attention_step_kernel<1, false, false>);
    } else {
        if (cap && bias) go(attention_step_kernel<2, true, true>);
        else if (cap) go(attention_step_kernel<2, true, false>);
        else if (bias) go(attention_step_kernel<2, false, true>);
        else go(attention_step_kernel<2, false, false>);
    }
    GATB_LAUNCH("masked_attention_step kernel");
    if (a.runs == 1) return 0;
    const bool many = uint64_t(nseg) * s.heads > uint64_t(2 * sms);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(nseg), unsigned(many ? (s.heads + 3) / 4 : s.heads));
    cfg.blockDim = dim3(kJoinTeams * 128);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    GATB_CUDA(many ? cudaLaunchKernelEx(&cfg, attention_join_kernel<4>, a)
                   : cudaLaunchKernelEx(&cfg, attention_join_kernel<1>, a));
    return 0;
}

}  // namespace gatb
