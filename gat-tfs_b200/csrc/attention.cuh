// Shared pieces of the masked attention kernels. Scores are kept in units of
// log2: z = log2(e) * (cap * tanh(scale q.k / cap) - slope |distance|), so that
// a weight is one ex2.
#pragma once
#include "device.cuh"

namespace gatb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// tanh(x / (2 log2 e)) = 1 - 2 / (2^x + 1): absolute error of a few 2^-24 over
// the whole range (2^x = inf gives 1, 2^x = 0 gives -1).
__device__ __forceinline__ float tanh_of_log2(float x) { return fmaf(-2.f, rcp(ex2(x) + 1.f), 1.f); }

// What attention_check() settles for both kernels.
struct AttentionShape {
    int heads, kv_heads, dim;
    float scale, cap;
    const float* slopes;
};
int attention_check(const char* what, const AttentionShape& s, uint64_t n_q, uint64_t n_k, int nseg, const void* q,
                    int ldq, const void* k, int ldk, const void* v, int ldv, const void* out, int ldo);

}  // namespace gatb
