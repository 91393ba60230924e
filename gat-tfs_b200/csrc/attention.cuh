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

// tanh(x) = x p(x^2), minimax polynomials (Remez exchange): five terms for
// |x| <= 0.6, relative error 7.4e-8, and three for |x| <= 0.2, 1.2e-7 (for
// |x| <= 0.3 it would be 1.2e-6, and show in the log-sum-exp).
constexpr float kTanhLimit = 0.6f;
constexpr float kTanh[5] = {0.999999926872f, -0.333323099889f, 0.133101737673f, -0.0521014822761f, 0.0154754278422f};
constexpr float kTanhShort[3] = {0.9999999f, -0.3332859f, 0.13015407f};
// cap log2 e tanh(t), t = scale s / cap, for any cap and score: where tanh(t)
// is small against 1 the exponentials would cancel.
__device__ __forceinline__ float capped_score(float t, float zcap) {
    const float u = t * t;
    float p = fmaf(0.0154754278422f, u, -0.0521014822761f);
    p = fmaf(p, u, 0.133101737673f);
    p = fmaf(p, u, -0.333323099889f);
    p = fmaf(p, u, 0.999999926872f);
    return zcap * (fabsf(t) <= kTanhLimit ? t * p : tanh_of_log2(t * (2.f * kLog2e)));
}

// What attention_check() settles for both kernels.
struct AttentionShape {
    int heads, kv_heads, dim;
    float scale, cap;
    const float* slopes;
};
int attention_check(const char* what, const AttentionShape& s, uint64_t n_q, uint64_t n_k, int nseg, const void* q,
                    int ldq, const void* k, int ldk, const void* v, int ldv, const void* out, int ldo);

}  // namespace gatb
