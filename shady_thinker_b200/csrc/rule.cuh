// Score rules of the rule attention kernels: what a query sees, and what happens to its scores (shady_score_rule).
#pragma once
#include <math.h>

#include "common.cuh"

namespace shady {

constexpr float kRuleLog2e = 1.4426950408889634f;
constexpr float kRuleLn2 = 0.6931471805599453f;

struct RuleArgs {
    float scale;          // z = q.k * scale
    float cap, inv_cap;   // cap > 0: z = cap * tanh(z * inv_cap)
    uint32_t window;      // 0 = none
    const float *slopes;
    const uint32_t *prefix, *doc;
};

// Checks a caller's rule and turns it into the device-side form (decode_rule.cu).
int fill_rule(shady_ctx *ctx, const shady_score_rule *rule, uint32_t head_dim, const char *who, RuleArgs *out);

__device__ __forceinline__ float rule_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rule_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rule_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh(z) = 1 - 2 / (1 + e^(2z)), with z2 = 2 z log2(e).  The absolute error is a few 2^-24 everywhere (near 0 the
// two halves cancel, but a score needs cap * tanh to an absolute error, not a relative one); tanh.approx is 2^-11 off,
// which a cap of 50 turns into 2 % of a weight.
__device__ __forceinline__ float rule_tanh_of_exp(float z2) { return 1.0f - 2.0f * rule_rcp(1.0f + rule_exp2(z2)); }

// tanh(x) = x P(x^2) for |x| <= 3/4, fitted to the least largest absolute error (Lawson's reweighted least squares):
// 9.5e-9, in f32 arithmetic 7.6e-8.  (One degree less would do for the weights, 1.9e-7, but near 0 it is 2.8e-6 of the score
// off, which the log-sum-exp shows.)
constexpr float kTanhSmall = 0.75f;
constexpr float kTanhC0 = 0.999999821f, kTanhC1 = -0.333324701f, kTanhC2 = 0.133205801f, kTanhC3 = -0.0531492606f, kTanhC4 = 0.0192372371f,
                kTanhC5 = -0.00449345633f;
// the same for |x| <= 1/5 with P of degree 2: 1.0e-8, in f32 arithmetic 2.5e-8
constexpr float kTanhTiny = 0.2f;
constexpr float kTanhT0 = 0.999999643f, kTanhT1 = -0.333259940f, kTanhT2 = 0.129634932f;
__device__ __forceinline__ float rule_tanh_small(float x) {
    const float t = x * x;
    return x * fmaf(fmaf(fmaf(fmaf(fmaf(kTanhC5, t, kTanhC4), t, kTanhC3), t, kTanhC2), t, kTanhC1), t, kTanhC0);
}

}  // namespace shady
