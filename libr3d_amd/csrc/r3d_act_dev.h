/* r3d_act_dev.h -- the activations of r3d_act.h on the device, in f32. */
#ifndef R3D_ACT_DEV_H
#define R3D_ACT_DEV_H

#include <hip/hip_runtime.h>

#include "r3d_act.h"

namespace r3d {

/* sigmoid(g) = 1 / (1 + exp(-g)) in f32, within 3 ulp where that is a normal number (g over -87.3; under that
 * it may be 0, off by less than 2^-126): exp2 of the product's high part (its
 * rounding error times ln 2 is a factor on top, which keeps large |g| exact) and a reciprocal with
 * one Newton step.  Past 100 exp is inf and the result 0, as 1 / (1 + inf). */
__device__ __forceinline__ float i8_sigmoid(float g) {
    const float x = __builtin_fminf(__builtin_fmaxf(-g, -100.0f), 100.0f);
    const float t = x * 1.44269504f;
    const float lo = __builtin_fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    const float d = 1.0f + __builtin_fmaf(e, lo * 0.693147181f, e);
    float r = __builtin_amdgcn_rcpf(d);
    r = d < 3.0e38f ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) : 0.0f;
    return g != g ? g : r;
}

/* sigmoid(x) = 1 / (1 + 2^(-x log2 e)) within 3 ulp where that is a normal number, under which it may be 0, in ten instructions for
 * i8_sigmoid's eighteen: r of the rounded product by the hardware's exp2 and reciprocal (an ulp each), then what its rounding and
 * the constant's left out, lo, by the slope: r - r (1 - r) ln 2 lo.  A NaN counts as a number: the caller's. */
__device__ __forceinline__ float act_sigmoid(float x) {
    const float c = __builtin_amdgcn_fmed3f(x, -1000.0f, 1000.0f);      /* inf - inf */
    const float t = c * -1.44269504f;
    const float lo = __builtin_fmaf(c, -1.92596299e-8f, __builtin_fmaf(c, -1.44269504f, -t));
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
    return __builtin_fmaf(__builtin_fmaf(r, r, -r) * 0.693147181f, lo, r);
}

/* The same without lo: a relative error of 1.25 |x| 2^-24 more in the lower tail.  For an x whose own roundings count for more than
 * that there (gelu_tanh's: 6 |x| 2^-24).  Six instructions fewer, and an epilogue over a large product's values is bound by
 * them (2048 x 21504 x 5376, int8, us: silu 238 by this one, 242 by act_sigmoid; none 233, gelu_tanh 242). */
__device__ __forceinline__ float act_sigmoid_of_rounded(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}

/* One activation over W values; `act` is the same on every lane, so one branch is taken.
 *   gelu       v Phi(v) = v erfc(-v / sqrt 2) / 2: erfc keeps the lower tail, where 1 + erf cancels
 *   gelu_tanh  v (1 + tanh(u)) / 2 with u = sqrt(2 / pi) (v + 0.044715 v^3), which is v sigmoid(2 u)
 * A NaN stays one; silu and both gelus of -inf are NaN (-inf * 0). */
template <int W>
__device__ __forceinline__ void act_values(int act, float* v) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
            break;
        case ACT_SILU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] *= act_sigmoid(v[i]);
            break;
        case ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = v[i] != v[i] ? v[i] : act_sigmoid(v[i]);
            break;
        case ACT_GELU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = 0.5f * v[i] * erfcf(v[i] * -0.707106781f);
            break;
        case ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < W; ++i)
                v[i] *= act_sigmoid_of_rounded(v[i] * __builtin_fmaf(v[i] * v[i], 1.59576912f * 0.044715f, 1.59576912f));
            break;
        default: break;
    }
}

}  // namespace r3d

#endif /* R3D_ACT_DEV_H */
