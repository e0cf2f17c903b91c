/* r3d_epi.h -- host-side plan of gemm_nt_epi: a product with bias, activation and residual in its epilogue,
 *     Y[m, n] = act(S * sum_k A[m, k] B[n, k] + bias[n]) + residual[m, n],
 * at bf16 (S = 1) and at i8a8 (S = a_scale[m] * b_scale[n], the sum exact in i32).  Pure host C++. */
#ifndef R3D_EPI_H
#define R3D_EPI_H

#include <stdint.h>
#include "r3d_i8.h"
#include "rad_abi.h"

namespace r3d {

/* f32 sums of bf16 products stay good to K / 2^24 of their terms' size */
constexpr int64_t kEpiMaxK = int64_t(1) << 20;

struct EpiPlan {
    I8Plan p;                /* A, B and K in bytes; SA and SB null at bf16; Y's elements are bf16 or f32 */
    int bf16;                /* the operands' type: bf16, or int8 */
    int64_t K;               /* in elements */
    const void* bias;
    const void* res;
    int64_t bias_stride, r_pitch;
    int act, bias_bf16, res_bf16, y_bf16;
};

/* The operands (a, a_scale?, b, b_scale?, bias?, residual?, y) and params of a call; bf16: which row. */
int plan_epi(const RadArgs* a, bool bf16, EpiPlan* P);

/* The planes that a call's best launch wants (the rows' scratch hook). */
int64_t epi_scratch_bytes(const RadArgs* a, bool bf16, int ncu);

/* describe() for gemm_nt_epi's rows; -1 when `row` is not one of them. */
int describe_epi(const char* row, const RadArgs* a, char* buf, int len);

bool env_no_epi();

}  // namespace r3d

#endif /* R3D_EPI_H */
