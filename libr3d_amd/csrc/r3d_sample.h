/* r3d_sample.h -- host-side plan of the sample_logits row (r3d_sample.hip).  Pure host C++. */
#ifndef R3D_SAMPLE_H
#define R3D_SAMPLE_H

#include <stdint.h>
#include "rad_abi.h"

namespace r3d {

constexpr int kSampleSeg = 4096;         /* tokens a segment: the unit of the index-order search */
constexpr int kSampleMaxSegs = 1024;
constexpr int64_t kSampleMaxVocab = (int64_t)kSampleSeg * kSampleMaxSegs;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 8192;        /* tokens of the border bins that are listed */

/* The launch scratch, one of these a row, then seg_max, seg_min and seg_mass of its segments. */
struct SampleRow {
    unsigned long long mass[kSampleBins];
    unsigned long long list[kSampleList];         /* ~key in the high half, index in the low */
    unsigned long long mass_k, mass_p;            /* mass above the border bins of top-k and top-p */
    unsigned int count[kSampleBins];
    unsigned int n_list;
    int kb, pb_lo, pb_hi;                         /* border bins; kSampleBins: that cut is off */
    int count_k;                                  /* tokens above bin kb */
    int pad[3];
};

struct SamplePlan {
    const uint8_t* logits;               /* f32 or bf16 [M, V] */
    const float* u;
    const float* temperature;            /* null: 1 */
    const int* top_k;                    /* null: off */
    const float* top_p;
    const float* min_p;
    int* token;
    float* prob;                         /* null: not asked for */
    int bf16;
    int64_t M, V, pitch;
    int64_t u_stride, t_stride, k_stride, p_stride, m_stride, token_stride, prob_stride;
};

int plan_sample(const RadArgs* a, SamplePlan* P);
int64_t sample_scratch_bytes(int64_t M, int64_t V);
int64_t sample_hook_bytes(const RadArgs* a);
/* describe() for the row; -1 when `row` is another. */
int describe_sample(const char* row, const RadArgs* a, char* buf, int len);

bool env_no_sample();

}  // namespace r3d

#endif /* R3D_SAMPLE_H */
