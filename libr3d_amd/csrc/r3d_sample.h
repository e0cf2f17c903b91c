/* r3d_sample.h -- host-side plan of the sample_logits row (r3d_sample.hip).  Pure host C++. */
#ifndef R3D_SAMPLE_H
#define R3D_SAMPLE_H

#include <stdint.h>
#include "rad_abi.h"

namespace r3d {

constexpr int kSampleSeg = 4096;         /* tokens a segment: the unit of the index-order search */
constexpr int kSampleMaxSegs = 1024;
constexpr int64_t kSampleMaxVocab = (int64_t)kSampleSeg * kSampleMaxSegs;
constexpr int kSampleChunk = 64;         /* tokens a chunk: the unit that is skipped by its largest logit */
constexpr int kSampleSegChunks = kSampleSeg / kSampleChunk;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 8192;        /* tokens that are listed and sorted, at most */
constexpr int kSampleListK = 2048;       /* the largest top-k that is looked for by chunks */

/* Where the cuts fall among the bins. */
struct SampleCut {
    int kb, pb_lo, pb_hi;        /* bins: top-k's, top-p's first and last; kSampleBins: that cut is off */
    int count_k;                 /* tokens above bin kb */
    unsigned long long mass_k, mass_p;             /* mass above bins kb and pb_lo */
    unsigned long long mass_kb, total;             /* mass of bin kb, of all bins */
};

/* The launch scratch: one of these a row; of every segment its mass, of every quarter of one its sum,
 * largest and least logit, and
 * of every chunk its largest. */
struct SampleRow {
    unsigned long long mass[kSampleBins];
    unsigned long long list[kSampleList];         /* ~key in the high half, index in the low */
    SampleCut cut;
    unsigned int count[kSampleBins];
    unsigned int n_list;
    int binned, n_binned;                         /* not of this row: the i-th row that has a use for bins (in
                                                     element i), and how many there are (in the first) */
    int pad;
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
