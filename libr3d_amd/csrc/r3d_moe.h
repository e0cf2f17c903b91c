/* r3d_moe.h -- host-side plan of moe_layer: a mixture-of-experts layer for a few tokens, in three launches (past 8 tokens four, and
 * more where an expert is wide).
 *     choice   the top_k largest router logits of a token, by falling logit, ties to the lower index
 *     weights  softmax over the logits, or a sigmoid of each; of the chosen ones' sum where renorm; times weight_scale
 *     h        weight * act(W_gate x) * (W_up x)          the chosen expert's f rows each
 *     y        the chosen experts' W_down h, added up
 * Expert planes in bf16, in int8 with one f32 scale a row, or in e2m1 with one E8M0 scale a row and 32 columns.
 * Pure host C++. */
#ifndef R3D_MOE_H
#define R3D_MOE_H

#include <stdint.h>
#include "rad_abi.h"

namespace r3d {

enum { MOE_BF16 = 0, MOE_I8, MOE_FP4 };

constexpr int kMoeMaxM = 64;            /* an expert's tokens are a 64-bit mask */
constexpr int kMoeMaxE = 512;           /* a lane of a workgroup an expert */
constexpr int kMoeMaxK = 16;            /* choices a token */
constexpr int64_t kMoeMaxN = 66560;     /* of one token's columns in LDS (int8, which keeps scales there too: 62464) */
constexpr int64_t kMoeMaxF = 1 << 16;
constexpr int kMoeMaxPairs = kMoeMaxM * kMoeMaxK;
constexpr int kMoeMaxBlocks = 256, kMoeMinBlocks = 32;      /* compute units of a device, and of its smallest partition */
/* h of all pairs lies under 32-bit offsets, units times workgroups under 2^32 (a unit is 8 rows of f or 16 of n), and
 * a run's spans (128 columns at least) times a workgroup's 8 waves under 2^31 */
static_assert(kMoeMaxPairs * kMoeMaxF * 4 <= int64_t(1) << 28, "h");
static_assert(kMoeMaxPairs * (kMoeMaxF / 8) * (kMoeMaxBlocks + 1) < int64_t(1) << 32, "units of gate and up");
static_assert(kMoeMaxPairs * ((kMoeMaxN + 15) / 16) * (kMoeMaxBlocks + 1) < int64_t(1) << 32, "units of down");
static_assert((kMoeMaxPairs * (kMoeMaxF / 8) / kMoeMinBlocks + 1) * (kMoeMaxN / 128) * 8 < int64_t(1) << 31, "spans of gate and up");
static_assert((kMoeMaxPairs * ((kMoeMaxN + 15) / 16) / kMoeMinBlocks + 1) * (kMoeMaxF / 128) * 8 < int64_t(1) << 31, "spans of down");

/* What the first kernel leaves for the others at the head of the scratch; h and the slots' sums follow.  A slot is a
 * chosen (token, expert), in the experts' order. */
struct MoeTable {
    int32_t jobs;                       /* the down kernel's groups of an expert's tokens, in the experts' order */
    int32_t pad[3];
    uint32_t job[kMoeMaxPairs];         /* expert | first slot << 9 | tokens << 20 */
    int16_t slot[kMoeMaxPairs];         /* by (token, choice); -1: none */
    int16_t id[kMoeMaxPairs];           /* choices of many tokens, and their weights */
    float w[kMoeMaxPairs];
};

struct MoePlan {
    const uint8_t* x;                   /* bf16 [M, n] */
    const uint8_t* logits;              /* f32 or bf16 [M, E] */
    const uint8_t* gu;                  /* [E, 2f, n]: gate rows, then up rows */
    const uint8_t* gus;
    const uint8_t* dn;                  /* [E, n, f] */
    const uint8_t* dns;
    uint8_t* y;                         /* bf16 or f32 [M, n] */
    int32_t* ids;                       /* [M, top_k], or null */
    float* weights;                     /* [M, top_k], or null */
    int64_t M, n, f, E, top_k;
    /* bytes, or scales' elements */
    int64_t x_pitch, l_pitch, y_pitch, gu_expert, gu_pitch, dn_expert, dn_pitch;
    int64_t gus_expert, gus_pitch, dns_expert, dns_pitch, i_pitch, w_pitch;
    int enc, l_bf16, y_bf16, act, sigmoid, renorm;
    float weight_scale;
};

int plan_moe(const RadArgs* a, MoePlan* P);

/* A product's launch: tokens a job (in 8 ct columns), and rows of them that LDS holds. */
struct MoeTiles {
    int ct, width, rows;
};
/* The launch on ncu compute units. */
struct MoeGeom {
    MoeTiles up, down;
    int parts;                          /* down: launches, of `spans` spans of a row of h each (the last may have fewer) */
    int64_t spans, blocks;
};
/* Columns of a span, 256 bytes of a row of an expert's plane. */
constexpr int64_t moe_span(int enc) { return enc == MOE_BF16 ? 128 : enc == MOE_I8 ? 256 : 512; }
/* false: LDS does not hold a single row */
bool moe_geom(const MoePlan& P, int ncu, MoeGeom* g);

/* Bytes of scratch that a call needs (the row's hook; 0 where the sizes are not given). */
int64_t moe_scratch_bytes(const RadArgs* a);
int64_t moe_scratch(const MoePlan& P);
int64_t moe_h_bytes(const MoePlan& P);

/* describe() for this row; -1 when `row` is another. */
int describe_moe(const char* row, const RadArgs* a, char* buf, int len);

bool env_no_moe();

}  // namespace r3d

#endif /* R3D_MOE_H */
