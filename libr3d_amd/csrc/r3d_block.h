/* r3d_block.h -- host-side plan of rmsnorm_block: what lies between two blocks of a model, in one pass,
 *     t = x rs(x) (w_post + wadd)          the norm after a block (without w_post: t = x)
 *     h = res_scale residual + gate t      its gate and the residual stream (each optional), to residual_out
 *     v = h rs(h) (w_pre + wadd)           the norm before the next block: out, and int8 or e4m3 codes of it
 * with rs(a) = 1 / sqrt(sum a^2 / n + eps).  Pure host C++. */
#ifndef R3D_BLOCK_H
#define R3D_BLOCK_H

#include <stdint.h>
#include "rad_abi.h"

namespace r3d {

enum { BLOCK_NO_CODES = 0, BLOCK_I8, BLOCK_E4M3 };
enum { BLOCK_NO_GATE = 0, BLOCK_GATE_ROWS, BLOCK_GATE_TOKEN };   /* [n] (pitch 0) or [M, n]; [M, 1] */

constexpr int64_t kBlockMaxN = 32768;      /* a row lies in the registers of 1024 lanes */

struct BlockPlan {
    const uint8_t* x;
    const uint8_t* res;          /* bf16 */
    const uint8_t* w_post;
    const uint8_t* gate;
    const uint8_t* w_pre;
    uint8_t* res_out;            /* bf16 */
    uint8_t* out;
    uint8_t* q;
    float* scale;
    int x_bf16, w_bf16, out_bf16;          /* w_bf16: the weights' and the gate's type */
    int gate_kind, codes;
    int64_t rows, n, x_pitch, r_pitch, g_pitch, ro_pitch, o_pitch, q_pitch, s_pitch;
    double eps;
    float wadd, res_scale;
};

int plan_block(const RadArgs* a, BlockPlan* P);

/* Lanes of a row's workgroup and 8-element chunks a lane holds; past: results are not kept in the caches. */
struct BlockGeom {
    int lanes, chunks, past;
};
BlockGeom block_geom(int64_t rows, int64_t n);

/* describe() for this row; -1 when `row` is another. */
int describe_block(const char* row, const RadArgs* a, char* buf, int len);

bool env_no_block();

}  // namespace r3d

#endif /* R3D_BLOCK_H */
