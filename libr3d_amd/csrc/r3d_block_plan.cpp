/* r3d_block_plan.cpp -- host plan of rmsnorm_block (see r3d_block.h). */
#include "r3d_block.h"

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rad_plugin.h"
#include "r3d_operands.h"

namespace r3d {

int plan_block(const RadArgs* a, BlockPlan* P) {
    const RadTensor* x  = rad_arg_in(a, 0);
    const RadTensor* rs = rad_arg_in(a, 1);
    const RadTensor* wp = rad_arg_in(a, 2);
    const RadTensor* g  = rad_arg_in(a, 3);
    const RadTensor* wn = rad_arg_in(a, 4);
    const RadTensor* ro = rad_arg_in(a, 5);
    const RadTensor* o  = rad_arg_in(a, 6);
    const RadTensor* q  = rad_arg_in(a, 7);
    const RadTensor* sc = rad_arg_in(a, 8);
    if (!x || (q == nullptr) != (sc == nullptr) || (!ro && !o && !q)) return RAD_E_INVAL;
    if ((wn == nullptr) != (!o && !q)) return RAD_E_INVAL;      /* a norm with no result, or a result with no norm */
    if (x->dtype != RAD_BF16 && x->dtype != RAD_F32) return RAD_E_DTYPE;
    const char* dt = rad_args_gets(a, "dtype");                 /* names x's type, if given */
    if (dt && strcmp(dt, x->dtype == RAD_BF16 ? "bf16" : "f32") != 0) return RAD_E_DTYPE;
    if ((rs && rs->dtype != RAD_BF16) || (ro && ro->dtype != RAD_BF16)) return RAD_E_DTYPE;
    if (o && o->dtype != RAD_BF16 && o->dtype != RAD_F32) return RAD_E_DTYPE;
    if (sc && sc->dtype != RAD_F32) return RAD_E_DTYPE;
    P->codes = !q ? BLOCK_NO_CODES : q->dtype == RAD_I8 ? BLOCK_I8
             : q->dtype == RAD_F8E4M3 || q->dtype == RAD_U8 ? BLOCK_E4M3 : -1;
    if (P->codes < 0) return RAD_E_DTYPE;
    uint32_t wt = RAD_BF16;                                     /* one type for the weights and the gate */
    bool any = false;
    for (const RadTensor* t : {wp, g, wn}) {
        if (!t) continue;
        if ((t->dtype != RAD_F32 && t->dtype != RAD_BF16) || (any && t->dtype != wt)) return RAD_E_DTYPE;
        wt = t->dtype;
        any = true;
    }
    long long v = 0;
    if (!rad_args_geti(a, "n", &v) || v <= 0 || v > kDimMax) return RAD_E_SHAPE;
    const int64_t n = v;
    if (n > kBlockMaxN) return RAD_E_UNSUPPORTED;
    if (rad_args_geti(a, "group", &v) && v > 0 && v != (P->codes == BLOCK_E4M3 ? 128 : n)) return RAD_E_UNSUPPORTED;
    const long long xn = rad_tensor_numel(x);
    if (xn <= 0 || xn % n) return RAD_E_SHAPE;
    const int64_t rows = xn / n;
    if (rows > 0x7FFFFFFF) return RAD_E_SHAPE;
    int rc = rows_of(x, rows, n, &P->x_pitch);
    if (!rc && rs) rc = rows_of(rs, rows, n, &P->r_pitch);
    if (!rc && ro) rc = rows_of(ro, rows, n, &P->ro_pitch);
    if (!rc && o) rc = rows_of(o, rows, n, &P->o_pitch);
    if (!rc && q) rc = rows_of(q, rows, n, &P->q_pitch);
    if (!rc && sc) {
        if (P->codes == BLOCK_I8) rc = scale_column(sc, rows, &P->s_pitch);
        else rc = rows_of(sc, rows, (n + 127) / 128, &P->s_pitch);
    }
    if (rc) return rc;
    for (const RadTensor* t : {wp, wn}) {
        if (t && (t->rank != 1 || t->shape[0] != n)) return RAD_E_SHAPE;
        if (t && t->stride[0] != 1) return RAD_E_STRIDE;
    }
    P->gate_kind = BLOCK_NO_GATE;
    if (g) {
        if (g->rank == 1 && g->shape[0] == n) {
            if (g->stride[0] != 1) return RAD_E_STRIDE;
            P->gate_kind = BLOCK_GATE_ROWS;
            P->g_pitch = 0;
        } else if (g->rank == 2 && g->shape[1] == 1 && n > 1) {
            if (g->shape[0] != rows) return RAD_E_SHAPE;
            P->gate_kind = BLOCK_GATE_TOKEN;
            P->g_pitch = g->stride[0];
            if (!pitch_ok(P->g_pitch)) return RAD_E_STRIDE;
        } else {
            if (g->rank < 2) return RAD_E_SHAPE;
            P->gate_kind = BLOCK_GATE_ROWS;
            if ((rc = rows_of(g, rows, n, &P->g_pitch))) return rc;
        }
    }
    /* outputs whose rows overlap would race */
    const int64_t s_cols = P->codes == BLOCK_E4M3 ? (n + 127) / 128 : 1;
    if (rows > 1 && ((ro && P->ro_pitch < n) || (o && P->o_pitch < n) || (q && P->q_pitch < n) ||
                     (sc && P->s_pitch < s_cols)))
        return RAD_E_STRIDE;
    for (const RadTensor* t : {x, rs, wp, g, wn, ro, o, sc})
        if (misaligned(t)) return RAD_E_STRIDE;
    /* an output may be x's, the residual's or the gate's own elements (a lane reads them before it writes);
     * any other overlap would be read after it is written */
    const int xb = elt_bytes(x->dtype), wb = elt_bytes(wt);
    struct { const RadTensor* t; Span s; } outs[4] = {
        {ro, {ro ? ro->data : nullptr, rows, n, P->ro_pitch, 2}},
        {o, {o ? o->data : nullptr, rows, n, P->o_pitch, o ? elt_bytes(o->dtype) : 0}},
        {q, {q ? q->data : nullptr, rows, n, P->q_pitch, 1}},
        {sc, {sc ? sc->data : nullptr, rows, s_cols, P->s_pitch, 4}}};
    for (int i = 0; i < 4; ++i) {
        if (!outs[i].t) continue;
        if (spans_clash(outs[i].s, Span{x->data, rows, n, P->x_pitch, xb})) return RAD_E_INVAL;
        if (rs && spans_clash(outs[i].s, Span{rs->data, rows, n, P->r_pitch, 2})) return RAD_E_INVAL;
        if (g && spans_clash(outs[i].s, Span{g->data, rows, P->gate_kind == BLOCK_GATE_TOKEN ? 1 : n, P->g_pitch, wb}))
            return RAD_E_INVAL;
        for (const RadTensor* w : {wp, wn})
            if (w && spans_meet(outs[i].s, Span{w->data, 1, n, n, wb})) return RAD_E_INVAL;
        for (int j = 0; j < i; ++j)
            if (outs[j].t && spans_meet(outs[i].s, outs[j].s)) return RAD_E_INVAL;
    }
    auto bytes = [](const RadTensor* t) { return t ? (uint8_t*)t->data : nullptr; };
    P->x = bytes(x);
    P->res = bytes(rs);
    P->w_post = bytes(wp);
    P->gate = bytes(g);
    P->w_pre = bytes(wn);
    P->res_out = bytes(ro);
    P->out = bytes(o);
    P->q = bytes(q);
    P->scale = (float*)bytes(sc);
    P->x_bf16 = x->dtype == RAD_BF16;
    P->w_bf16 = wt == RAD_BF16;
    P->out_bf16 = o && o->dtype == RAD_BF16;
    P->rows = rows;
    P->n = n;
    P->eps = rad_args_getf_or(a, "eps", 1e-6);
    P->wadd = (float)rad_args_getf_or(a, "wadd", 0.0);
    P->res_scale = (float)rad_args_getf_or(a, "res_scale", 1.0);
    if (!(P->eps >= 0.0)) return RAD_E_INVAL;
    if (rows * block_geom(rows, n).lanes > 0xFFFFFFFFLL) return RAD_E_UNSUPPORTED;   /* lanes a launch */
    return RAD_OK;
}

BlockGeom block_geom(int64_t rows, int64_t n) {
    const int64_t nc = (n + 7) / 8;
    auto lanes = [&](int c) { return (int)(((nc + c - 1) / c + 63) / 64 * 64); };
    /* Few values: one row's chain, as few chunks a lane as some 768 lanes allow.  us at the chunks named, 64 rows of n:
     *     2048     1: 3.5   2: 3.8   4: 4.4        5376     1: 5.5   2: 6.0   3: 5.9
     *     8192     1: 5.9   2: 5.5   4: 5.7       16384     2: 7.9   3: 8.5   4: 7.5
     * and on both sides of the limit, f32 weights within 4 % of these:
     *     256 x 5376 (172032)  1: 6.9  2: 7.4  3: 7.2      333 x 5376 (223776)   1: 8.7  2: 9.1  3: 8.1
     *     512 x 2048 (131072)  1: 5.2  2: 5.5  4: 5.7      1024 x 2048 (262144)  1: 7.1  2: 6.7  4: 6.6
     *     333 x 4096 (170496)  1: 6.5  2: 6.1  4: 7.2      512 x 4096 (262144)   1: 7.3  2: 6.9  4: 7.9 (taken, the worst case) */
    if (rows * nc < 200000) {
        const int c = nc <= 768 ? 1 : nc <= 1536 ? 2 : 4;
        return BlockGeom{lanes(c), c, 0};
    }
    /* Many: as many chunks in flight a compute unit as registers hold, fewer a lane where they tie.  The waves are the kernel's with
     * bf16 weights (32, 28, 20 and 16 at 1 to 4 chunks a lane); f32 weights hold 32, 20, 16 to 20 and 16 and are as fast by the same
     * choice (2048 rows of 5376 22.6, 2560 13.9, 8192 24.6 us).  2048 rows, results as below:
     *     1024     1: 6.9   2: 6.3   3: 7.9   4: 9.4        5376     1: 28.1  2: 24.5  3: 20.8  4: 21.1
     *     2560     1: 14.8  2: 14.8  3: 14.1  4: 15.9       8192     1: 29.8  2: 24.2  3: 31.3  4: 23.4
     *     4096     1: 14.8  2: 12.9  3: 16.0  4: 12.0       16384 (1024 rows)   2: 33.4  3: 34.8  4: 25.4 */
    static const int kWaves[] = {0, 32, 28, 20, 16};
    int best = 4;
    int64_t most = 0;
    for (int c = 1; c <= 4; ++c) {
        const int64_t held = lanes(c) <= 1024 ? kWaves[c] / (lanes(c) / 64) * nc : 0;
        if (held > most) {
            most = held;
            best = c;
        }
    }
    /* From 2^20 chunks on, where two bf16 results fill the 32 MB of the XCDs' L2, results of every kind are written past the caches: alone
     * 2048 x 5376 24.2 -> 20.8 us; with a product of 2048 columns behind, whose weights come from HBM, 76.2 -> 73.3, int8 codes 55.3 ->
     * 52.4, one bf16 result 71.6 -> 70.4, f32 45.5 -> 44.3 (a pass over them behind).  It costs where that product's weights are
     * still in the 256 MB before HBM: 60.6 -> 71.5, and at 512 x 5376, which stays under the limit, 31.7 -> 38.4 (from HBM 41.9 -> 40.0). */
    return BlockGeom{lanes(best), best, rows * nc >= (1 << 20)};
}

int describe_block(const char* row, const RadArgs* a, char* buf, int len) {
    if (strcmp(row, "rmsnorm_block")) return -1;
    BlockPlan P{};
    const int rc = plan_block(a, &P);
    if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
    static const char* const kGate[] = {"none", "rows", "token"};
    static const char* const kCodes[] = {"none", "i8", "e4m3"};
    const BlockGeom g = block_geom(P.rows, P.n);
    snprintf(buf, (size_t)len, "arm=band op=rmsnorm_block x=%s w=%s rows=%lld n=%lld lanes=%d chunks=%d post=%d "
             "residual=%d gate=%s pre=%d residual_out=%d out=%s codes=%s", P.x_bf16 ? "bf16" : "f32",
             P.w_bf16 ? "bf16" : "f32", (long long)P.rows, (long long)P.n, g.lanes, g.chunks, P.w_post != nullptr,
             P.res != nullptr, kGate[P.gate_kind], P.w_pre != nullptr, P.res_out != nullptr,
             P.out ? (P.out_bf16 ? "bf16" : "f32") : "none", kCodes[P.codes]);
    return RAD_OK;
}

bool env_no_block() { static const bool v = getenv("R3D_NO_BLOCK_NORM") != nullptr; return v; }

}  // namespace r3d
