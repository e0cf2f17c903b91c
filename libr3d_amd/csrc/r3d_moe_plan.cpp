/* r3d_moe_plan.cpp -- host plan of moe_layer (see r3d_moe.h). */
#include "r3d_moe.h"

#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rad_plugin.h"
#include "r3d_act.h"
#include "r3d_operands.h"

namespace r3d {

/* The strides of an [E, rows, cols] operand, its last axis dense. */
static int planes_of(const RadTensor* t, int64_t E, int64_t rows, int64_t cols, int64_t* expert, int64_t* pitch) {
    if (t->rank != 3 || t->shape[0] != E || t->shape[1] != rows || t->shape[2] != cols) return RAD_E_SHAPE;
    if (t->stride[2] != 1) return RAD_E_STRIDE;
    *expert = t->stride[0];
    *pitch = t->stride[1];
    return pitch_ok(*expert) && pitch_ok(*pitch) ? RAD_OK : RAD_E_STRIDE;
}

/* A plane of codes and its scales. */
struct Experts {
    const RadTensor* w;
    const RadTensor* s;
    int64_t expert, pitch, s_expert, s_pitch, bytes, s_bytes;   /* bytes: of an expert's codes, and of its scales */
};

static int plan_experts(int enc, int64_t E, int64_t rows, int64_t cols, Experts* X) {
    static const uint32_t kType[] = {RAD_BF16, RAD_I8, RAD_FP4E2M1};
    if (X->w->dtype != kType[enc]) return RAD_E_DTYPE;
    if ((enc == MOE_BF16) != (X->s == nullptr)) return RAD_E_INVAL;
    if (X->s && X->s->dtype != (enc == MOE_I8 ? RAD_F32 : RAD_E8M0)) return RAD_E_DTYPE;
    int rc = planes_of(X->w, E, rows, cols, &X->expert, &X->pitch);
    if (rc) return rc;
    if (enc == MOE_FP4 && ((X->expert | X->pitch) & 1)) return RAD_E_STRIDE;      /* nibbles: whole bytes */
    X->expert = enc == MOE_BF16 ? 2 * X->expert : enc == MOE_FP4 ? X->expert / 2 : X->expert;
    X->pitch = enc == MOE_BF16 ? 2 * X->pitch : enc == MOE_FP4 ? X->pitch / 2 : X->pitch;
    const int64_t row = enc == MOE_BF16 ? 2 * cols : enc == MOE_FP4 ? cols / 2 : cols;
    /* 16 bytes a lane: whole pieces on their own alignment, an expert's plane under 32-bit offsets */
    if ((row | X->expert | X->pitch) & 15 || (uintptr_t)X->w->data & 15) return RAD_E_UNSUPPORTED;
    if (X->pitch > (int64_t(1) << 31) / rows || (rows - 1) * X->pitch + row > 0x7FFFFFFF) return RAD_E_UNSUPPORTED;
    X->bytes = (rows - 1) * X->pitch + row;
    if (enc == MOE_I8) {
        if (X->s->rank == 3) {                                       /* [E, rows, 1] */
            if (X->s->shape[0] != E || X->s->shape[1] != rows || X->s->shape[2] != 1) return RAD_E_SHAPE;
        } else if (X->s->rank != 2 || X->s->shape[0] != E || X->s->shape[1] != rows) {
            return RAD_E_SHAPE;
        }
        if (X->s->stride[1] != 1) return RAD_E_STRIDE;
        X->s_expert = X->s->stride[0];
        if (!pitch_ok(X->s_expert)) return RAD_E_STRIDE;
        X->s_bytes = 4 * rows;
    } else if (enc == MOE_FP4) {
        if ((rc = planes_of(X->s, E, rows, cols / 32, &X->s_expert, &X->s_pitch))) return rc;
        /* a load takes four scales, the plane's last four at most: rows that are apart, so that a plane has that many */
        if (X->s_pitch < cols / 32) return RAD_E_STRIDE;
        if (X->s_pitch > (int64_t(1) << 31) / rows) return RAD_E_UNSUPPORTED;
        X->s_bytes = (rows - 1) * X->s_pitch + cols / 32;
    }
    return RAD_OK;
}

int plan_moe(const RadArgs* a, MoePlan* P) {
    const RadTensor* x  = rad_arg_in(a, 0);
    const RadTensor* lg = rad_arg_in(a, 1);
    const RadTensor* y  = rad_arg_in(a, 6);
    const RadTensor* id = rad_arg_in(a, 7);
    const RadTensor* wt = rad_arg_in(a, 8);
    Experts up{rad_arg_in(a, 2), rad_arg_in(a, 3), 0, 0, 0, 0, 0, 0}, down{rad_arg_in(a, 4), rad_arg_in(a, 5), 0, 0, 0, 0, 0, 0};
    if (!x || !lg || !up.w || !down.w || !y) return RAD_E_INVAL;
    const char* dt = rad_args_gets(a, "dtype");
    P->enc = !dt ? -1 : !strcmp(dt, "bf16") ? MOE_BF16 : !strcmp(dt, "i8") ? MOE_I8 : !strcmp(dt, "mxfp4") ? MOE_FP4 : -1;
    if (P->enc < 0) return RAD_E_UNSUPPORTED;
    if (x->dtype != RAD_BF16 || (lg->dtype != RAD_F32 && lg->dtype != RAD_BF16) ||
        (y->dtype != RAD_F32 && y->dtype != RAD_BF16) || (id && id->dtype != RAD_I32) || (wt && wt->dtype != RAD_F32))
        return RAD_E_DTYPE;
    const char* act = rad_args_gets(a, "act");
    P->act = act ? act_by_name(act) : ACT_SILU;
    const char* score = rad_args_gets(a, "score");
    P->sigmoid = score && !strcmp(score, "sigmoid");
    if (P->act < 0 || (score && !P->sigmoid && strcmp(score, "softmax"))) return RAD_E_UNSUPPORTED;
    long long n = 0, f = 0, E = 0, k = 0, v = 0;
    if (!rad_args_geti(a, "n", &n) || !rad_args_geti(a, "f", &f) || !rad_args_geti(a, "E", &E) ||
        !rad_args_geti(a, "top_k", &k) || n <= 0 || f <= 0 || E <= 0 || k <= 0 || n > kDimMax || f > kDimMax || k > E)
        return RAD_E_SHAPE;
    if (E > kMoeMaxE || k > kMoeMaxK || n > kMoeMaxN || f > kMoeMaxF) return RAD_E_UNSUPPORTED;
    /* whole 16-byte pieces of codes (plan_experts), and 8 rows of an expert a wave */
    if ((n | f) & (P->enc == MOE_FP4 ? 31 : P->enc == MOE_I8 ? 15 : 7)) return RAD_E_UNSUPPORTED;
    const long long yn = rad_tensor_numel(y);
    if (yn <= 0 || yn % n) return RAD_E_SHAPE;
    const int64_t M = yn / n;
    if (M > kMoeMaxM) return RAD_E_UNSUPPORTED;
    int rc = rows_of(x, M, n, &P->x_pitch);
    if (!rc) rc = rows_of(lg, M, E, &P->l_pitch);
    if (!rc) rc = rows_of(y, M, n, &P->y_pitch);
    if (!rc && id) rc = rows_of(id, M, k, &P->i_pitch);
    if (!rc && wt) rc = rows_of(wt, M, k, &P->w_pitch);
    if (!rc) rc = plan_experts(P->enc, E, 2 * f, n, &up);
    if (!rc) rc = plan_experts(P->enc, E, n, f, &down);
    if (rc) return rc;
    if (M > 1 && (P->y_pitch < n || (id && P->i_pitch < k) || (wt && P->w_pitch < k))) return RAD_E_STRIDE;
    for (const RadTensor* t : {x, lg, up.s, down.s, y, id, wt})
        if (misaligned(t)) return RAD_E_STRIDE;
    P->x_pitch *= 2;
    if ((uintptr_t)x->data & 15 || (M > 1 && (P->x_pitch & 15 || P->x_pitch > (1 << 24)))) return RAD_E_UNSUPPORTED;
    if (M == 1) P->x_pitch = 2 * n;                             /* a single row has no next one */
    /* ids and weights are written while other workgroups still read x and the logits; y when nobody does */
    const Span outs[3] = {{y->data, M, n, P->y_pitch, elt_bytes(y->dtype)},
                          {id ? id->data : nullptr, M, k, P->i_pitch, 4}, {wt ? wt->data : nullptr, M, k, P->w_pitch, 4}};
    const Span ins[2] = {{x->data, M, n, P->x_pitch / 2, 2}, {lg->data, M, E, P->l_pitch, elt_bytes(lg->dtype)}};
    for (int i = 0; i < 3; ++i) {
        if (!outs[i].data) continue;
        for (int j = 0; j < i; ++j)
            if (outs[j].data && spans_meet(outs[i], outs[j])) return RAD_E_INVAL;
        /* the planes and their scales, from an expert's first byte to the last one's last */
        for (const Experts* X : {&up, &down})
            if (spans_meet(outs[i], Span{X->w->data, 1, (E - 1) * X->expert + X->bytes, 0, 1}) ||
                (X->s && spans_meet(outs[i], Span{X->s->data, 1, (E - 1) * X->s_expert * elt_bytes(X->s->dtype) + X->s_bytes, 0, 1})))
                return RAD_E_INVAL;
        if (i == 0) continue;
        for (const Span& in : ins)
            if (spans_meet(outs[i], in)) return RAD_E_INVAL;
    }
    P->x = (const uint8_t*)x->data;
    P->logits = (const uint8_t*)lg->data;
    P->l_bf16 = lg->dtype == RAD_BF16;
    P->gu = (const uint8_t*)up.w->data;
    P->gus = up.s ? (const uint8_t*)up.s->data : nullptr;
    P->dn = (const uint8_t*)down.w->data;
    P->dns = down.s ? (const uint8_t*)down.s->data : nullptr;
    P->gu_expert = up.expert;
    P->gu_pitch = up.pitch;
    P->gus_expert = up.s_expert;
    P->gus_pitch = up.s_pitch;
    P->dn_expert = down.expert;
    P->dn_pitch = down.pitch;
    P->dns_expert = down.s_expert;
    P->dns_pitch = down.s_pitch;
    P->y = (uint8_t*)y->data;
    P->y_bf16 = y->dtype == RAD_BF16;
    P->ids = id ? (int32_t*)id->data : nullptr;
    P->weights = wt ? (float*)wt->data : nullptr;
    P->M = M;
    P->n = n;
    P->f = f;
    P->E = E;
    P->top_k = k;
    P->renorm = !rad_args_geti(a, "renorm", &v) || v != 0;
    P->weight_scale = (float)rad_args_getf_or(a, "weight_scale", 1.0);
    return RAD_OK;
}

/* LDS a workgroup: 160 KB, less its tables, the waves' shared units and int8's scales */
static int64_t moe_lds(const MoePlan& P, int ct, bool up) {
    return 160 * 1024 - (up ? 21 : 5) * 1024 - 8 * 1024 * ct - (P.enc == MOE_I8 ? 8 * 1024 : 0);
}

/* The tokens of a job, `row` bytes of LDS each: a job's part of the planes is read once for all of them, 8 at most, 16 where
 * experts have more than 6 tokens (crowded) and LDS holds 16.  us of a call of 2048 x 1024, 64 experts top 8, with 16 and 8 in the
 * gate and up product:
 *     M = 24 to 48 (3 to 6 tokens)   mxfp4 59 to 66, 59 to 64      i8 79 to 90, 78 to 88      bf16 135 to 153, 134 to 148
 *     M = 56 and 64                  mxfp4 67 and 70, 68 and 74    i8 92 and 100, 95 and 104  bf16 154 and 161, 158 and 180
 * In the down product, whose tokens are in three parts each, the second eight cost mxfp4 and int8 more matrix cycles (and
 * registers) than a second read takes.  M = 64, with 8 and 16:
 *     2048 x 1024, 16 experts top 4  mxfp4 42.4, 54.1              i8 48.9, 53.7              bf16 62.4, 62.6
 *     2048 x 768, 64 experts top 8   mxfp4 60.7, 78.4              i8 73.2, 74.8              bf16 121, 112
 *     4096 x 1024, 8 experts top 8   mxfp4 87, 96                  i8 124, 118                bf16 243, 210 */
static bool moe_tiles(const MoePlan& P, bool up, int64_t row, bool crowded, MoeTiles* t) {
    t->ct = crowded && (up || P.enc == MOE_BF16) && moe_lds(P, 2, up) / row >= 16 ? 2 : 1;
    int64_t rows = moe_lds(P, t->ct, up) / row;
    const int64_t pairs = P.M * P.top_k, most = pairs < 64 ? pairs : 64;      /* rows whose tokens lie in a wave's lanes */
    if (rows > most) rows = most;
    t->rows = (int)rows;
    t->width = rows < 8 * t->ct ? (int)rows : 8 * t->ct;
    return rows >= 1;
}

bool moe_geom(const MoePlan& P, int ncu, MoeGeom* g) {
    if (ncu <= 0 || ncu > kMoeMaxBlocks) ncu = kMoeMaxBlocks;
    g->blocks = ncu;
    /* experts that someone chose, and their tokens, of choices spread evenly */
    const double read = (double)P.E * (1.0 - pow(1.0 - (double)P.top_k / (double)P.E, (double)P.M));
    const double tokens = (double)(P.M * P.top_k) / read;
    if (!moe_tiles(P, true, (2 * P.n + 1023) / 1024 * 1024 + 64, tokens > 6, &g->up)) return false;
    /* LDS holds few tokens of a long row of h, and the planes would be read again for every few: the row may be cut into parts, a
     * launch each, that add to the slots' sums.  A launch costs some 6 us, a read goes at 4.5 TB/s.  4096 x 14336, 8 experts top 2, us in
     * 1, 2, 3, 4 and 6 parts: M = 64 mxfp4 760, 426, 397, 412, 418, i8 1167, 698, 632, 602, 592; M = 16 mxfp4 238, 177, 172, 179, 187;
     * M = 1 46, 53, 60, 65, 79.  Of 28 such calls the parts taken were 6 % from the best at most.  More than 8 tokens are not worth
     * another launch: bf16 4096 x 2048, M = 64, 150 in one, 157 in two with 16; x 3584 261 and 267. */
    const int64_t span = moe_span(P.enc), spans = (P.f + span - 1) / span;
    const double plane = (double)P.n * (double)P.f * (P.enc == MOE_BF16 ? 2.0 : P.enc == MOE_I8 ? 1.0 : 0.53);
    double best = 0.0;
    g->parts = 0;
    for (int64_t parts = 1; parts <= 16 && parts <= spans && (g->parts == 0 || g->down.width < 8); ++parts) {
        const int64_t each = (spans + parts - 1) / parts, K = parts == 1 ? P.f : each * span;
        MoeTiles t;
        if (!moe_tiles(P, false, 3 * ((2 * K + 1023) / 1024 * 1024) + 64, tokens > 6, &t)) continue;
        const double reads = tokens > t.width ? (tokens + 0.5 * (t.width - 1)) / t.width : 1.0;
        const double us = 6.0 * (double)parts + reads * read * plane / 4.5e6;
        if (g->parts > 0 && us >= best) continue;
        best = us;
        g->down = t;
        g->parts = (int)((spans + each - 1) / each);
        g->spans = each;
    }
    return g->parts > 0;
}

/* four bytes a value; where y is f32 six are asked for, which keeps the hook's answers what they were */
int64_t moe_h_bytes(const MoePlan& P) {
    return (P.M * P.top_k * P.f * (P.y_bf16 ? 4 : 6) + 15) / 16 * 16;
}

int64_t moe_scratch(const MoePlan& P) {
    return (int64_t)sizeof(MoeTable) + moe_h_bytes(P) + P.M * P.top_k * P.n * 4;
}

int64_t moe_scratch_bytes(const RadArgs* a) {
    MoePlan P{};
    if (plan_moe(a, &P) == RAD_OK) return moe_scratch(P);
    long long n = 0, f = 0, k = 0, M = 0;                       /* not a whole call yet: y in f32 */
    if (!rad_args_geti(a, "n", &n) || !rad_args_geti(a, "f", &f) || !rad_args_geti(a, "top_k", &k) || n <= 0 || f <= 0 ||
        k <= 0 || n > kMoeMaxN || f > kMoeMaxF || k > kMoeMaxK)
        return 0;
    const RadTensor* y = rad_arg_in(a, 6);
    if (y) M = rad_tensor_numel(y) / n;
    else if (!rad_args_geti(a, "M", &M)) M = kMoeMaxM;
    if (M <= 0 || M > kMoeMaxM) return 0;
    P.M = M;
    P.n = n;
    P.f = f;
    P.top_k = k;
    P.y_bf16 = 0;
    return moe_scratch(P);
}

int describe_moe(const char* row, const RadArgs* a, char* buf, int len) {
    if (strcmp(row, "moe_layer")) return -1;
    MoePlan P{};
    const int rc = plan_moe(a, &P);
    if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
    if (!a->scratch || (uintptr_t)a->scratch & 15 || a->scratch_bytes < moe_scratch(P)) {
        snprintf(buf, (size_t)len, "refused rc=%d (scratch)", RAD_E_UNSUPPORTED);
        return RAD_E_UNSUPPORTED;
    }
    static const char* const kEnc[] = {"bf16", "i8", "mxfp4"};
    MoeGeom g;
    if (!moe_geom(P, 256, &g)) {
        snprintf(buf, (size_t)len, "refused rc=%d (LDS)", RAD_E_UNSUPPORTED);
        return RAD_E_UNSUPPORTED;
    }
    snprintf(buf, (size_t)len, "arm=moe enc=%s M=%lld n=%lld f=%lld E=%lld top_k=%lld score=%s renorm=%d act=%d y=%s up_ct=%d "
             "up_width=%d up_rows=%d down_ct=%d down_width=%d down_rows=%d parts=%d blocks=%lld",
             kEnc[P.enc], (long long)P.M, (long long)P.n, (long long)P.f,
             (long long)P.E, (long long)P.top_k, P.sigmoid ? "sigmoid" : "softmax", P.renorm, P.act,
             P.y_bf16 ? "bf16" : "f32", g.up.ct, g.up.width, g.up.rows, g.down.ct, g.down.width, g.down.rows, g.parts, (long long)g.blocks);
    return RAD_OK;
}

bool env_no_moe() { static const bool v = getenv("R3D_NO_MOE") != nullptr; return v; }

}  // namespace r3d
