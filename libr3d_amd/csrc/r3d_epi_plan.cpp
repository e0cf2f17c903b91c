/* r3d_epi_plan.cpp -- host plan of gemm_nt_epi (see r3d_epi.h). */
#include "r3d_epi.h"

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rad_plugin.h"
#include "r3d_act.h"
#include "r3d_operands.h"
#include "r3d_plan.h"

namespace r3d {

/* Bases, pitches and K that the 16-byte kernels take, from their bytes. */
static void epi_alignment(I8Plan* p) {
    p->chain = 1;
    p->ua = (p->K & 15) || (((uintptr_t)p->A | (uintptr_t)p->B) & 15) || ((p->a_pitch | p->b_pitch) & 15) ||
            p->a_pitch > (1 << 22) || p->b_pitch > (1 << 22);
    p->off = (((uintptr_t)p->A | (uintptr_t)p->B) & 127) || ((p->a_pitch | p->b_pitch) & 127);
}

int plan_epi(const RadArgs* a, bool bf16, EpiPlan* P) {
    const RadTensor* A  = rad_arg_in(a, 0);
    const RadTensor* AS = rad_arg_in(a, 1);
    const RadTensor* B  = rad_arg_in(a, 2);
    const RadTensor* BS = rad_arg_in(a, 3);
    const RadTensor* C  = rad_arg_in(a, 4);
    const RadTensor* R  = rad_arg_in(a, 5);
    const RadTensor* Y  = rad_arg_in(a, 6);
    if (!A || !B || !Y || (!bf16 && (!AS || !BS))) return RAD_E_INVAL;
    if (bf16 && (AS || BS)) return RAD_E_INVAL;                 /* bf16 operands have no scales */
    const char* dtype = rad_args_gets(a, "dtype");
    if (!dtype || strcmp(dtype, bf16 ? "bf16" : "i8a8") != 0) return RAD_E_UNSUPPORTED;
    const uint32_t want = bf16 ? RAD_BF16 : RAD_I8;
    if (A->dtype != want || B->dtype != want) return RAD_E_DTYPE;
    for (const RadTensor* t : {C, R, Y})
        if (t && t->dtype != RAD_F32 && t->dtype != RAD_BF16) return RAD_E_DTYPE;
    const char* act = rad_args_gets(a, "act");
    P->act = act ? act_by_name(act) : ACT_NONE;
    if (P->act < 0) return RAD_E_UNSUPPORTED;
    long long N = 0, K = 0;
    if (!rad_args_geti(a, "N", &N) || !rad_args_geti(a, "K", &K)) return RAD_E_SHAPE;
    if (N <= 0 || K <= 0 || N > kDimMax) return RAD_E_SHAPE;
    if (K > (bf16 ? kEpiMaxK : kI8MaxK)) return RAD_E_UNSUPPORTED;
    const long long yn = rad_tensor_numel(Y);
    if (yn <= 0 || yn % N) return RAD_E_SHAPE;
    const int64_t M = yn / N;
    if (M > kDimMax) return RAD_E_SHAPE;
    I8Plan& p = P->p;
    int rc = rows_of(A, M, K, &p.a_pitch);
    if (!rc) rc = rows_of(B, N, K, &p.b_pitch);
    if (!rc) rc = rows_of(Y, M, N, &p.y_pitch);
    if (!rc && R) rc = rows_of(R, M, N, &P->r_pitch);
    if (!rc && !bf16) {
        rc = scale_column(AS, M, &p.sa_stride);
        if (!rc) rc = scale_column(BS, N, &p.sb_stride);
        if (rc == RAD_E_UNSUPPORTED) rc = RAD_E_DTYPE;
    }
    if (rc) return rc;
    if (C) {
        if (C->rank != 1 || C->shape[0] != N) return RAD_E_SHAPE;
        P->bias_stride = C->stride[0];
        if (!pitch_ok(P->bias_stride)) return RAD_E_STRIDE;
    }
    if (p.y_pitch < N && M > 1) return RAD_E_STRIDE;            /* rows of y overlap */
    for (const RadTensor* t : {A, AS, B, BS, C, R, Y})
        if (misaligned(t)) return RAD_E_STRIDE;
    /* y may be the residual itself; anything else that overlaps it would be read after it is written */
    const Span y{Y->data, M, N, p.y_pitch, elt_bytes(Y->dtype)};
    if (R && spans_clash(y, Span{R->data, M, N, P->r_pitch, elt_bytes(R->dtype)})) return RAD_E_INVAL;
    const int e = bf16 ? 2 : 1;
    if (spans_meet(y, Span{A->data, M, K, p.a_pitch, e}) || spans_meet(y, Span{B->data, N, K, p.b_pitch, e}) ||
        (C && spans_meet(y, Span{C->data, N, 1, P->bias_stride, elt_bytes(C->dtype)})) ||
        (AS && spans_meet(y, Span{AS->data, M, 1, p.sa_stride, 4})) || (BS && spans_meet(y, Span{BS->data, N, 1, p.sb_stride, 4})))
        return RAD_E_INVAL;
    p.a_pitch *= e;
    p.b_pitch *= e;
    /* every kernel's least: 16 rows under 32-bit offsets */
    if ((M > 1 && p.a_pitch > (1 << 26)) || (N > 1 && p.b_pitch > (1 << 26))) return RAD_E_UNSUPPORTED;
    if (M == 1 && p.a_pitch > (1 << 22)) p.a_pitch = e * K;     /* a single row has no next one */
    if (N == 1 && p.b_pitch > (1 << 22)) p.b_pitch = e * K;
    p.A = (const uint8_t*)A->data;
    p.B = (const uint8_t*)B->data;
    p.SA = bf16 ? nullptr : (const float*)AS->data;
    p.SB = bf16 ? nullptr : (const float*)BS->data;
    p.Y = (uint16_t*)Y->data;
    p.M = M;
    p.N = N;
    p.K = e * K;
    epi_alignment(&p);
    if (p.ua && M > 65535 * 32) return RAD_E_UNSUPPORTED;      /* its grid's second axis */
    P->bf16 = bf16;
    P->K = K;
    P->bias = C ? C->data : nullptr;
    P->res = R ? R->data : nullptr;
    P->bias_bf16 = C && C->dtype == RAD_BF16;
    P->res_bf16 = R && R->dtype == RAD_BF16;
    P->y_bf16 = Y->dtype == RAD_BF16;
    return RAD_OK;
}

int64_t epi_scratch_bytes(const RadArgs* a, bool bf16, int ncu) {
    EpiPlan P{};
    if (plan_epi(a, bf16, &P) != RAD_OK) {
        /* not a whole call yet: dense operands on lines */
        long long N = 0, K = 0, M = 0;
        P = EpiPlan{};
        if (!rad_args_geti(a, "N", &N) || !rad_args_geti(a, "K", &K) || N <= 0 || K <= 0 || N > kDimMax ||
            K > (bf16 ? kEpiMaxK : kI8MaxK))
            return 0;
        const RadTensor* Y = rad_arg_in(a, 6);
        if (Y) M = rad_tensor_numel(Y) / N;
        else if (!rad_args_geti(a, "M", &M)) M = 128;
        if (M <= 0 || M > kDimMax) return 0;
        P.p.M = M;
        P.p.N = N;
        P.p.K = P.p.a_pitch = P.p.b_pitch = (bf16 ? 2 : 1) * K;
        epi_alignment(&P.p);
    }
    return i8_planes_bytes(P.p, ncu);
}

int describe_epi(const char* row, const RadArgs* a, char* buf, int len) {
    const bool bf16 = !strcmp(row, "gemm_nt_epi_bf16");
    if (!bf16 && strcmp(row, "gemm_nt_epi_i8a8")) return -1;
    EpiPlan P{};
    const int rc = plan_epi(a, bf16, &P);
    if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
    I8Geom g;
    const bool sc = a->scratch && ((uintptr_t)a->scratch & 15) == 0;
    i8_geom(P.p, 256, sc ? a->scratch_bytes : 0, &g);
    static const char* kArm[] = {"any", "gemv", "tile"};
    snprintf(buf, (size_t)len, "arm=%s enc=%s M=%lld N=%lld K=%lld act=%d bias=%d residual=%d y=%s bn=%d bm=%d "
             "tiles=%lld kc=%d per=%d waves=%d blocks=%lld", kArm[g.arm], bf16 ? "bf16" : "i8a8", (long long)P.p.M,
             (long long)P.p.N, (long long)P.K, P.act, P.bias != nullptr, P.res != nullptr, P.y_bf16 ? "bf16" : "f32",
             g.bn, g.bm, (long long)g.tiles, g.kc, g.per, g.waves, (long long)g.blocks);
    return RAD_OK;
}

bool env_no_epi() { static const bool v = getenv("R3D_NO_EPI") != nullptr; return v; }

}  // namespace r3d
