/* r3d_sample_plan.cpp -- host plan of the sample_logits row (see r3d_sample.h). */
#include "r3d_sample.h"

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rad_plugin.h"

namespace r3d {

/* One element a row: rank 1 [M] or rank 2 [M, 1]; an input's stride may be 0 (one for all). */
static int column(const RadTensor* t, uint32_t dtype, int64_t M, bool out, int64_t* stride) {
    if (!t) return RAD_OK;
    if (t->dtype != dtype) return RAD_E_DTYPE;
    if ((t->rank != 1 && t->rank != 2) || (t->rank == 2 && t->shape[1] != 1) || t->shape[0] < M)
        return RAD_E_SHAPE;
    *stride = t->stride[0];
    if (*stride < 0 || *stride > ((int64_t)1 << 40) || (out && M > 1 && *stride < 1)) return RAD_E_STRIDE;
    return (uintptr_t)t->data & 3 ? RAD_E_STRIDE : RAD_OK;
}

int64_t sample_scratch_bytes(int64_t M, int64_t V) {
    const int64_t segs = (V + kSampleSeg - 1) / kSampleSeg;
    return M * ((int64_t)sizeof(SampleRow) + segs * (8 + 4 * 16 + 4 * kSampleSegChunks));
}

int plan_sample(const RadArgs* a, SamplePlan* P) {
    const RadTensor* x = rad_arg_in(a, 0);
    const RadTensor* u = rad_arg_in(a, 1);
    const RadTensor* T = rad_arg_in(a, 2);
    const RadTensor* k = rad_arg_in(a, 3);
    const RadTensor* p = rad_arg_in(a, 4);
    const RadTensor* m = rad_arg_in(a, 5);
    const RadTensor* tok = rad_arg_in(a, 6);
    const RadTensor* prob = rad_arg_in(a, 7);
    if (!x || !u || !tok) return RAD_E_INVAL;
    if (x->dtype != RAD_F32 && x->dtype != RAD_BF16) return RAD_E_DTYPE;
    const char* dt = rad_args_gets(a, "dtype");                /* names the logits' type, if given */
    if (dt && strcmp(dt, x->dtype == RAD_BF16 ? "bf16" : "f32") != 0) return RAD_E_DTYPE;
    long long V = 0;
    if (!rad_args_geti(a, "n_vocab", &V) || V <= 0 || V > kSampleMaxVocab) return RAD_E_SHAPE;
    const long long xn = rad_tensor_numel(x);
    if (xn <= 0 || xn % V || xn / V > 65535) return RAD_E_SHAPE;
    const int64_t M = xn / V;
    if (x->rank < 1 || x->shape[x->rank - 1] != V) return RAD_E_SHAPE;
    if (x->stride[x->rank - 1] != 1) return RAD_E_STRIDE;
    for (int i = 0; i + 2 < (int)x->rank; ++i) {
        int64_t span = 0;
        if (__builtin_mul_overflow(x->shape[i + 1], x->stride[i + 1], &span) || x->stride[i] != span)
            return RAD_E_STRIDE;
    }
    P->pitch = x->rank >= 2 ? x->stride[x->rank - 2] : V;
    if (P->pitch < 0 || P->pitch > ((int64_t)1 << 40)) return RAD_E_STRIDE;
    if ((uintptr_t)x->data & (x->dtype == RAD_BF16 ? 1 : 3)) return RAD_E_STRIDE;
    int rc = column(u, RAD_F32, M, false, &P->u_stride);
    if (!rc) rc = column(T, RAD_F32, M, false, &P->t_stride);
    if (!rc) rc = column(k, RAD_I32, M, false, &P->k_stride);
    if (!rc) rc = column(p, RAD_F32, M, false, &P->p_stride);
    if (!rc) rc = column(m, RAD_F32, M, false, &P->m_stride);
    if (!rc) rc = column(tok, RAD_I32, M, true, &P->token_stride);
    if (!rc) rc = column(prob, RAD_F32, M, true, &P->prob_stride);
    if (rc) return rc;
    P->logits = (const uint8_t*)x->data;
    P->u = (const float*)u->data;
    P->temperature = T ? (const float*)T->data : nullptr;
    P->top_k = k ? (const int*)k->data : nullptr;
    P->top_p = p ? (const float*)p->data : nullptr;
    P->min_p = m ? (const float*)m->data : nullptr;
    P->token = (int*)tok->data;
    P->prob = prob ? (float*)prob->data : nullptr;
    P->bf16 = x->dtype == RAD_BF16;
    P->M = M;
    P->V = V;
    return RAD_OK;
}

int64_t sample_hook_bytes(const RadArgs* a) {
    long long V = 0, M = 0;
    if (!rad_args_geti(a, "n_vocab", &V) || V <= 0 || V > kSampleMaxVocab) return 0;
    const RadTensor* x = rad_arg_in(a, 0);
    if (x) M = rad_tensor_numel(x) / V;
    else if (!rad_args_geti(a, "M", &M)) return 0;
    return M > 0 && M <= 65535 ? sample_scratch_bytes(M, V) : 0;
}

int describe_sample(const char* row, const RadArgs* a, char* buf, int len) {
    if (strcmp(row, "sample_logits") != 0) return -1;
    SamplePlan P{};
    const int rc = plan_sample(a, &P);
    if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
    snprintf(buf, (size_t)len, "arm=sample logits=%s M=%lld V=%lld segs=%lld temperature=%d top_k=%d "
             "top_p=%d min_p=%d prob=%d scratch=%lld", P.bf16 ? "bf16" : "f32", (long long)P.M,
             (long long)P.V, (long long)((P.V + kSampleSeg - 1) / kSampleSeg), P.temperature != nullptr,
             P.top_k != nullptr, P.top_p != nullptr, P.min_p != nullptr, P.prob != nullptr,
             (long long)sample_scratch_bytes(P.M, P.V));
    return RAD_OK;
}

bool env_no_sample() { static const bool v = getenv("R3D_NO_SAMPLE") != nullptr; return v; }

}  // namespace r3d
