/* r3d_i8_plan.cpp -- host plans of the int8 rows (see r3d_i8.h). */
#include "r3d_i8.h"

#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rad_plugin.h"
#include "r3d_operands.h"
#include "r3d_plan.h"

namespace r3d {

int plan_i8(const RadArgs* a, int64_t m_max, I8Plan* P) {
    const RadTensor* A  = rad_arg_in(a, 0);
    const RadTensor* AS = rad_arg_in(a, 1);
    const RadTensor* B  = rad_arg_in(a, 2);
    const RadTensor* BS = rad_arg_in(a, 3);
    const RadTensor* Y  = rad_arg_in(a, 4);
    if (!A || !AS || !B || !BS || !Y) return RAD_E_UNSUPPORTED;
    if (rad_arg_in(a, 5) || rad_arg_in(a, 6)) return RAD_E_UNSUPPORTED;   /* symmetric codes only */
    const char* dtype = rad_args_gets(a, "dtype");
    if (!dtype || strcmp(dtype, "i8a8") != 0) return RAD_E_UNSUPPORTED;
    long long v = 0;
    if (rad_args_geti(a, "pb1", &v) && v > 0) return RAD_E_UNSUPPORTED;
    if (rad_args_geti(a, "pb2", &v) && v > 0) return RAD_E_UNSUPPORTED;
    if (A->dtype != RAD_I8 || B->dtype != RAD_I8 || Y->dtype != RAD_BF16) return RAD_E_UNSUPPORTED;
    long long N = 0, K = 0;
    if (!rad_args_geti(a, "N", &N) || !rad_args_geti(a, "K", &K)) return RAD_E_SHAPE;
    if (N <= 0 || K <= 0 || N > kDimMax) return RAD_E_SHAPE;
    if (K > kI8MaxK) return RAD_E_UNSUPPORTED;                  /* the sum could leave i32 */
    const long long yn = rad_tensor_numel(Y);
    if (yn <= 0 || yn % N) return RAD_E_SHAPE;
    const int64_t M = yn / N;
    if (M > kDimMax) return RAD_E_SHAPE;
    if (m_max > 0 && M > m_max) return RAD_E_UNSUPPORTED;       /* the band's own bound */
    /* one scale a row of K: a group that says otherwise contradicts the scales */
    if (rad_args_geti(a, "group", &v) && v > 0 && v != K) return RAD_E_SHAPE;
    int rc = scale_column(AS, M, &P->sa_stride);
    if (!rc) rc = scale_column(BS, N, &P->sb_stride);
    if (!rc) rc = rows_of(A, M, K, &P->a_pitch);
    if (!rc) rc = rows_of(B, N, K, &P->b_pitch);
    if (!rc) rc = rows_of(Y, M, N, &P->y_pitch);
    if (rc) return rc;
    if (P->y_pitch < N && M > 1) return RAD_E_STRIDE;           /* rows of Y overlap */
    if (((uintptr_t)AS->data | (uintptr_t)BS->data) & 3 || (uintptr_t)Y->data & 1)
        return RAD_E_STRIDE;
    /* every kernel's least: 16 rows under 32-bit offsets */
    if ((M > 1 && P->a_pitch > (1 << 26)) || (N > 1 && P->b_pitch > (1 << 26)))
        return RAD_E_UNSUPPORTED;
    P->A = (const uint8_t*)A->data;
    P->SA = (const float*)AS->data;
    P->B = (const uint8_t*)B->data;
    P->SB = (const float*)BS->data;
    P->Y = (uint16_t*)Y->data;
    P->M = M;
    P->N = N;
    P->K = K;
    /* the fast kernels move 16 bytes a lane and walk 256 rows with 32-bit offsets */
    P->ua = (K & 15) || (((uintptr_t)P->A | (uintptr_t)P->B) & 15) ||
            ((P->a_pitch | P->b_pitch) & 15) || P->a_pitch > (1 << 22) || P->b_pitch > (1 << 22);
    P->off = (((uintptr_t)P->A | (uintptr_t)P->B) & 127) || ((P->a_pitch | P->b_pitch) & 127);
    if (P->ua && M > 65535 * 32) return RAD_E_UNSUPPORTED;     /* its grid's second axis */
    return RAD_OK;
}

/* What a launch of a tile takes, in ns:
 *     a + sqrt(work^2 + stream^2) + the planes and their sum
 *     work: ceil(units / ncu) * q * steps a unit; rows that begin inside lines (a base or a pitch off 128):
 *           * off / 100 (4000 launches of each tile over 22167 such shapes)
 *     stream: the weights at 6.12 TB/s, or at what the units in flight ask for, `one` bytes a us each
 *           with one tile of tokens, `more` where tiles of tokens share them in L2
 * Least squares over 5230 shapes (M 9..2048, N and K 512..21504) and 4 to 40 launches of each.  The pick is
 * 1.6 % slower than the best launch on average (geometric), 7 % at the ninth decile; with the larger of
 * work and stream in place of the root 2.8 % and 11 %.
 * Powers of two alone leave compute units idle at common widths: tiles of 96 and 192 tokens are taken by a
 * fifth of the shapes, 8 % faster there (512 x 5376 x 5376 27.5 -> 23.6 us, 1024 x 5376 x 5376 49.9 -> 41.8).
 * Tiles of 32 weight rows cover few tokens in as many workgroups as two planes of 64 (13 x 8192 x 5376 12.8
 * -> 10.3 us, 12 x 5376 x 4096 9.7 -> 7.9). */
struct I8Cost {
    int bn, bm, resident;    /* workgroups a compute unit holds (LDS) */
    int a, q, off, one, more;
};
constexpr int kI8Any = 1000000;                                     /* a unit's rate never the bound */
static const I8Cost kI8Cost[I8_TILES] = {
    {256, 256, 1, 8244, 1034, 121, kI8Any, kI8Any},
    {128, 256, 1, 4783,  852, 122, kI8Any, kI8Any},
    {128, 192, 1, 3379,  776, 122, kI8Any,  21400},
    {128, 128, 1, 4258,  445, 110, kI8Any, kI8Any},
    {128,  96, 1, 3856,  422, 111, kI8Any, kI8Any},
    {128,  64, 1, 3480,  343, 109, kI8Any, kI8Any},
    { 64,  64, 2, 3242,  226, 116, kI8Any, kI8Any},
    { 64,  32, 2, 3052,  175, 121, kI8Any, kI8Any},
    { 32,  32, 2, 3319,  134, 130,  65500,  26700},
    { 32,  16, 3, 3088,   96, 130,  43100,  19400},
};

static double i8_tile_ns(const I8Cost& c, const I8Plan& P, int64_t per, int64_t kc, int ncu) {
    const int64_t M = P.M, N = P.N, gm = (M + c.bm - 1) / c.bm, units = (N + c.bn - 1) / c.bn * gm * kc;
    const double work = (double)((units + ncu - 1) / ncu) * c.q * per * (P.off ? c.off / 100.0 : 1.0);
    const int64_t busy = units < c.resident * ncu ? units : c.resident * ncu;
    int64_t rate = busy * (gm == 1 ? c.one : c.more);               /* bytes a us */
    if (rate > 6120000) rate = 6120000;
    const double stream = (double)N * P.K * 1000 / rate;
    return c.a + sqrt(work * work + stream * stream) + (kc > 1 ? 2260 + 1.83e-3 * kc * M * N : 0.0);
}

/* The GEMV's time in the same terms, work growing with the tokens: over 13494 shapes of 1..8 tokens the
 * cheaper of it and a tile is 1.0 % slower than the best launch, the GEMV wherever it fits 3.4 % (8 x 8192 x
 * 5376 12.1 -> 10.4 us on tiles of 32 rows; up to 3 tokens it is the faster one nearly everywhere).
 * gemm_nt_epi counts one thing more: with a workgroup a compute unit or less, a wave's chain of `per` lines may be longer than
 * all that.  us by the GEMV and on tiles, 128 rows of 10752, 21504 and 43008 bytes: 1 token 5.7, 6.9; 8.4, 7.8; 13.4, 8.6; 2 tokens 6.0,
 * 7.1; 9.0, 7.6; 4 tokens 6.6, 7.2 (past that its LDS holds no more tokens); 1024 rows 1 token 6.2, 7.6; 8.7, 9.4; 13.7, 12.3.  Of 24 such
 * shapes, 128 to 1024 rows, bf16 and int8, at 1, 2, 4 and 8 tokens each takes its faster one, ties within 2 % aside. */
static double i8_gemv_ns(const I8Plan& P, int ncu, const I8Geom& g) {
    const double lines = (double)((P.N + 7) / 8) * ((P.K + 127) / 128) / ncu;
    const double chain = P.chain && g.blocks <= ncu ? 165.0 * (1.0 + 0.06 * P.M) * g.per : 0.0;
    const double work = fmax(11.8 * (1.0 + 0.0841 * P.M) * lines, chain);
    const double stream = (double)P.N * P.K * 1000 / 6120000 * (P.off ? 1.3 : 1.0);
    return 3610 + 32 * P.M + sqrt(work * work + stream * stream);
}

constexpr int64_t kI8MaxPlanes = (int64_t)1 << 28;                 /* bytes of planes, at most */

void i8_geom(const I8Plan& P, int ncu, int64_t scratch, I8Geom* g) {
    *g = I8Geom{};
    if (P.ua) return;
    if (ncu <= 0) ncu = 256;
    const int64_t steps = (P.K + 127) / 128;
    double best = 0;
    if (P.M <= 8 && P.M * i8_gemv_row(P.K) <= kI8GemvLds && !env_no_i8_dec()) {
        /* 8 weight rows a wave; K over waves until about 1600 of them stream (the K chunks of a row
         * block are waves of one workgroup), two lines a wave at least */
        const int64_t rows = (P.N + 7) / 8;
        int kc = 1;
        while (kc < 8 && rows * kc < 1600 && steps / (2 * kc) >= 2) kc *= 2;
        g->arm = I8_GEMV;
        g->bn = 8;
        g->bm = 8;
        g->tiles = rows;
        g->kc = kc;
        g->per = (int)((steps + kc - 1) / kc);
        g->waves = kc > 4 ? kc : 4;
        g->blocks = (rows + g->waves / kc - 1) / (g->waves / kc);
        best = i8_gemv_ns(P, ncu, *g);
    }
    for (int t = 0; t < I8_TILES; ++t) {
        const I8Cost& c = kI8Cost[t];
        const int64_t tiles = (P.N + c.bn - 1) / c.bn * ((P.M + c.bm - 1) / c.bm);
        for (int64_t kc : {1, 2, 3, 4, 5, 6, 8, 12, 16, 24}) {
            if (kc > 1 && steps / kc < 3) break;
            const int64_t per = (steps + kc - 1) / kc;
            if ((steps + per - 1) / per != kc || tiles * kc > 0x7FFFFF) continue;      /* 2^32 lanes a launch */
            if (kc > 1 && (P.M > 65535 || tiles * kc > 4 * ncu || kc * P.M * P.N * 4 > scratch)) break;
            const double ns = i8_tile_ns(c, P, per, kc, ncu);
            if (best > 0 && ns >= best) continue;
            best = ns;
            g->arm = I8_TILE;
            g->tile = t;
            g->bn = c.bn;
            g->bm = c.bm;
            g->tiles = tiles;
            g->kc = (int)kc;
            g->per = (int)per;
            g->blocks = tiles * kc;
            g->waves = 0;
        }
    }
}

int64_t i8_scratch_bytes(const RadArgs* a, int ncu) {
    I8Plan P{};
    if (plan_i8(a, 0, &P) != RAD_OK) {
        /* not a whole call yet: dense operands on lines */
        long long N = 0, K = 0, M = 0;
        P = I8Plan{};
        if (!rad_args_geti(a, "N", &N) || !rad_args_geti(a, "K", &K) || N <= 0 || K <= 0 || N > kDimMax ||
            K > kI8MaxK)
            return 0;
        const RadTensor* Y = rad_arg_in(a, 4);
        if (Y) M = rad_tensor_numel(Y) / N;
        else if (!rad_args_geti(a, "M", &M)) M = 128;
        if (M <= 0 || M > kDimMax) return 0;
        P.M = M;
        P.N = N;
        P.K = K;
        P.ua = (K & 15) != 0;
        P.off = (K & 127) != 0;
    }
    return i8_planes_bytes(P, ncu);
}

int64_t i8_planes_bytes(const I8Plan& P, int ncu) {
    I8Geom g;
    i8_geom(P, ncu, kI8MaxPlanes, &g);
    return g.arm == I8_TILE && g.kc > 1 ? (int64_t)g.kc * P.M * P.N * 4 : 0;
}

int plan_i8_band(const RadArgs* a, int op, I8BandPlan* P) {
    /* operands: x, q, scale (quant); gate_up, q, scale, out? (gated);
     * x, residual?, w, q, scale, out?, residual_out? (rmsnorm) */
    const bool norm = op == I8_NORM;
    const int iq = norm ? 3 : 1;
    const RadTensor* x  = rad_arg_in(a, 0);
    const RadTensor* rs = norm ? rad_arg_in(a, 1) : nullptr;
    const RadTensor* w  = norm ? rad_arg_in(a, 2) : nullptr;
    const RadTensor* q  = rad_arg_in(a, iq);
    const RadTensor* sc = rad_arg_in(a, iq + 1);
    const RadTensor* ob = op == I8_QUANT ? nullptr : rad_arg_in(a, iq + 2);
    const RadTensor* ro = norm ? rad_arg_in(a, 6) : nullptr;
    if (!x || !q || !sc || (norm && !w) || (rs == nullptr) != (ro == nullptr)) return RAD_E_INVAL;
    if (x->dtype != RAD_BF16 && (norm || x->dtype != RAD_F32)) return RAD_E_DTYPE;
    if (q->dtype != RAD_I8 || sc->dtype != RAD_F32) return RAD_E_DTYPE;
    if (ob && ob->dtype != RAD_F32 && ob->dtype != RAD_BF16) return RAD_E_DTYPE;
    if (norm && w->dtype != RAD_F32 && w->dtype != RAD_BF16) return RAD_E_DTYPE;
    if (rs && (rs->dtype != RAD_BF16 || ro->dtype != RAD_BF16)) return RAD_E_DTYPE;
    const char* dt = rad_args_gets(a, "dtype");            /* names x's type, if given */
    if (dt && strcmp(dt, x->dtype == RAD_BF16 ? "bf16" : "f32") != 0) return RAD_E_DTYPE;
    const int64_t per = op == I8_GATED ? 2 : 1;
    long long v = 0;
    if (!rad_args_geti(a, "n", &v) || v <= 0 || v > kDimMax) return RAD_E_SHAPE;
    const int64_t n = v;
    const long long xn = rad_tensor_numel(x);
    if (xn <= 0 || xn % (per * n)) return RAD_E_SHAPE;
    const int64_t rows = xn / (per * n);
    if (rows > 0x7FFFFFFF) return RAD_E_SHAPE;
    const char* act = rad_args_gets(a, "act");
    if (op == I8_GATED && act && strcmp(act, "silu") != 0 && strcmp(act, "sigmoid") != 0)
        return RAD_E_UNSUPPORTED;
    P->silu = !act || strcmp(act, "silu") == 0;
    int rc = rows_of(x, rows, per * n, &P->x_pitch);
    if (!rc) rc = rows_of(q, rows, n, &P->q_pitch);
    if (!rc) {
        rc = scale_column(sc, rows, &P->s_stride);
        if (rc == RAD_E_UNSUPPORTED) rc = RAD_E_DTYPE;
    }
    if (!rc && ob) rc = rows_of(ob, rows, n, &P->ob_pitch);
    if (!rc && rs) rc = rows_of(rs, rows, n, &P->r_pitch);
    if (!rc && ro) rc = rows_of(ro, rows, n, &P->ro_pitch);
    if (rc) return rc;
    if (norm && (rad_tensor_numel(w) != n || w->rank != 1)) return RAD_E_SHAPE;
    if (norm && w->stride[0] != 1) return RAD_E_STRIDE;
    /* outputs whose rows overlap would race */
    if (rows > 1 && (P->q_pitch < n || P->s_stride < 1 || (ob && P->ob_pitch < n) ||
                     (ro && P->ro_pitch < n)))
        return RAD_E_STRIDE;
    /* elements lie on their own alignment; nothing more is asked of any operand */
    auto off = [](const RadTensor* t) {
        return t && ((uintptr_t)t->data & (t->dtype == RAD_F32 ? 3 : t->dtype == RAD_BF16 ? 1 : 0));
    };
    if (off(x) || off(rs) || off(w) || off(sc) || off(ob) || off(ro)) return RAD_E_STRIDE;
    P->x = (const uint8_t*)x->data;
    P->res = rs ? (const uint8_t*)rs->data : nullptr;
    P->res_out = ro ? (uint8_t*)ro->data : nullptr;
    P->w = w ? (const uint8_t*)w->data : nullptr;
    P->q = (uint8_t*)q->data;
    P->scale = (float*)sc->data;
    P->ob = ob ? (uint8_t*)ob->data : nullptr;
    P->x_bf16 = x->dtype == RAD_BF16;
    P->w_bf16 = w && w->dtype == RAD_BF16;
    P->ob_bf16 = ob && ob->dtype == RAD_BF16;
    P->rows = rows;
    P->n = n;
    P->eps = rad_args_getf_or(a, "eps", 1e-6);
    P->wadd = (float)rad_args_getf_or(a, "wadd", 0.0);
    if (!(P->eps >= 0.0)) return RAD_E_INVAL;
    if (rows * i8_band_geom(rows, n).lanes > 0xFFFFFFFFLL) return RAD_E_UNSUPPORTED;   /* lanes a launch */
    return RAD_OK;
}

I8BandGeom i8_band_geom(int64_t rows, int64_t n) {
    const int64_t nc = (n + 7) / 8;
    if (nc > 4096) return I8BandGeom{1024, 0};
    auto lanes = [&](int c) { return (int)(((nc + c - 1) / c + 63) / 64 * 64); };
    /* us at the chunks a lane named, rows of n (norm; gated g):
     *     1 x 5376     1: 4.3   2: 5.2   3: 5.4        1 x 8192     1: 4.9   2: 4.5   3: 5.7
     *     1 x 21504 g  3: 6.5   4: 6.6                 1 x 12000 g  2: 4.4   3: 4.7   4: 5.4
     *  2048 x 5376     1: 27.1  2: 24.2  3: 21.8    2048 x 8192     1: 30.8  2: 27.7  3: 31.1
     *  4096 x 2304     1: 23.7  2: 21.2  3: 19.7    4096 x 2000 g   1: 12.0  2: 12.5  3: 15.9
     * Few rows, or short ones: as few chunks as some 768 lanes allow.  Many long rows: two to four,
     * the fewest idle lanes, three where they tie. */
    if (nc <= 256 || rows * nc < 400000) {
        const int c = nc <= 768 ? 1 : nc <= 1536 ? 2 : lanes(3) <= 1024 ? 3 : 4;
        return I8BandGeom{lanes(c), c};
    }
    int best = 0;
    for (int c : {3, 2, 4})
        if (lanes(c) <= 1024 && (!best || lanes(c) * c < lanes(best) * best)) best = c;
    return I8BandGeom{lanes(best), best};
}

int describe_i8(const char* row, const RadArgs* a, char* buf, int len) {
    const bool gemm = !strcmp(row, "gemm_nt_q_i8a8"), dec = !strcmp(row, "gemm_nt_q_i8a8_decode");
    if (gemm || dec) {
        I8Plan P{};
        const int rc = plan_i8(a, dec ? 16 : 0, &P);
        if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
        I8Geom g;
        const bool sc = a->scratch && ((uintptr_t)a->scratch & 15) == 0;
        i8_geom(P, 256, sc ? a->scratch_bytes : 0, &g);
        static const char* kArm[] = {"any", "gemv", "tile"};
        snprintf(buf, (size_t)len, "arm=%s enc=i8a8 M=%lld N=%lld K=%lld bn=%d bm=%d tiles=%lld kc=%d "
                 "per=%d waves=%d blocks=%lld", kArm[g.arm], (long long)P.M, (long long)P.N,
                 (long long)P.K, g.bn, g.bm, (long long)g.tiles, g.kc, g.per, g.waves,
                 (long long)g.blocks);
        return RAD_OK;
    }
    const int op = !strcmp(row, "quant_act_i8") ? I8_QUANT : !strcmp(row, "gated_quant_i8") ? I8_GATED
                 : !strcmp(row, "rmsnorm_quant_i8") ? I8_NORM : -1;
    if (op < 0) return -1;
    I8BandPlan P{};
    const int rc = plan_i8_band(a, op, &P);
    if (rc) { snprintf(buf, (size_t)len, "refused rc=%d (plan)", rc); return rc; }
    const I8BandGeom g = i8_band_geom(P.rows, P.n);
    snprintf(buf, (size_t)len, "arm=band op=%s x=%s rows=%lld n=%lld lanes=%d chunks=%d residual=%d "
             "ob=%s", row, P.x_bf16 ? "bf16" : "f32", (long long)P.rows, (long long)P.n, g.lanes,
             g.chunks, P.res != nullptr, P.ob ? (P.ob_bf16 ? "bf16" : "f32") : "none");
    return RAD_OK;
}

bool env_no_i8()     { static const bool v = getenv("R3D_NO_I8") != nullptr;     return v; }
bool env_no_i8_dec() { static const bool v = getenv("R3D_NO_I8_DEC") != nullptr; return v; }

}  // namespace r3d
