/* r3d_moe.hip -- moe_layer on gfx950 (r3d_moe.h has the formulas): kernels and entry.
 *
 * Few tokens choose among many experts, so the chosen experts' planes are the work: each is to be read once, and
 * HBM bounds it.  A wave takes 8 rows of a plane as i8_gemv_kernel does (r3d_i8_gemv.h): a 16-byte load a lane
 * brings a 128-byte line of each, and v_mfma_f32_16x16x32_bf16 is fed with (row i % 8, pieces of parity i / 8)
 * against (token j % 8, parity j / 8), of whose 16 x 16 results those with i / 8 = j / 8 are wanted.  Codes become
 * bf16 in registers: int8 and e2m1 with its E8M0 scale are exact there (E8M0 0 is 2^-127, 255 NaN, and what leaves
 * bf16's range infinite), so the sums are f32 sums of exact products.
 *
 *   up    every workgroup makes the same choice from the logits for itself (a few hundred cycles a token and wave,
 *         which costs less than a kernel of its own before this one), so that it knows the jobs: an expert and up
 *         to 8 CT of its tokens.  Units of (job, 8 of f) go round the workgroups; a unit's gate and up rows are KC
 *         waves', K cut between them.  h leaves with its weight, to slot (job's first + token).
 *   down  a workgroup owns 8 RT rows of y, its waves the jobs' lines in equal runs; a wave adds each job's rows to
 *         its own sums in LDS by token, and the waves' sums are added in their order.  Nothing is added in an order
 *         that changes from run to run.
 *
 * h is bf16 where y is: its rounding (2^-9 of each of f terms at most, of random sign) is under y's own.  Where y is f32 it
 * is two bf16 numbers, high and low, 2^-17 together. */
#include <hip/hip_runtime.h>

#include <stdio.h>

#include "r3d_act_dev.h"
#include "r3d_device.h"
#include "r3d_dump.h"
#include "r3d_i8_launch.h"
#include "r3d_moe.h"
#include "r3d_wave.h"

namespace r3d {

struct MoeUpArgs {
    const uint8_t* x;
    const uint8_t* logits;
    const uint8_t* w;
    const uint8_t* ws;
    MoeTable* table;
    uint16_t* h;
    uint16_t* h_lo;                     /* null: h is bf16 alone */
    int32_t* ids;
    float* weights;
    int M, n, f, E, top_k, x_pitch, w_pitch, kc, act, sigmoid, renorm, l_bf16;
    int64_t w_expert, ws_expert, ws_pitch, l_pitch, i_pitch, wt_pitch;
    float weight_scale;
};
struct MoeDownArgs {
    const uint8_t* h;
    const uint8_t* h_lo;
    const uint8_t* w;
    const uint8_t* ws;
    const MoeTable* table;
    uint8_t* y;
    int M, n, f, pairs, w_pitch, y_bf16;
    int64_t w_expert, ws_expert, ws_pitch, y_pitch;
};

/* 16 bytes of codes: how many weights, and 16-byte pieces of bf16 that these become */
template <int ENC>
struct MoeCodes {
    static constexpr int N = ENC == MOE_BF16 ? 8 : ENC == MOE_I8 ? 16 : 32, X = N / 8;
};

__device__ __forceinline__ r3d_f32x4 moe_mfma(r3d_i32x4 w, r3d_i32x4 x, r3d_f32x4 c) {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
}

template <int ENC>
__device__ __forceinline__ void moe_bf16(r3d_i32x4 w, uint32_t scale, r3d_i32x4 (&b)[MoeCodes<ENC>::X]) {
    if constexpr (ENC == MOE_BF16) {
        b[0] = w;
    } else if constexpr (ENC == MOE_I8) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int v = w[d];
            b[d >> 1][2 * (d & 1)] = (int)r3d_pack_bf16x2((float)(int8_t)v, (float)(int8_t)(v >> 8));
            b[d >> 1][2 * (d & 1) + 1] = (int)r3d_pack_bf16x2((float)(int8_t)(v >> 16), (float)(v >> 24));
        }
    } else {
        const float s = __uint_as_float(scale << 23);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            b[d][0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)w[d], s, 0));
            b[d][1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)w[d], s, 1));
            b[d][2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)w[d], s, 2));
            b[d][3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)w[d], s, 3));
        }
    }
}

/* ------------------------------------------------------------------------------ the choice */

constexpr int kMoeThreads = 512, kMoeWaves = 8;

struct MoeChoice {                      /* in LDS, the same in every workgroup */
    uint64_t mask[kMoeMaxE];            /* an expert's tokens */
    uint64_t scan[kMoeWaves];
    float w[kMoeMaxPairs];              /* by (token, choice) */
    float slot_w[kMoeMaxPairs];         /* by slot */
    uint32_t job[kMoeMaxPairs];
    int16_t id[kMoeMaxPairs];           /* by (token, choice); -1: none */
    uint16_t first[kMoeMaxE];           /* an expert's first slot */
    uint8_t tok[kMoeMaxPairs];          /* by slot */
    int jobs;
};

/* Token t's choices and weights, a wave's work: lane l holds the logits of experts J l .. J l + J - 1 as whole
 * numbers in the same order, 0 for what is not there (NaN, -inf); each round takes the wave's largest, of equals the
 * first lane's first. */
template <int J>
__device__ __forceinline__ void moe_choose(const MoeUpArgs& P, MoeChoice& S, int t) {
    const int lane = threadIdx.x & 63;
    float v[J];
    uint32_t key[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = J * lane + j;
        v[j] = -__builtin_inff();
        if (e < P.E)
            v[j] = P.l_bf16 ? r3d_bf16_to_f32(reinterpret_cast<const uint16_t*>(P.logits)[t * P.l_pitch + e])
                            : reinterpret_cast<const float*>(P.logits)[t * P.l_pitch + e];
        const uint32_t u = __float_as_uint(v[j] + 0.0f);                 /* -0 is 0 */
        key[j] = v[j] > -__builtin_inff() ? u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u) : 0u;
    }
    int id = -1;
    float mine = 0.0f;
    int count = 0;
    for (int i = 0; i < P.top_k; ++i) {
        uint32_t m = key[0];
#pragma unroll
        for (int j = 1; j < J; ++j) m = m > key[j] ? m : key[j];
        const uint32_t top = r3d_wave_max(m);
        if (top == 0) break;
        const int from = __builtin_ctzll(__ballot(m == top));
        int at = 0;
#pragma unroll
        for (int j = J - 1; j >= 0; --j) at = key[j] == top ? j : at;
        const int e = __builtin_amdgcn_readlane(J * lane + at, from);
        if (lane == from) {
#pragma unroll
            for (int j = 0; j < J; ++j) key[j] = j == at ? 0u : key[j];
        }
        if (lane == i) {
            id = e;
            mine = __uint_as_float(top ^ ((top >> 31) ? 0x80000000u : 0xFFFFFFFFu));
        }
        ++count;
    }
    const bool there = lane < count;
    const float top = __uint_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), 0));
    float p, total;
    if (!P.sigmoid) {
        /* an infinite logit counts as the largest finite one would beside it: e^0 */
        p = there ? (mine == top ? 1.0f : expf(mine - top)) : 0.0f;
        double sum = p;
        if (!P.renorm) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (v[j] > -__builtin_inff()) s += v[j] == top ? 1.0f : expf(v[j] - top);
            sum = s;
        }
        total = (float)r3d_wave_sum(sum);
    } else if (P.renorm) {
        /* of sigmoids all far below zero the ratio: e^(v - top) / (1 + e^v), which no exponent range ends */
        p = !there ? 0.0f : top < 0.0f ? expf(mine - top) / (1.0f + expf(mine)) : i8_sigmoid(mine);
        total = (float)r3d_wave_sum((double)p);
    } else {
        p = there ? i8_sigmoid(mine) : 0.0f;
        total = 1.0f;
    }
    if (lane < P.top_k) {
        S.id[t * P.top_k + lane] = (int16_t)id;
        S.w[t * P.top_k + lane] = there ? p / total * P.weight_scale : 0.0f;
    }
}

/* Choices of every token, then the experts' slots and jobs.  All lanes of the workgroup. */
template <int CT>
__device__ __forceinline__ void moe_plan(const MoeUpArgs& P, MoeChoice& S) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    S.mask[tid] = 0;
    for (int t = wave; t < P.M; t += kMoeWaves) {
        if (P.E <= 64) moe_choose<1>(P, S, t);
        else if (P.E <= 128) moe_choose<2>(P, S, t);
        else if (P.E <= 256) moe_choose<4>(P, S, t);
        else moe_choose<8>(P, S, t);
    }
    __syncthreads();
    const int pairs = P.M * P.top_k;
    for (int i = tid; i < pairs; i += kMoeThreads) {
        const int e = S.id[i];
        if (e >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&S.mask[e]), 1ull << (i / P.top_k));
    }
    __syncthreads();
    /* a lane an expert: slots and jobs before it */
    const int cnt = __popcll(S.mask[tid]), nj = (cnt + 8 * CT - 1) / (8 * CT);
    const uint64_t own = (uint64_t)nj << 32 | (uint32_t)cnt;
    uint64_t upto = r3d_wave_scan(own);
    if (lane == 63) S.scan[wave] = upto;
    __syncthreads();
    uint64_t all = 0;
    for (int i = 0; i < kMoeWaves; ++i) {
        if (i == wave) upto += all;
        all += S.scan[i];
    }
    const int slot = (int)(uint32_t)(upto - own), j0 = (int)((upto - own) >> 32);
    S.first[tid] = (uint16_t)slot;
    for (int j = 0; j < nj; ++j) {
        const int left = cnt - 8 * CT * j;
        S.job[j0 + j] = (uint32_t)tid | (uint32_t)(slot + 8 * CT * j) << 9 | (uint32_t)(left < 8 * CT ? left : 8 * CT) << 20;
    }
    if (tid == 0) S.jobs = (int)(all >> 32);
    __syncthreads();
    for (int i = tid; i < pairs; i += kMoeThreads) {
        const int e = S.id[i], t = i / P.top_k;
        if (e < 0) continue;
        const int at = S.first[e] + __popcll(S.mask[e] & ((1ull << t) - 1));
        S.tok[at] = (uint8_t)t;
        S.slot_w[at] = S.w[i];
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = tid; i < kMoeMaxPairs; i += kMoeThreads) {
            if (i < S.jobs) P.table->job[i] = S.job[i];
            if (i < pairs) {
                P.table->tok[i] = S.tok[i];
                if (P.ids) P.ids[i / P.top_k * P.i_pitch + i % P.top_k] = S.id[i];
                if (P.weights) P.weights[i / P.top_k * P.wt_pitch + i % P.top_k] = S.w[i];
            }
        }
        if (tid == 0) P.table->jobs = S.jobs;
    }
}

/* ------------------------------------------------------------------------------ products */

/* One line of 8 rows of R planes' blocks and of 8 CT columns, on its way. */
template <int ENC, int R, int CT, int XH>
struct MoeStep {
    r3d_i32x4 w[R];
    uint32_t s[R];                                              /* e2m1: the piece's scale */
    r3d_i32x4 x[CT][XH * MoeCodes<ENC>::X];
};

template <int ENC, int R, int CT, int XH>
__device__ __forceinline__ void moe_products(const MoeStep<ENC, R, CT, XH>& st, r3d_f32x4 (&acc)[R][CT]) {
    constexpr int X = MoeCodes<ENC>::X;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        r3d_i32x4 b[X];
        moe_bf16<ENC>(st.w[r], st.s[r], b);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < XH * X; ++i) acc[r][c] = moe_mfma(b[i % X], st.x[c][i], acc[r][c]);
    }
}

/* The sum of a result's two halves, (0, 0) and (1, 1), 40 lanes apart: lanes 0-7 and 16-23 then hold rows
 * 4 (lane / 16) .. + 3 of column lane % 8. */
__device__ __forceinline__ r3d_f32x4 moe_halves(r3d_f32x4 a) {
    const int from = ((threadIdx.x & 63) + 40) & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += __shfl(a[i], from, 64);
    return a;
}

template <int ENC, int CT>
__global__ __launch_bounds__(kMoeThreads) void moe_up_kernel(MoeUpArgs P) {
    constexpr int N = MoeCodes<ENC>::N, X = MoeCodes<ENC>::X, D = CT == 1 ? 4 : 2;
    __shared__ MoeChoice S;
    __shared__ r3d_f32x4 s_part[kMoeWaves][CT][2][16];
    moe_plan<CT>(P, S);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r8 = lane & 7, piece = ((lane >> 3) & 1) | ((lane >> 4) << 1);
    const int fb = P.f >> 3, units = S.jobs * fb, kc = P.kc, upw = kMoeWaves / kc;
    const int sub = i8_uniform(wave / kc), c = wave - sub * kc;
    const int pieces = P.n / N, lines = (pieces + 7) >> 3, per = (lines + kc - 1) / kc;
    const int l0 = c * per, l1 = l0 + per < lines ? l0 + per : lines;
    const __amdgpu_buffer_rsrc_t rX = r3d_rsrc(P.x, (int64_t)(P.M - 1) * P.x_pitch + 2 * (int64_t)P.n);
    const int64_t plane = (int64_t)(2 * P.f - 1) * P.w_pitch + (int64_t)pieces * 16;

    for (int u0 = blockIdx.x * upw; u0 < units; u0 += gridDim.x * upw) {
        const int u = u0 + sub, live = u < units;
        const int jb = i8_uniform(live ? u / fb : 0), b0 = 8 * (live ? u - jb * fb : 0);
        const uint32_t job = i8_uniform(S.job[jb]);
        const int e = job & 511, slot0 = (job >> 9) & 2047, cnt = live ? job >> 20 : 0;
        if (live) {
            const __amdgpu_buffer_rsrc_t rW = r3d_rsrc(P.w + e * P.w_expert, plane);
            const __amdgpu_buffer_rsrc_t rS = r3d_rsrc(ENC == MOE_FP4 ? P.ws + e * P.ws_expert : nullptr,
                                                       ENC == MOE_FP4 ? (2 * P.f - 1) * P.ws_pitch + pieces : 0);
            const uint32_t wo[2] = {(uint32_t)((b0 + r8) * P.w_pitch + 16 * piece),
                                    (uint32_t)((P.f + b0 + r8) * P.w_pitch + 16 * piece)};
            const uint32_t so[2] = {(uint32_t)((b0 + r8) * P.ws_pitch + piece),
                                    (uint32_t)((P.f + b0 + r8) * P.ws_pitch + piece)};
            uint32_t xo[CT];
#pragma unroll
            for (int t = 0; t < CT; ++t)
                xo[t] = 8 * t + r8 < cnt ? (uint32_t)(S.tok[slot0 + 8 * t + r8] * P.x_pitch + 16 * X * piece) : kI8Oob;
            MoeStep<ENC, 2, CT, 1> ring[D];
            auto load = [&](MoeStep<ENC, 2, CT, 1>& st, int l) __attribute__((always_inline)) {
                const bool in = l < l1 && 8 * l + piece < pieces;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    st.w[r] = i8_buf16<2>(rW, in ? wo[r] : kI8Oob, 128 * l);
                    if (ENC == MOE_FP4)
                        st.s[r] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rS, (int)(in ? so[r] : kI8Oob), 8 * l, 0);
                }
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int i = 0; i < X; ++i)
                        st.x[t][i] = i8_buf16<0>(rX, in ? xo[t] + 16 * i : kI8Oob, 128 * X * l);
            };
            r3d_f32x4 acc[2][CT];
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[0][t] = acc[1][t] = r3d_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < D; ++d) load(ring[d], l0 + d);
            for (int l = l0; l < l1; l += D) {
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    moe_products(ring[d], acc);
                    load(ring[d], l + D + d);
                }
            }
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const r3d_f32x4 v = moe_halves(acc[r][t]);
                    if (lane < 32 && !(lane & 8)) s_part[wave][t][r][(lane >> 4) * 8 + r8] = v;
                }
        }
        __syncthreads();
        if (live && c == 0 && lane < 16 * CT) {
            /* lane (t, half, column): rows 4 half .. + 3 of token 8 t + column */
            const int t = lane >> 4, half = (lane >> 3) & 1, col = 8 * t + (lane & 7);
            r3d_f32x4 g = s_part[wave][t][0][lane & 15], w = s_part[wave][t][1][lane & 15];
            for (int o = 1; o < kc; ++o) {
                g += s_part[wave + o][t][0][lane & 15];
                w += s_part[wave + o][t][1][lane & 15];
            }
            if (col < cnt) {
                const int row = b0 + 4 * half, slot = slot0 + col;
                float a[4], v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = g[i];
                    v[i] = w[i];
                    if (ENC == MOE_I8) {
                        const float* s = reinterpret_cast<const float*>(P.ws) + e * P.ws_expert + row + i;
                        a[i] *= s[0];
                        v[i] *= s[P.f];
                    }
                }
                act_values<4>(P.act, a);
                const float wt = S.slot_w[slot];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = a[i] * v[i] * wt;
                const uint32_t h0 = r3d_pack_bf16x2(a[0], a[1]), h1 = r3d_pack_bf16x2(a[2], a[3]);
                *reinterpret_cast<uint2*>(P.h + (int64_t)slot * P.f + row) = make_uint2(h0, h1);
                if (P.h_lo) {
                    float lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t d = i < 2 ? h0 : h1;
                        const float hi = __uint_as_float(i & 1 ? d & 0xFFFF0000u : d << 16);
                        lo[i] = __builtin_fabsf(hi) < __builtin_inff() ? a[i] - hi : 0.0f;   /* inf - inf; NaN is in hi */
                    }
                    *reinterpret_cast<uint2*>(P.h_lo + (int64_t)slot * P.f + row) =
                        make_uint2(r3d_pack_bf16x2(lo[0], lo[1]), r3d_pack_bf16x2(lo[2], lo[3]));
                }
            }
        }
        __syncthreads();
    }
}

/* XH 2: h in two parts */
template <int ENC, int CT, int RT, int XH>
__global__ __launch_bounds__(kMoeThreads) void moe_down_kernel(MoeDownArgs P) {
    constexpr int N = MoeCodes<ENC>::N, X = MoeCodes<ENC>::X, D = CT * RT * XH == 1 ? 4 : 2;
    __shared__ uint32_t s_job[kMoeMaxPairs];
    __shared__ uint8_t s_tok[kMoeMaxPairs];
    extern __shared__ __attribute__((aligned(16))) float s_y[];     /* [waves][M][8 RT] */
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jobs = P.table->jobs;
    /* past the table's own entries: what lies there is not used */
    *reinterpret_cast<uint2*>(s_job + 2 * tid) = *reinterpret_cast<const uint2*>(P.table->job + 2 * tid);
    *reinterpret_cast<uint16_t*>(s_tok + 2 * tid) = *reinterpret_cast<const uint16_t*>(P.table->tok + 2 * tid);
    for (int i = tid; i < kMoeWaves * P.M * 8 * RT; i += kMoeThreads) s_y[i] = 0.0f;
    __syncthreads();
    const int r8 = lane & 7, piece = ((lane >> 3) & 1) | ((lane >> 4) << 1);
    const int pieces = P.f / N, lines = (pieces + 7) >> 3;
    const int64_t total = (int64_t)jobs * lines;
    const int s0 = (int)(total * wave / kMoeWaves), s1 = (int)(total * (wave + 1) / kMoeWaves);
    const int row0 = blockIdx.x * 8 * RT;
    float* const ys = s_y + wave * P.M * 8 * RT;
    const int64_t plane = (int64_t)(P.n - 1) * P.w_pitch + (int64_t)pieces * 16;
    const int64_t h_bytes = (int64_t)P.pairs * P.f * 2;
    const __amdgpu_buffer_rsrc_t rH = r3d_rsrc(P.h, h_bytes);
    const __amdgpu_buffer_rsrc_t rL = r3d_rsrc(XH == 2 ? P.h_lo : P.h, XH == 2 ? h_bytes : 0);
    uint32_t wo[RT], so[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {                                    /* rows past n are past the plane: zeros */
        wo[r] = (uint32_t)(row0 + 8 * r + r8) * (uint32_t)P.w_pitch + 16 * piece;
        so[r] = (uint32_t)((row0 + 8 * r + r8) * P.ws_pitch + piece);
    }
    struct Ring {
        MoeStep<ENC, RT, CT, XH> st;
        r3d_f32x4 scale[RT];                                          /* int8: of the job's rows, with its last line */
    } ring[D];
    /* the run that loads walk, D steps ahead of the products */
    int lj = lines ? s0 / lines : 0, ll = s0 - lj * lines;
    __amdgpu_buffer_rsrc_t rW = r3d_rsrc(P.w, 0), rS = rW;
    uint32_t xo[CT];
    int64_t sc_at = 0;
    auto enter = [&](int j) __attribute__((always_inline)) {
        const uint32_t job = i8_uniform(s_job[j]);
        const int64_t e = job & 511;
        const int slot0 = (job >> 9) & 2047, cnt = job >> 20;
        rW = r3d_rsrc(P.w + e * P.w_expert, plane);
        if (ENC == MOE_FP4) rS = r3d_rsrc(P.ws + e * P.ws_expert, (P.n - 1) * P.ws_pitch + pieces);
        if (ENC == MOE_I8) sc_at = e * P.ws_expert;
#pragma unroll
        for (int t = 0; t < CT; ++t)
            xo[t] = 8 * t + r8 < cnt ? (uint32_t)((slot0 + 8 * t + r8) * P.f * 2 + 16 * X * piece) : kI8Oob;
    };
    auto load = [&](Ring& g, int s) __attribute__((always_inline)) {
        const bool run = s < s1;
        if (run && (ll == 0 || s == s0)) enter(lj);
        const bool in = run && 8 * ll + piece < pieces;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            g.st.w[r] = i8_buf16<2>(rW, in ? wo[r] : kI8Oob, 128 * ll);
            if (ENC == MOE_FP4)
                g.st.s[r] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rS, (int)(in ? so[r] : kI8Oob), 8 * ll, 0);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int i = 0; i < X; ++i) {
                g.st.x[t][i] = i8_buf16<0>(rH, in ? xo[t] + 16 * i : kI8Oob, 128 * X * ll);
                if (XH == 2) g.st.x[t][(XH - 1) * X + i] = i8_buf16<0>(rL, in ? xo[t] + 16 * i : kI8Oob, 128 * X * ll);
            }
        if (ENC == MOE_I8 && run && (ll == lines - 1 || s == s1 - 1)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                int at = row0 + 8 * r + 4 * ((lane >> 4) & 1);
                at = at + 4 <= P.n ? at : 0;
                g.scale[r] = *reinterpret_cast<const r3d_f32x4_u4*>(reinterpret_cast<const float*>(P.ws) + sc_at + at);
            }
        }
        if (++ll == lines) {
            ll = 0;
            ++lj;
        }
    };
    r3d_f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[r][t] = r3d_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int cj = lj, cl = ll;
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(ring[d], s0 + d);
    }
    for (int s = s0; s < s1; s += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (s + d < s1) {
                moe_products(ring[d].st, acc);
                if (++cl == lines || s + d + 1 == s1) {               /* the job's end, or the run's */
                    const uint32_t job = i8_uniform(s_job[cj]);
                    const int slot0 = (job >> 9) & 2047, cnt = job >> 20;
#pragma unroll
                    for (int t = 0; t < CT; ++t)
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            r3d_f32x4 v = moe_halves(acc[r][t]);
                            acc[r][t] = r3d_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                            if (ENC == MOE_I8) v *= ring[d].scale[r];
                            if (lane < 32 && !(lane & 8) && 8 * t + r8 < cnt) {
                                /* a token comes once a job: no two lanes meet */
                                r3d_f32x4* const to = reinterpret_cast<r3d_f32x4*>(
                                    ys + s_tok[slot0 + 8 * t + r8] * 8 * RT + 8 * r + 4 * (lane >> 4));
                                *to += v;
                            }
                        }
                    cl = 0;
                    ++cj;
                }
            }
            load(ring[d], s + D + d);
        }
    }
    __syncthreads();
    for (int i = tid; i < P.M * 8 * RT; i += kMoeThreads) {
        const int m = i / (8 * RT), row = row0 + i % (8 * RT);
        float v = s_y[i];
        for (int w = 1; w < kMoeWaves; ++w) v += s_y[w * P.M * 8 * RT + i];
        if (row >= P.n) continue;
        if (P.y_bf16) reinterpret_cast<uint16_t*>(P.y)[m * P.y_pitch + row] = r3d_bf16_rne(v);
        else reinterpret_cast<float*>(P.y)[m * P.y_pitch + row] = v;
    }
}

template <int ENC, int CT>
static int moe_launch(const MoePlan& P, const MoeGeom& g, void* scratch, hipStream_t stream) {
    MoeTable* const table = static_cast<MoeTable*>(scratch);
    uint16_t* const h = reinterpret_cast<uint16_t*>(table + 1);
    uint16_t* const lo = P.y_bf16 ? nullptr : h + P.M * P.top_k * P.f;
    const MoeUpArgs u{P.x, P.logits, P.gu, P.gus, table, h, lo, P.ids, P.weights, (int)P.M, (int)P.n, (int)P.f, (int)P.E,
                      (int)P.top_k, (int)P.x_pitch, (int)P.gu_pitch, g.kc, P.act, P.sigmoid, P.renorm, P.l_bf16,
                      P.gu_expert, P.gus_expert, P.gus_pitch, P.l_pitch, P.i_pitch, P.w_pitch, P.weight_scale};
    hipLaunchKernelGGL((moe_up_kernel<ENC, CT>), dim3((unsigned)g.up_blocks), dim3(kMoeThreads), 0, stream, u);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) {
        const MoeDownArgs d{(const uint8_t*)h, (const uint8_t*)lo, P.dn, P.dns, table, P.y, (int)P.M, (int)P.n, (int)P.f,
                            (int)(P.M * P.top_k), (int)P.dn_pitch, P.y_bf16, P.dn_expert, P.dns_expert, P.dns_pitch, P.y_pitch};
        const size_t lds = (size_t)(kMoeWaves * P.M * 8) * 4;
        const dim3 grid((unsigned)g.down_blocks);
        if (lo) hipLaunchKernelGGL((moe_down_kernel<ENC, CT, 1, 2>), grid, dim3(kMoeThreads), lds, stream, d);
        else hipLaunchKernelGGL((moe_down_kernel<ENC, CT, 1, 1>), grid, dim3(kMoeThreads), lds, stream, d);
        e = hipGetLastError();
    }
    return e == hipSuccess ? RAD_OK : i8_failed("moe_layer", e);
}

static int moe_entry(const RadArgs* a, RadStream s) {
    if (env_no_moe()) return RAD_E_UNSUPPORTED;
    MoePlan P{};
    const int rc = plan_moe(a, &P);
    if (rc) return rc;
    if (!a->scratch || (uintptr_t)a->scratch & 15 || a->scratch_bytes < moe_scratch(P)) return RAD_E_UNSUPPORTED;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    MoeGeom g;
    moe_geom(P, cu_count(), &g);
    hipStream_t t = (hipStream_t)s;
#define R3D_MOE(ENC_)                                                              \
    return g.ct == 1 ? moe_launch<ENC_, 1>(P, g, a->scratch, t)                     \
         : g.ct == 2 ? moe_launch<ENC_, 2>(P, g, a->scratch, t) : moe_launch<ENC_, 4>(P, g, a->scratch, t)
    if (P.enc == MOE_BF16) R3D_MOE(MOE_BF16);
    if (P.enc == MOE_I8) R3D_MOE(MOE_I8);
    R3D_MOE(MOE_FP4);
#undef R3D_MOE
}

}  // namespace r3d

extern "C" {

int r3d_rad_moe_layer(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("moe_layer", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::moe_entry(x, t);
    });
}
int64_t r3d_rad_moe_layer_scratch(const RadArgs* a) { return r3d::moe_scratch_bytes(a); }

}  /* extern "C" */
