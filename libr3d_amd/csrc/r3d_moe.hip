/* r3d_moe.hip -- moe_layer on gfx950 (r3d_moe.h has the formulas): kernels and entry.
 *
 * Few tokens choose among many experts, so the chosen experts' planes are the work: each is read once for every 8 of
 * its tokens (16 where many share it), for fewer where LDS does not hold as many of them, and HBM bounds it.  A 16-byte
 * load a lane brings a wave 256 bytes of 4 rows of a plane, a piece of 16 a lane, four lanes to 64 bytes of a row: the
 * order of K in a product is free as long as both sides share it, so v_mfma_f32_16x16x32_bf16 is fed with (row i / 4,
 * pieces of class i % 4) against (token j / 4, class j % 4), and of the 16 x 16 results those with i % 4 = j % 4 are
 * wanted.  Three quarters of the matrix core's work is thrown away and it still idles; the loads are what counts, and
 * the cache looks up 64 bytes at a time only where lanes beside each other ask for them (with 128 bytes of 8 rows a
 * load, two lanes beside each other: 28 look-ups for 16, 57 cycles a load, which bound it).  Codes become bf16 in
 * registers: int8 and e2m1 with its E8M0 scale are exact there (E8M0 0 is 2^-127, 255 NaN, and what leaves bf16's range
 * infinite), so the sums are f32 sums of exact products.
 *
 *   up    every workgroup makes the same choice from the logits for itself, a wave a token (3.4 us with the first loads,
 *         which costs less than a kernel of its own before this one; past 8 tokens, two rounds, a kernel of its own,
 *         a workgroup a token, costs less), so that it knows the jobs: an expert and some of its tokens.  A unit is a job's 8 gate and 8 up rows of f; h leaves with its weight, to its token's slot.
 *   down  a unit is a job's 16 rows of n; its sums leave to its tokens' slots in f32.  Long rows of h may take several launches.
 *   sum   y of each token's slots, in the order of its choice: nothing is added in an order that changes from run to run.
 *
 * up and down are one kernel: the units lie in a row, and each workgroup, one a compute unit, takes an equal run of
 * them; of a run's spans each of its 8 waves takes an equal run again, and what it leaves of a unit to the next wave
 * meets through LDS.  The tokens' rows of a run's jobs are in LDS, where the waves read them beside their weights'
 * loads, and the line's loads are the only ones in the stream: with the tokens read from memory too, the
 * address unit was busy 9 cycles of 10 at 2.5 TB/s (64 tokens, 128 e2m1 experts).
 *
 * h is kept in f32, and its bits go into the products as the sum of three bf16 numbers, which holds all 24 of them: those of
 * the parts cost matrix cycles, which idle here.  (Two parts, 2^-17 of it at most, put 0.22 % of 64 x 8 / 128's bf16 results on
 * the other side of a rounding, where f32 sums put 0.05 % and this puts 0.03; they took 287 us.)
 *
 * Measured on MI355X (tokens x choices / experts): 1 x 8 / 128 mxfp4, 5376 x 1344 32.3 us and 4 x 4 / 64 int8, 2048 x 768 25, each
 * launch's beginning and end 6 to 7 us of it; 13 x 4 / 32 bf16, 2048 x 1408 77 to 84, 5.3 to 5.8 TB/s; 64 x 8 / 128 mxfp4 300 to
 * 307, gate and up 5.8 TB/s, down 3.6 (three parts, and jobs past four tokens take a second tile). */
#include <hip/hip_runtime.h>

#include <stdio.h>

#include <type_traits>

#include "r3d_act_dev.h"
#include "r3d_device.h"
#include "r3d_dump.h"
#include "r3d_i8_launch.h"
#include "r3d_moe.h"
#include "r3d_wave.h"

namespace r3d {

/* u / d for a d that the host knows (any u, d >= 1), without the forty instructions of a division */
struct MoeDiv {
    uint32_t d, m;                      /* m = (2^32 - 1) / d, rounded down: the quotient is short by one at most */
    __device__ __forceinline__ uint32_t of(uint32_t u) const {
        const uint32_t q = __umulhi(u, m);
        return q + (u - q * d >= d ? 1u : 0u);
    }
};

struct MoeArgs {
    MoeTable* table;
    const uint8_t* logits;              /* up: null for down */
    int64_t l_pitch;
    int M, E, top_k, l_bf16, K, rows, pairs, x_pitch;    /* K columns of `rows` rows (gate rows, or rows of y) */
    const uint8_t* x;                   /* up: the tokens; down: h */
    const uint8_t* w;
    const uint8_t* ws;
    float* out;                         /* up: h [pairs][f]; down: sums [pairs][n] */
    int64_t w_expert, ws_expert, ws_pitch;
    int w_pitch, job_rows, spans, cpr;  /* spans of 256 bytes a row of the plane, 1 KB pieces of a token's row in bf16 */
    MoeDiv unit, line, grid, choice, chunk;      /* by units a job, spans, workgroups, top_k, cpr */
    /* up */
    int32_t* ids;
    float* weights;
    int64_t i_pitch, wt_pitch;
    MoeDiv width, down_width;           /* tokens a job */
    int act, sigmoid, renorm;
    float weight_scale;
    int add;                            /* down: to the sums of the columns before */
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
        const float s = __uint_as_float(scale);                      /* of which the conversion takes bits 23 to 30 alone */
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

/* Two waves a SIMD.  Four were no faster at any of the sizes below, and neither were more spans in flight a wave: the
 * CUs' share of HBM is reached with these. */
constexpr int kMoeWaves = 8, kMoeThreads = 64 * kMoeWaves;
constexpr int kMoeUnits = 128;          /* units whose scales lie in LDS at a time */

struct MoeChoice {                      /* in LDS, the same in every workgroup */
    uint64_t mask[kMoeMaxE];            /* an expert's tokens */
    float w[kMoeMaxPairs];              /* by (token, choice) */
    float slot_w[kMoeMaxPairs];         /* by slot */
    uint32_t job[kMoeMaxPairs];
    int16_t id[kMoeMaxPairs];           /* by (token, choice); -1: none */
    uint16_t first[kMoeMaxE];           /* an expert's first slot */
    uint8_t tok[kMoeMaxPairs];          /* by slot */
    int jobs;
};

/* A lane's logits of token t as they lie in memory, experts J l .. J l + J - 1; -inf past the last one.  Every load before
 * a use of one. */
template <int J>
__device__ __forceinline__ void moe_logits(const MoeArgs& P, int t, uint32_t (&raw)[J]) {
    const int e0 = J * (threadIdx.x & 63);
    if (P.l_bf16) {
        const uint16_t* const row = reinterpret_cast<const uint16_t*>(P.logits) + t * P.l_pitch;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            raw[j] = 0xFF80u;
            if (e0 + j < P.E) raw[j] = row[e0 + j];
        }
    } else {
        const uint32_t* const row = reinterpret_cast<const uint32_t*>(P.logits) + t * P.l_pitch;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            raw[j] = 0xFF800000u;
            if (e0 + j < P.E) raw[j] = row[e0 + j];
        }
    }
}

/* Token t's choices and weights, a wave's work: a lane's logits as whole numbers in the same order, 0 for what is not
 * there (NaN, -inf); each round takes the wave's largest, of equals the first lane's first.  ids and weights are S's, or
 * memory's. */
template <int J, class Id>
__device__ __forceinline__ void moe_choose(const MoeArgs& P, int t, const uint32_t (&raw)[J], Id* ids, float* weights, uint64_t* mask) {
    const int lane = threadIdx.x & 63;
    float v[J];
    uint32_t key[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        v[j] = __uint_as_float(P.l_bf16 ? raw[j] << 16 : raw[j]);
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
        ids[t * P.top_k + lane] = (Id)id;
        weights[t * P.top_k + lane] = there ? p / total * P.weight_scale : 0.0f;
        if (mask && there) atomicOr(reinterpret_cast<unsigned long long*>(mask + id), 1ull << t);
    }
}

template <int J>
__device__ __forceinline__ void moe_choose_own(const MoeArgs& P, MoeChoice& S) {
    const int t = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t raw[J];
    if (t < P.M) moe_logits<J>(P, t, raw);
    __syncthreads();                                                 /* the masks are clear */
    if (t < P.M) moe_choose<J>(P, t, raw, S.id, S.w, S.mask);
}

/* Choices of more tokens than a workgroup has waves: a wave a token, in a launch of its own (64 tokens made by every
 * workgroup for itself took 17 us, 2.1 a token and wave). */
__global__ __launch_bounds__(64) void moe_route_kernel(MoeArgs P) {
    const int t = blockIdx.x;
    int16_t* const id = P.table->id;
    float* const w = P.table->w;
    if (P.E <= 128) {
        uint32_t raw[2];
        moe_logits<2>(P, t, raw);
        moe_choose<2>(P, t, raw, id, w, nullptr);
    } else {
        uint32_t raw[8];
        moe_logits<8>(P, t, raw);
        moe_choose<8>(P, t, raw, id, w, nullptr);
    }
}

/* Choices of every token (or what moe_route_kernel made of them), then the experts' slots and jobs, up to `width` tokens each;
 * workgroup 0 writes the down kernel's too, whose rows in LDS are longer or shorter.  All lanes of the workgroup. */
__device__ __forceinline__ void moe_plan(const MoeArgs& P, MoeChoice& S) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < kMoeMaxE; i += kMoeThreads) S.mask[i] = 0;
    if (P.M > kMoeWaves) {
        constexpr int EACH = kMoeMaxPairs / kMoeThreads;
        int id[EACH];
        float w[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = tid + i * kMoeThreads;
            id[i] = at < P.pairs ? P.table->id[at] : -1;
            w[i] = at < P.pairs ? P.table->w[at] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = tid + i * kMoeThreads;
            S.id[at] = (int16_t)id[i];
            S.w[at] = w[i];
            if (id[i] >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&S.mask[id[i]]), 1ull << P.choice.of(at));
        }
    } else if (P.E <= 128) {
        moe_choose_own<2>(P, S);
    } else {
        moe_choose_own<8>(P, S);
    }
    __syncthreads();
    if (wave == 0) {                                             /* a lane eight experts: slots and jobs before each */
        uint32_t cnt[8];
        uint64_t own = 0;                                        /* slots, jobs and the down kernel's jobs, 21 bits each */
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            cnt[i] = __popcll(S.mask[8 * lane + i]);
            own += (uint64_t)P.down_width.of(cnt[i] + P.down_width.d - 1) << 42 |
                   (uint64_t)P.width.of(cnt[i] + P.width.d - 1) << 21 | cnt[i];
        }
        const uint64_t upto = r3d_wave_scan(own);
        uint32_t slot = (uint32_t)(upto - own) & 0x1FFFFF;
        auto write = [&](uint32_t* job, uint32_t j, const MoeDiv& width) __attribute__((always_inline)) {
            uint32_t s = slot;
            for (int i = 0; i < 8; ++i)
                for (uint32_t left = cnt[i]; left > 0; ++j) {
                    const uint32_t n = left < width.d ? left : width.d;
                    job[j] = (uint32_t)(8 * lane + i) | s << 9 | n << 20;
                    s += n;
                    left -= n;
                }
        };
        write(S.job, (uint32_t)((upto - own) >> 21) & 0x1FFFFF, P.width);
        if (blockIdx.x == 0) write(P.table->job, (uint32_t)((upto - own) >> 42), P.down_width);
        if (lane == 63) {
            S.jobs = (int)(upto >> 21) & 0x1FFFFF;
            if (blockIdx.x == 0) P.table->jobs = (int32_t)(upto >> 42);
        }
        for (int i = 0; i < 8; ++i) {
            S.first[8 * lane + i] = (uint16_t)slot;
            slot += cnt[i];
        }
    }
    __syncthreads();
    for (int at = tid; at < P.pairs; at += kMoeThreads) {            /* a lane a (token, choice) */
        const int t = P.choice.of(at), i = at - t * P.top_k, e = S.id[at];
        int slot = -1;
        if (e >= 0) {
            slot = S.first[e] + __popcll(S.mask[e] & ((1ull << t) - 1));
            S.tok[slot] = (uint8_t)t;
            S.slot_w[slot] = S.w[at];
        }
        if (blockIdx.x == 0) {                                       /* and what the others and the caller need */
            P.table->slot[at] = (int16_t)slot;
            if (P.ids) P.ids[t * P.i_pitch + i] = e;
            if (P.weights) P.weights[t * P.wt_pitch + i] = S.w[at];
        }
    }
    __syncthreads();
}

/* ------------------------------------------------------------------------------ products */

/* Four results v[T][t] of row tiles T and token tiles t, of which lane (i / 4, j) holds rows i .. i + 3 of column j and the
 * class j % 4's is wanted: the sum over the classes of row lane / 16 and token lane / 4 % 4, of tile T = lane % 2 and
 * t = lane / 2 % 2.  A sum over four lanes each, and a choice. */
__device__ __forceinline__ float moe_value(r3d_f32x4 v00, r3d_f32x4 v10, r3d_f32x4 v01, r3d_f32x4 v11) {
    const bool b0 = threadIdx.x & 1, b1 = threadIdx.x & 2;
    auto mine = [&](r3d_f32x4 v) __attribute__((always_inline)) {
        const float lo = b0 ? v[1] : v[0], hi = b0 ? v[3] : v[2];
        return b1 ? hi : lo;
    };
    /* lanes 2 apart exchange what the other's token tile needs, then lanes beside each other the row tile's */
    const float p00 = mine(v00), p10 = mine(v10), p01 = mine(v01), p11 = mine(v11);
    auto from = [](float v, auto ctrl) __attribute__((always_inline)) {
        return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(ctrl)::value, 15, 15, true));
    };
    using Two = std::integral_constant<int, 0x4E>;              /* lanes 2 3 0 1 of each four */
    using One = std::integral_constant<int, 0xB1>;              /* 1 0 3 2 */
    const float q0 = (b1 ? p01 : p00) + from(b1 ? p00 : p01, Two{});
    const float q1 = (b1 ? p11 : p10) + from(b1 ? p10 : p11, Two{});
    return (b0 ? q1 : q0) + from(b0 ? q0 : q1, One{});
}

/* Eight f32 values as sums of three bf16 ones each: the bits of a number cut in three, eight each.  Infinities and NaN (quiet ones,
 * as arithmetic leaves them) stand alone. */
__device__ __forceinline__ void moe_parts(r3d_i32x4 lo, r3d_i32x4 hi, r3d_i32x4 (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = __int_as_float(i < 2 ? lo[2 * i] : hi[2 * i - 4]), b = __int_as_float(i < 2 ? lo[2 * i + 1] : hi[2 * i - 3]);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            part[p][i] = (int)__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);   /* the upper halves */
            a = __builtin_fabsf(a) < __builtin_inff() ? a - __uint_as_float(__float_as_uint(a) & 0xFFFF0000u) : 0.0f;
            b = __builtin_fabsf(b) < __builtin_inff() ? b - __uint_as_float(__float_as_uint(b) & 0xFFFF0000u) : 0.0f;
        }
    }
}

/* LDS that a row of K columns in XH parts takes: whole 1 KB pieces, and what keeps the pieces that eight lanes read, four of
 * two tokens, apart. */
constexpr int moe_row(int64_t K, int parts, int enc) {
    return (int)(parts * ((2 * K + 1023) / 1024) * 1024 + (enc == MOE_BF16 ? 64 : 16));
}

/* L spans of 4 KB a step.  A row's last step may be short, and what it lacks is missing in flight: e2m1 takes two a step, and
 * three where a row of h has three, nine, .. (f = 1344, top 8 of 128: 64 tokens 315 -> 301 us, 8 105 -> 102, one 32.6 -> 32.7; 64 x 4 /
 * 64, n = 4096, f = 1536 137.6 -> 137.2; elsewhere three are up to 2 % slower).  The others have two steps of one in flight. */
template <int ENC, int CT, bool UP, int L>
__global__ __launch_bounds__(kMoeThreads) void moe_stream_kernel(MoeArgs P) {
    constexpr int N = MoeCodes<ENC>::N, X = MoeCodes<ENC>::X, XH = UP ? 1 : 3;   /* parts of a token's values */
    constexpr int D = ENC == MOE_FP4 ? 1 : 2;                        /* steps in flight */
    struct Jobs {
        uint32_t job[kMoeMaxPairs];
    };
    __shared__ typename std::conditional<UP, MoeChoice, Jobs>::type S;
    __shared__ float s_part[kMoeWaves][2][2][CT][64];            /* a wave's last unit and its first, where shared */
    __shared__ __attribute__((aligned(16))) float s_scale[ENC == MOE_I8 ? kMoeUnits * 16 : 1];
    extern __shared__ __attribute__((aligned(16))) uint8_t s_x[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int jobs;
    if constexpr (UP) {
        /* the arguments' loads go out here, beside the logits', and not where each is first used */
        asm volatile("" ::"s"(P.x), "s"(P.w), "s"(P.ws), "s"(P.w_expert), "s"(P.w_pitch), "s"(P.line.m), "s"(P.choice.m));
        moe_plan(P, S);
        jobs = i8_uniform(S.jobs);
    } else {
        constexpr int EACH = kMoeMaxPairs / kMoeThreads;
        uint32_t job[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) job[i] = P.table->job[EACH * tid + i];    /* what lies past the jobs is not used */
        jobs = P.table->jobs;
        asm volatile("" ::"s"(P.x), "s"(P.w), "s"(P.ws), "s"(P.w_expert), "s"(P.w_pitch), "s"(P.line.m), "s"(P.grid.m));
#pragma unroll
        for (int i = 0; i < EACH; ++i) S.job[EACH * tid + i] = job[i];
        __syncthreads();
    }
    const int r4 = (lane >> 2) & 3, cls = lane & 3, piece = (lane >> 4) * 4 + cls;   /* row, or column, and piece of a span */
    const int row1 = (lane >> 4) + 4 * (lane & 1), col1 = r4 + 2 * (lane & 2);       /* of the lane's result (moe_value) */
    const int nb = P.unit.d, spans = P.spans, pieces = P.K / N;      /* units a job */
    const int part_lds = P.cpr * 1024, row_lds = moe_row(P.K, XH, ENC);
    /* a run an XCD, so that its L2 sees few jobs' tokens */
    const uint32_t G = P.grid.d, per = G >> 3, rem = G & 7, xcd = blockIdx.x & 7;
    const uint32_t g = xcd * per + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
    const uint32_t units = (uint32_t)jobs * nb;                      /* times G under 2^32 (r3d_moe.h) */
    const int u_end = i8_uniform((int)P.grid.of(units * (g + 1)));
    const int64_t x_rows = UP ? P.M : P.pairs;
    const int64_t x_bytes = (x_rows - 1) * P.x_pitch + (UP ? 2 : 4) * (int64_t)P.K;
    const int64_t plane = (int64_t)((UP ? 2 * P.rows : P.rows) - 1) * P.w_pitch + (int64_t)pieces * 16;
    const int64_t s_plane = (int64_t)((UP ? 2 * P.rows : P.rows) - 1) * P.ws_pitch + pieces;

    for (int u = i8_uniform((int)P.grid.of(units * g)); u < u_end;) {
        /* as many units of the run as LDS holds the tokens (and the scales) of */
        const int j0 = i8_uniform((int)P.unit.of(u)), slot_base = i8_uniform((S.job[j0] >> 9) & 2047);
        int end = u, held = 0;
        for (int j = j0; end < u_end && end - u < (ENC == MOE_I8 ? kMoeUnits : 1 << 30); ++j) {
            const uint32_t job = i8_uniform(S.job[j]);
            const int upto = (int)((job >> 9) & 2047) + (int)(job >> 20) - slot_base;
            if (upto > P.job_rows) break;
            held = upto;
            end = (j + 1) * nb < u_end ? (j + 1) * nb : u_end;
        }
        if (ENC == MOE_I8 && end - u > kMoeUnits) end = u + kMoeUnits;
        if constexpr (ENC == MOE_I8) {
            for (int i = tid; i < 16 * (end - u); i += kMoeThreads) {
                const int un = u + (i >> 4), j = P.unit.of(un), blk = un - j * nb, r = i & 15;
                int row = UP ? (r >> 3) * P.rows + 8 * blk + (r & 7) : 16 * blk + r;
                if (!UP && row >= P.rows) row = P.rows - 1;
                s_scale[i] = reinterpret_cast<const float*>(P.ws)[(int64_t)(S.job[j] & 511) * P.ws_expert + row];
            }
        }
        /* this wave's spans, L a step and a unit's last ones fewer */
        const int total = (end - u) * spans;                         /* times 8 under 2^31 (r3d_moe.h) */
        const int a = i8_uniform(total * wave / kMoeWaves), b = i8_uniform(total * (wave + 1) / kMoeWaves);
        int tokens = 0;                                              /* of the rows to be held, a lane each */
        if constexpr (UP) tokens = lane < held ? S.tok[slot_base + lane] : 0;
        struct Step {
            r3d_i32x4 w[L][4];
            uint32_t s[L];                                           /* e2m1: four scales of row lane / 4, a span each */
        } ring[D];
        const int ua = i8_uniform((int)P.line.of(a));
        int ll = a - ua * spans, lj = i8_uniform((int)P.unit.of(u + ua)), lb = u + ua - lj * nb, left = b - a;   /* where loads are */
        int cl = ll, cj = lj, cb = lb, cu = ua, todo = left;         /* where products are */
        __amdgpu_buffer_rsrc_t rW = r3d_rsrc(P.w, 0);
        const uint8_t* s_base = P.ws;
        uint32_t w_at[2] = {0, 0}, s_at[2] = {0, 0};
        bool both = true, entered = false;
        /* A span's scales are 16 bytes of each of the 16 rows, a byte a lane and row tile.  A step loads them four a lane, at
         * any alignment (the plane's last four in place of some that lie past it), 16 bytes of a row by four lanes beside
         * each other; a lane's byte is then another lane's. */
        const uint32_t s_last = (uint32_t)s_plane - 4;
        auto load = [&](Step& st) __attribute__((always_inline)) {
            const int n = left < spans - ll ? left : spans - ll;     /* 0: the wave's spans are done */
            if (n > 0 && (ll == 0 || !entered)) {                    /* a unit's first line here */
                entered = true;
                const int64_t e = i8_uniform(S.job[lj]) & 511;
                rW = r3d_rsrc(P.w + e * P.w_expert, plane);
                if (ENC == MOE_FP4) s_base = P.ws + e * P.ws_expert;
                const uint32_t r0 = (UP ? 8 : 16) * lb, r1 = UP ? r0 + P.rows : r0 + 8;
                both = UP || (int)r1 < P.rows;
                w_at[0] = r0 * (uint32_t)P.w_pitch;
                w_at[1] = r1 * (uint32_t)P.w_pitch;
                s_at[0] = r0 * (uint32_t)P.ws_pitch;
                s_at[1] = r1 * (uint32_t)P.ws_pitch;
            }
            const uint32_t wo = (uint32_t)(r4 * P.w_pitch + 16 * piece);
            if (ENC == MOE_FP4) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    typedef uint32_t u32_u1 __attribute__((aligned(1)));
                    const uint32_t o = (lane < 32 ? s_at[0] : s_at[1]) + ((lane >> 2) & 7) * (uint32_t)P.ws_pitch + 16 * (ll + i) + 4 * cls;
                    st.s[i] = *reinterpret_cast<const u32_u1*>(s_base + (o < s_last ? o : s_last));
                }
            }
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const bool in = i < n && 16 * (ll + i) + piece < pieces;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    st.w[i][r] = i8_buf16<2>(rW, in && (r < 2 || both) ? wo : kI8Oob,
                                             w_at[r >> 1] + (r & 1) * 4 * (uint32_t)P.w_pitch + 256 * (ll + i));
            }
            const int m = n < L ? n : L;
            left -= m;
            ll += m;
            if (ll == spans) {
                ll = 0;
                if (++lb == nb) {
                    lb = 0;
                    ++lj;
                }
            }
        };
#pragma unroll
        for (int d = 0; d < D; ++d) {
            load(ring[d]);
            __builtin_amdgcn_sched_barrier(0);                       /* in this order everywhere: a step waits for its own */
        }
        /* behind the weights' loads, and with no read of LDS among them, which would wait for them all */
        const __amdgpu_buffer_rsrc_t rX = r3d_rsrc(P.x, x_bytes);
        if constexpr (UP) {
            for (int c = wave; c < P.cpr; c += kMoeWaves) {          /* the tokens: 1 KB of each row a turn */
                const uint32_t at = 1024 * c + 16 * lane;            /* past the row's end: zeros */
                const bool in = at < 2 * (uint32_t)P.K;
                for (int r = 0; r < held; ++r) {
                    const int row = __builtin_amdgcn_readlane(tokens, r & 63);
                    r3d_buf_lds<16>(rX, s_x + r * row_lds + 1024 * c, in ? (uint32_t)row * (uint32_t)P.x_pitch + at : kI8Oob, 0);
                }
            }
        } else {
            constexpr int B = 4;                                     /* h: 512 columns of a row a wave, B of them in flight */
            const int items = held * P.cpr;
            for (int c0 = wave; c0 < items; c0 += B * kMoeWaves) {
                r3d_i32x4 v[B][2];
                uint32_t to[B];
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const int c = c0 + i * kMoeWaves, r = i8_uniform((int)P.chunk.of(c)), k = c - r * P.cpr;
                    const uint32_t col = 512 * k + 8 * lane;         /* past the row's end: zeros */
                    const bool in = c < items && col < (uint32_t)P.K;
                    const uint32_t at = in ? (uint32_t)(slot_base + r) * (uint32_t)P.x_pitch + 4 * col : kI8Oob;
                    v[i][0] = i8_buf16<0>(rX, at, 0);
                    v[i][1] = i8_buf16<0>(rX, at, 16);
                    to[i] = r * row_lds + 1024 * k + 16 * lane;
                }
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    if (c0 + i * kMoeWaves >= items) break;
                    r3d_i32x4 part[3];
                    moe_parts(v[i][0], v[i][1], part);
#pragma unroll
                    for (int p = 0; p < 3; ++p) *reinterpret_cast<r3d_i32x4*>(s_x + to[i] + p * part_lds) = part[p];
                }
            }
        }
        __syncthreads();

        int slot0 = 0, cnt = 0;
        uint32_t xa[2 * CT];
        auto job_of = [&](int j) __attribute__((always_inline)) {
            const uint32_t job = i8_uniform(S.job[j]);
            slot0 = (job >> 9) & 2047;
            cnt = job >> 20;
#pragma unroll
            for (int t = 0; t < 2 * CT; ++t)                         /* a column without a token repeats the first one's */
                xa[t] = (slot0 - slot_base + (4 * t + r4 < cnt ? 4 * t + r4 : 0)) * row_lds + 16 * X * piece;
        };
        if (a < b) job_of(cj);
        const int s_turn = (8 * cls + 9) & 31;
        const int s_from = 4 * (4 * r4 + (lane >> 4));               /* plus 16 lanes a row tile */
        uint32_t c_at[2] = {(uint32_t)((UP ? 8 : 16) * cb) * (uint32_t)P.ws_pitch, 0};
        c_at[1] = c_at[0] + (uint32_t)(UP ? P.rows : 8) * (uint32_t)P.ws_pitch;
        r3d_f32x4 acc[4][2 * CT];
        auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < 2 * CT; ++t) acc[r][t] = r3d_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        };
        /* a whole unit's results */
        auto finish = [&](int un, int blk, const float (&val)[2][CT]) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int col = 8 * t + col1;
                const int64_t slot = slot0 + (col < cnt ? col : 0);
                float v[2] = {val[0][t], val[1][t]};
                if constexpr (ENC == MOE_I8) {
                    v[0] *= s_scale[16 * un + row1];
                    v[1] *= s_scale[16 * un + 8 + row1];
                }
                if constexpr (UP) {
                    act_values<1>(P.act, v);
                    const float h = v[0] * v[1] * S.slot_w[slot];
                    if (col < cnt) P.out[slot * P.rows + 8 * blk + row1] = h;
                } else if (col < cnt) {
                    float* const to = P.out + slot * P.rows + 16 * blk + row1;
                    to[0] = P.add ? to[0] + v[0] : v[0];
                    if (16 * blk + 8 < P.rows) to[8] = P.add ? to[8] + v[1] : v[1];
                }
            }
        };
        clear();
        bool whole = cl == 0;                                        /* this wave has the unit from its first line on */
        while (todo > 0) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (todo > 0) {
                    int n = todo < spans - cl ? todo : spans - cl;
                    n = n < L ? n : L;
                    /* e2m1: a step with pieces past the row, or with scales that loads past the plane's end stand for */
                    const bool edge = 16 * (cl + n) > pieces || c_at[1] + 7 * (uint32_t)P.ws_pitch + 16 * cl + 32 > s_last;
#pragma unroll
                    for (int i = 0; i < L; ++i) {
                        if (i >= n) break;
                        uint32_t scale[4] = {0, 0, 0, 0};
                        if constexpr (ENC == MOE_FP4) {
                            /* byte cls of the dword lane / 16 of the row's span, to bits 23-30 */
                            uint32_t four[4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) four[r] = (uint32_t)__builtin_amdgcn_ds_bpermute(s_from + 64 * r, (int)ring[d].s[i]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) scale[r] = __builtin_amdgcn_alignbit(four[r], four[r], s_turn);
                            if (edge) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const uint32_t o = c_at[r >> 1] + ((4 * r + r4) & 7) * (uint32_t)P.ws_pitch + 16 * (cl + i) + (piece & 12);
                                    const uint32_t back = o < s_last ? 0 : o - s_last;
                                    scale[r] = __builtin_amdgcn_ubfe(four[r], 8 * (back + cls), 8) << 23;
                                    /* past the row: 2^-127 of its zeros, not the next row's */
                                    scale[r] = 16 * (cl + i) + piece < pieces ? scale[r] : 0u;
                                }
                            }
                        }
#pragma unroll
                        for (int h = 0; h < CT; ++h) {
                            if (h > 0 && 8 * h >= cnt) break;        /* columns without a token */
                            const bool two = 8 * h + 4 < cnt;
                            r3d_i32x4 x[2][XH * X];
#pragma unroll
                            for (int k = 0; k < XH * X; ++k)
                                x[0][k] = *reinterpret_cast<const r3d_i32x4*>(
                                    s_x + xa[2 * h] + k / X * part_lds + 256 * X * (cl + i) + 16 * (k % X));
                            if (two) {
#pragma unroll
                                for (int k = 0; k < XH * X; ++k)
                                    x[1][k] = *reinterpret_cast<const r3d_i32x4*>(
                                        s_x + xa[2 * h + 1] + k / X * part_lds + 256 * X * (cl + i) + 16 * (k % X));
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                r3d_i32x4 w[X];
                                moe_bf16<ENC>(ring[d].w[i][r], scale[r], w);
#pragma unroll
                                for (int k = 0; k < XH * X; ++k) acc[r][2 * h] = moe_mfma(w[k % X], x[0][k], acc[r][2 * h]);
                                if (two) {
#pragma unroll
                                    for (int k = 0; k < XH * X; ++k) acc[r][2 * h + 1] = moe_mfma(w[k % X], x[1][k], acc[r][2 * h + 1]);
                                }
                            }
                        }
                    }
                    cl += n;
                    todo -= n;
                    if (cl == spans || todo == 0) {                  /* the unit's end, or the run's */
                        float val[2][CT];
#pragma unroll
                        for (int t = 0; t < CT; ++t) {
                            val[0][t] = moe_value(acc[0][2 * t], acc[1][2 * t], acc[0][2 * t + 1], acc[1][2 * t + 1]);
                            val[1][t] = moe_value(acc[2][2 * t], acc[3][2 * t], acc[2][2 * t + 1], acc[3][2 * t + 1]);
                        }
                        if (whole && cl == spans) {
                            finish(cu, cb, val);
                        } else {
#pragma unroll
                            for (int t = 0; t < CT; ++t)
#pragma unroll
                                for (int r = 0; r < 2; ++r) s_part[wave][whole ? 0 : 1][r][t][lane] = val[r][t];
                        }
                        if (cl == spans) {
                            clear();
                            whole = true;
                            cl = 0;
                            ++cu;
                            if (++cb == nb) {
                                cb = 0;
                                if (todo > 0) job_of(++cj);
                            }
                            if (ENC == MOE_FP4) {
                                c_at[0] = (uint32_t)((UP ? 8 : 16) * cb) * (uint32_t)P.ws_pitch;
                                c_at[1] = c_at[0] + (uint32_t)(UP ? P.rows : 8) * (uint32_t)P.ws_pitch;
                            }
                        }
                    }
                }
                load(ring[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
        if (a < b && cl > 0 && whole) {                              /* begun here, ended by the waves after */
            const int stop = (cu + 1) * spans;
            float val[2][CT];
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float v = s_part[wave][0][r][t][lane];
                    for (int o = wave + 1; o < kMoeWaves; ++o) {
                        const int ao = total * o / kMoeWaves;
                        if (ao >= stop) break;
                        if (ao < total * (o + 1) / kMoeWaves) v += s_part[o][1][r][t][lane];
                    }
                    val[r][t] = v;
                }
            finish(cu, cb, val);
        }
        u = end;
        if (u < u_end) __syncthreads();                              /* the scales are read */
    }
}

/* y of the slots' sums: four columns a lane, (ceil(n / 1024), M) workgroups of 256. */
__global__ __launch_bounds__(256) void moe_sum_kernel(const float* __restrict__ sums, const MoeTable* __restrict__ table,
                                                      void* y, int64_t y_pitch, int n, int top_k, int y_bf16) {
    const int m = blockIdx.y, c = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (c >= n) return;                                              /* n is a multiple of 8 */
    r3d_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int U = 8;                                             /* loads in flight (1 x 8 / 128 35.2 us by ones, 32.5) */
    for (int i = 0; i < top_k; i += U) {
        int slot[U];
        r3d_f32x4 s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) slot[u] = table->slot[m * top_k + (i + u < top_k ? i + u : top_k - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            s[u] = *reinterpret_cast<const r3d_f32x4*>(sums + (int64_t)(slot[u] < 0 ? 0 : slot[u]) * n + c);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u < top_k && slot[u] >= 0) v += s[u];
    }
    if (y_bf16)
        *reinterpret_cast<r3d_u32x2_u2*>(static_cast<uint16_t*>(y) + m * y_pitch + c) =
            r3d_u32x2_u2{r3d_pack_bf16x2(v[0], v[1]), r3d_pack_bf16x2(v[2], v[3])};
    else
        *reinterpret_cast<r3d_f32x4_u4*>(static_cast<float*>(y) + m * y_pitch + c) = v;
}

template <int ENC>
static int moe_launch(const MoePlan& P, const MoeGeom& g, void* scratch, hipStream_t stream) {
    MoeTable* const table = static_cast<MoeTable*>(scratch);
    const int64_t pairs = P.M * P.top_k;
    float* const h = reinterpret_cast<float*>(table + 1);
    float* const sums = h + moe_h_bytes(P) / 4;
    const auto div = [](int64_t d) { return MoeDiv{(uint32_t)d, (uint32_t)(0xFFFFFFFFu / (uint32_t)d)}; };
    const auto spans = [](int64_t K) { return (K / MoeCodes<ENC>::N + 15) / 16; };
    const auto loads = [](int64_t K) { return (int)((2 * K + 1023) / 1024); };
    const MoeArgs u{table, P.logits, P.l_pitch, (int)P.M, (int)P.E, (int)P.top_k, P.l_bf16, (int)P.n, (int)P.f, (int)pairs,
                    (int)P.x_pitch, P.x, P.gu, P.gus, h, P.gu_expert, P.gus_expert, P.gus_pitch, (int)P.gu_pitch, g.up.rows,
                    (int)spans(P.n), loads(P.n), div(P.f / 8), div(spans(P.n)), div(g.blocks), div(P.top_k),
                    div(loads(P.n)), P.ids, P.weights, P.i_pitch, P.w_pitch, div(g.up.width), div(g.down.width), P.act, P.sigmoid,
                    P.renorm, P.weight_scale};
    if (P.M > kMoeWaves) hipLaunchKernelGGL(moe_route_kernel, dim3((unsigned)P.M), dim3(64), 0, stream, u);
    constexpr int L = ENC == MOE_FP4 ? 2 : 1, L3 = ENC == MOE_FP4 ? 3 : 1;
    const dim3 grid((unsigned)g.blocks), block(kMoeThreads);
    const size_t up_lds = (size_t)g.up.rows * moe_row(P.n, 1, ENC);
    if (g.up.ct == 1) hipLaunchKernelGGL((moe_stream_kernel<ENC, 1, true, L>), grid, block, up_lds, stream, u);
    else hipLaunchKernelGGL((moe_stream_kernel<ENC, 2, true, L>), grid, block, up_lds, stream, u);
    hipError_t e = hipGetLastError();
    for (int part = 0; part < g.parts && e == hipSuccess; ++part) {
        const int64_t k0 = part * g.spans * moe_span(ENC), left = P.f - k0;
        const int64_t K = part + 1 < g.parts ? g.spans * moe_span(ENC) : left;
        MoeArgs d{table, nullptr, 0, (int)P.M, (int)P.E, (int)P.top_k, 0, (int)K, (int)P.n, (int)pairs, (int)(4 * P.f),
                  reinterpret_cast<const uint8_t*>(h + k0), P.dn + part * g.spans * 256, P.dns, sums, P.dn_expert, P.dns_expert,
                  P.dns_pitch, (int)P.dn_pitch, g.down.rows, (int)spans(K), loads(K), div((P.n + 15) / 16), div(spans(K)),
                  div(g.blocks), div(P.top_k), div(loads(K))};
        if (ENC == MOE_FP4) d.ws += part * g.spans * 16;
        d.add = part > 0;
        const size_t lds = (size_t)g.down.rows * moe_row(K, 3, ENC);
        constexpr int CT = ENC == MOE_BF16 ? 2 : 1;
        if (g.down.ct == 2) hipLaunchKernelGGL((moe_stream_kernel<ENC, CT, false, L>), grid, block, lds, stream, d);
        else if (d.spans % 6 == 3) hipLaunchKernelGGL((moe_stream_kernel<ENC, 1, false, L3>), grid, block, lds, stream, d);
        else hipLaunchKernelGGL((moe_stream_kernel<ENC, 1, false, L>), grid, block, lds, stream, d);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        hipLaunchKernelGGL(moe_sum_kernel, dim3((unsigned)((P.n + 1023) / 1024), (unsigned)P.M), dim3(256), 0, stream, sums,
                           table, P.y, P.y_pitch, (int)P.n, (int)P.top_k, P.y_bf16);
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
    if (!moe_geom(P, cu_count(), &g)) return RAD_E_UNSUPPORTED;
    hipStream_t t = (hipStream_t)s;
    return P.enc == MOE_BF16 ? moe_launch<MOE_BF16>(P, g, a->scratch, t)
           : P.enc == MOE_I8 ? moe_launch<MOE_I8>(P, g, a->scratch, t)
                             : moe_launch<MOE_FP4>(P, g, a->scratch, t);
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
