/* r3d_sample.hip -- the sample_logits row: one token a row of logits from a given uniform number.
 *
 * With z = (x - max) / T and w = exp(z) of a row's tokens (NaN and -inf: not there),
 *   top-k  keeps the k first by (x falling, index rising);
 *   top-p  keeps of those the shortest prefix whose mass is at least p times their mass, one at least;
 *   min-p  keeps of those the ones with w >= min_p (w of the likeliest token is 1);
 * and the token is the first kept one, in index order, at which the running mass passes u times the
 * kept mass.  T <= 0 (or NaN) takes the lowest index of the maximum.  A row with nothing in it gives
 * token -1 and probability 0.
 *
 * Masses are 64-bit integers, w * 2^s to nearest with V 2^s < 2^63, s <= 51 (44 at V = 262144), from an
 * exp in f64: integer sums do not depend on their order, so atomics may make them, a cut and the
 * search see the same numbers, and a run repeats bit for bit.  A border moves by about
 * 2^-s sqrt(V) / mass, 2^-35 at V = 262144, where f32 sums would move it by 2^-20 and pick a
 * neighbour now and then.
 *
 * A row is sorted nowhere; its cuts are looked for where they can be.  Four launches, for all rows:
 *   1 the largest and least logit of every quarter of a segment (4096 tokens), and the largest of every
 *     chunk (64 tokens).  Of a row without a cut also the quarters' sums of w, in f64: that row needs
 *     no other pass but the last.  Greedy rows need the largest logits only
 *   2 of rows whose cut may lie anywhere (top-p without a small top-k, or a top-k of more than a chunk in
 *     four): count and mass in 2048 bins, of equal width in x over the row's range (at most 32 T: below
 *     that w is 0); bins are in the order of x, so a cut falls into one bin
 *   3 of these rows the border bins are found from the 2048 sums; the tokens above them are added up a
 *     segment at a time, the tokens in them are listed.  Chunks below the borders are not read
 *   4 a workgroup a row: the listed tokens are sorted, the cuts placed, the segment that holds u * mass
 *     found, and the token in it.  Rows with a small top-k, or with min-p alone, are listed here: k chunks
 *     whose largest logits are the k largest such hold the k first tokens above the least of those, so
 *     only chunks above that are read.  Past 8192 listed tokens (many equal logits) the cuts are
 *     placed by radix selection over the row instead.
 * Passes 2 and 3 are not launched without a top-k or top-p operand.
 *
 * Bound by the one read of the row in pass 1 and by the four launches' chains of dependent loads.
 * Measured on MI355X at V = 262144, f32: one row 8 us greedy, 13 without a cut, 15 with min-p, 21, 22 and 26 with a
 * top-k of 50, 200 and 1000 (of those 12, 14 and 19 in pass 4), 47 with top-p alone; 128 rows, each with settings of
 * its own, 86 to 92 us (of which pass 1's read of 134 MB 29 us, 4.6 TB/s; passes 2 and 3, f64 exps for the 22
 * to 30 rows that have a use for them, 16 to 20 and 19 to 25; pass 4 23, of them 6 to list 1000 chunks).  bf16: the
 * same within a tenth (pass 1 25, pass 4 27).  With bins for every row, no chunks and a sort that waited at a
 * barrier for every step one row took 27.7 and 128 143 us.
 * The radix selection over the row takes 2.2 ms (2.5 with top-p as well, 4.1 so over a row of equal logits): some
 * eight sweeps by one workgroup, half of them with an exp and two atomics a token, nearly all at one address.  A mask
 * of a finite number leads there where a small top-k asks for more tokens than are allowed; one of -inf does
 * not. */
#include <hip/hip_runtime.h>

#include <stdio.h>

#include "r3d_device.h"
#include "r3d_dump.h"
#include "r3d_plan.h"
#include "r3d_sample.h"
#include "r3d_wave.h"

namespace r3d {

bool chip_ok();                  /* r3d_gemm.hip */

typedef unsigned long long u64;

struct SampleArgs {
    SamplePlan P;
    SampleRow* rows;
    u64* seg_mass;               /* [M][segs] */
    double* q_sum;               /* [M][4 segs], of every quarter of a segment: rows without a cut, the sum of
                                    exp((x - its largest) / T); */
    float* q_max;                /* its largest */
    float* q_min;                /* and least logit */
    float* chunk_max;            /* [M][64 segs] */
    int segs, per, shift;        /* per: segments a workgroup; shift: s of the masses */
};

/* A row's settings, and what its tokens are measured against. */
struct SampleSet {
    float top;                   /* the largest logit; -inf: the row is empty */
    float bin;                   /* bins a unit of x */
    float T;
    double inv_t, p, min_p;
    int k;
    bool greedy, use_k, use_p;
    bool listed;                 /* cut by a small top-k, or by min-p alone: the row's last pass lists
                                    what can be kept by way of the chunks' maxima */
    bool plain;                  /* no cut at all */
    bool binned;                 /* the others that are not greedy: passes 2 and 3 */
};

__device__ __forceinline__ SampleSet sample_set(const SampleArgs& a, int64_t row) {
    const SamplePlan& P = a.P;
    SampleSet s;
    const float T = P.temperature ? P.temperature[row * P.t_stride] : 1.0f;
    const int k = P.top_k ? P.top_k[row * P.k_stride] : 0;
    const float p = P.top_p ? P.top_p[row * P.p_stride] : 1.0f;
    const float m = P.min_p ? P.min_p[row * P.m_stride] : 0.0f;
    s.top = s.bin = 0.0f;
    s.T = T;
    s.greedy = !(T > 0.0f);
    s.inv_t = 1.0 / (double)T;
    s.k = k;
    s.use_k = k > 0 && k < P.V;
    s.p = (double)p;
    s.use_p = p < 1.0f;
    s.min_p = m > 0.0f ? (m < 1.0f ? (double)m : 1.0) : 0.0;
    s.plain = !s.use_k && !s.use_p && s.min_p == 0.0;
    s.listed = s.use_k ? P.V <= kSampleList || (k <= kSampleListK && k <= (P.V / kSampleChunk) / 4)
                       : !s.use_p && s.min_p > 0.0;
    s.binned = !s.greedy && !s.plain && !s.listed;
    return s;
}

/* exp(z) for z <= 0, within 2^-50: z = n ln 2 + r, |r| <= ln 2 / 2, the series of exp(r) to r^12
 * (r^13 / 13! < 2^-52), times 2^n.  Past the least f64 (and for NaN, which the maximum passes over) 0. */
__device__ __forceinline__ double sample_exp(double z) {
    z = __builtin_fmax(z, -1100.0);
    const double n = __builtin_rint(z * 1.4426950408889634);
    double r = __builtin_fma(n, -0.6931471824645996, z);          /* ln 2 in f32 (n times it is exact), */
    r = __builtin_fma(n, 1.904654299957768e-09, r);                /* and what is left of it */
    double e = 1.0 / 479001600.0;
    e = __builtin_fma(e, r, 1.0 / 39916800.0);
    e = __builtin_fma(e, r, 1.0 / 3628800.0);
    e = __builtin_fma(e, r, 1.0 / 362880.0);
    e = __builtin_fma(e, r, 1.0 / 40320.0);
    e = __builtin_fma(e, r, 1.0 / 5040.0);
    e = __builtin_fma(e, r, 1.0 / 720.0);
    e = __builtin_fma(e, r, 1.0 / 120.0);
    e = __builtin_fma(e, r, 1.0 / 24.0);
    e = __builtin_fma(e, r, 1.0 / 6.0);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return __builtin_amdgcn_ldexp(e, (int)n);
}

__device__ __forceinline__ bool sample_in(float x) { return x > -__builtin_inff(); }   /* NaN: no */

__device__ __forceinline__ double sample_w(const SampleSet& s, float x) {
    return x == s.top ? 1.0 : sample_exp(((double)x - (double)s.top) * s.inv_t);
}
/* w 2^shift to nearest, w 2^shift < 2^52: in the low bits of w 2^shift + 2^52. */
__device__ __forceinline__ u64 sample_mass(double w, int shift) {
    const double big = 4503599627370496.0;
    return (u64)__double_as_longlong(__builtin_fma(w, __longlong_as_double((long long)(1023 + shift) << 52), big)) -
           (u64)__double_as_longlong(big);
}
/* The same to 2^63, for sums. */
__device__ __forceinline__ u64 sample_mass_sum(double w, int shift) {
    return (u64)__builtin_rint(w * __longlong_as_double((long long)(1023 + shift) << 52));
}
__device__ __forceinline__ int sample_bin(const SampleSet& s, float x) {
    return x == s.top ? 0 : (int)__builtin_fminf((s.top - x) * s.bin, (float)(kSampleBins - 1));
}
/* Bits in the order of x, -0 as 0. */
__device__ __forceinline__ uint32_t sample_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ const uint8_t* sample_row(const SamplePlan& P, int64_t row) {
    return P.logits + row * P.pitch * (P.bf16 ? 2 : 4);
}

template <bool BF16>
__device__ __forceinline__ float sample_ld1(const uint8_t* x, int64_t i) {
    return BF16 ? r3d_bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i]) : reinterpret_cast<const float*>(x)[i];
}
/* Four logits from index i on; -inf past V. */
template <bool BF16>
__device__ __forceinline__ void sample_ld4(const uint8_t* x, int64_t i, int64_t V, float* v) {
    if (i + 4 <= V) {
        if (BF16) {
            const r3d_u32x2_u2 d = *reinterpret_cast<const r3d_u32x2_u2*>(x + 2 * i);
            v[0] = __uint_as_float(d[0] << 16);
            v[1] = __uint_as_float(d[0] & 0xFFFF0000u);
            v[2] = __uint_as_float(d[1] << 16);
            v[3] = __uint_as_float(d[1] & 0xFFFF0000u);
        } else {
            const r3d_f32x4_u4 d = *reinterpret_cast<const r3d_f32x4_u4*>(x + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = d[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = -__builtin_inff();
            if (i + j < V) v[j] = sample_ld1<BF16>(x, i + j);
        }
    }
}

constexpr int kSampleT = 256;                      /* lanes of passes 1 to 3 */
constexpr int kSampleU = kSampleSeg / 4 / 64 / 4;    /* loads a lane and quarter of a segment */

/* A lane's loads are in flight together and worked on one after the other from the same registers:
 * unrolled, 16 exps side by side need twice the registers and four times the code. */
template <int U>
__device__ __forceinline__ void sample_next(float (*v)[4]) {
#pragma unroll
    for (int j = 0; j + 1 < U; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = v[j + 1][i];
}

/* Over a workgroup of T lanes, up to 16 waves: their own results meet in 16 lanes of every wave. */
template <int T>
__device__ __forceinline__ float sample_block_max(float v, float* s) {
    const int lane = threadIdx.x & 63;
    v = r3d_max16(v);
#pragma unroll
    for (int off = 32; off >= 16; off >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, off, 64));
    __syncthreads();
    if (lane == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return r3d_max16(s[lane & (T / 64 - 1)]);
}
/* The sum over the lanes before this one; *total over all. */
template <int T, class V>
__device__ __forceinline__ V sample_block_scan(V v, V* s, V* total) {
    const V in = r3d_wave_scan(v);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __syncthreads();
    if (lane == 63) s[wave] = in;
    __syncthreads();
    const V waves = r3d_scan16(s[lane & (T / 64 - 1)]);
    *total = r3d_lane(waves, T / 64 - 1);
    return (wave ? r3d_lane(waves, wave - 1) : V(0)) + (in - v);
}
template <int T>
__device__ __forceinline__ u64 sample_block_sum(u64 v, u64* s) {
    u64 total;
    sample_block_scan<T>(v, s, &total);
    return total;
}

/* The row's largest and least logit from its quarters', into the set. */
template <int T>
__device__ __forceinline__ void sample_range(const SampleArgs& a, int64_t row, float* s, SampleSet* set) {
    float hi = -__builtin_inff(), lo = __builtin_inff();
    for (int i = threadIdx.x; i < 4 * a.segs; i += T) {
        hi = __builtin_fmaxf(hi, a.q_max[row * 4 * a.segs + i]);
        lo = __builtin_fminf(lo, a.q_min[row * 4 * a.segs + i]);
    }
    hi = sample_block_max<T>(hi, s);
    lo = -sample_block_max<T>(-lo, s);
    set->top = hi;
    set->bin = (float)(kSampleBins - 1) / __builtin_fminf(hi - lo, 32.0f * set->T);
}

/* Pass 1: a wave a quarter of a segment at a time, no barrier.  Bound by the read. */
template <bool BF16>
__global__ __launch_bounds__(kSampleT) void sample_range_kernel(SampleArgs a) {
    const int64_t row = blockIdx.y;
    if (row == 0 && blockIdx.x == 0) {
        __shared__ unsigned int on[kSampleT / 64];
        int n = 0;
        for (int64_t r0 = 0; r0 < a.P.M; r0 += kSampleT) {
            const u64 mask = __ballot(r0 + threadIdx.x < a.P.M && sample_set(a, r0 + threadIdx.x).binned);
            if ((threadIdx.x & 63) == 0) on[threadIdx.x >> 6] = (unsigned int)__builtin_popcountll(mask);
            __syncthreads();
            int at = n + __builtin_popcountll(mask & (((u64)1 << (threadIdx.x & 63)) - 1));
#pragma unroll
            for (int i = 0; i < kSampleT / 64; ++i) {
                if (i < (int)threadIdx.x >> 6) at += (int)on[i];
                n += (int)on[i];
            }
            if (mask >> (threadIdx.x & 63) & 1) a.rows[at].binned = (int)(r0 + threadIdx.x);
            __syncthreads();
        }
        if (threadIdx.x == 0) a.rows[0].n_binned = n;
    }
    const SampleSet set = sample_set(a, row);
    if (set.binned) {
        SampleRow& R = a.rows[row];
        for (int i = blockIdx.x * kSampleT + threadIdx.x; i < kSampleBins; i += gridDim.x * kSampleT) {
            R.mass[i] = 0;
            R.count[i] = 0;
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) R.n_list = 0;
    }
    const uint8_t* x = sample_row(a.P, row);
    const int lane = threadIdx.x & 63;
    const int s1 = ((int)blockIdx.x + 1) * a.per < a.segs ? ((int)blockIdx.x + 1) * a.per : a.segs;
    for (int seg = blockIdx.x * a.per; seg < s1; ++seg) {
        const int64_t q = (int64_t)seg * 4 + (threadIdx.x >> 6);
        float v[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sample_ld4<BF16>(x, q * (kSampleSeg / 4) + 4 * (lane + 64 * j), a.P.V, v[j]);
        float hi = -__builtin_inff(), lo = __builtin_inff();
        float* const cm = a.chunk_max + row * a.segs * kSampleSegChunks + q * (kSampleSegChunks / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float m = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m = __builtin_fmaxf(m, v[j][i]);                      /* a NaN is passed over */
                lo = __builtin_fminf(lo, sample_in(v[j][i]) ? v[j][i] : lo);
            }
            m = r3d_max16(m);
            if ((lane & 15) == 0) cm[lane / 16 + 4 * j] = m;
            hi = __builtin_fmaxf(hi, m);
        }
#pragma unroll
        for (int off = 32; off >= 16; off >>= 1) hi = __builtin_fmaxf(hi, __shfl_xor(hi, off, 64));
        lo = -r3d_max16(-lo);
#pragma unroll
        for (int off = 32; off >= 16; off >>= 1) lo = __builtin_fminf(lo, __shfl_xor(lo, off, 64));
        if (lane == 0) {
            a.q_max[row * 4 * a.segs + q] = hi;
            a.q_min[row * 4 * a.segs + q] = lo;
        }
        if (set.plain && !set.greedy) {
            SampleSet here = set;
            here.top = hi;
            double sum = 0.0;
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (sample_in(v[0][i])) sum += sample_w(here, v[0][i]);
                sample_next<kSampleU>(v);
            }
            sum = r3d_wave_scan(sum);
            if (lane == 63) a.q_sum[row * 4 * a.segs + q] = sum;
        }
    }
}

/* Passes 2 and 3, a wave a quarter of a segment at a time.  The binned rows are dealt out to
 * all workgroups, a row to as many as there are for it.  (Over every row's parts, where 22 of 128 rows
 * have something to do, some CUs had two or three of those and others none: 26 us for 17.) */
constexpr int kBinT = 1024, kBinWaves = kBinT / 64, kBinGrid = 256, kBinLeast = kBinWaves / 4;
constexpr unsigned int kBinList = 2048;
struct SampleShare {
    int items, parts, per;       /* shares in all, a row, and segments a share */
};
__device__ __forceinline__ SampleShare sample_share_out(const SampleArgs& a) {
    const int rows = a.rows[0].n_binned;
    int parts = rows ? (int)gridDim.x / rows : 1;
    if (parts < 1) parts = 1;
    int per = (a.segs + parts - 1) / parts;
    if (per < kBinLeast) per = kBinLeast;          /* a quarter a wave at least */
    parts = (a.segs + per - 1) / per;
    return {rows * parts, parts, per};
}

template <bool BF16>
__global__ __launch_bounds__(kBinT) void sample_hist_kernel(SampleArgs a) {
    __shared__ u64 mass[kSampleBins];
    __shared__ unsigned int count[kSampleBins];
    __shared__ float s[kBinT / 64];
    const SampleShare share = sample_share_out(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= share.items) return;
    const int64_t row = a.rows[blockIdx.x / share.parts].binned;
    const int s0 = (int)blockIdx.x % share.parts * share.per;
    const int s1 = s0 + share.per < a.segs ? s0 + share.per : a.segs;
    SampleSet set = sample_set(a, row);
    sample_range<kBinT>(a, row, s, &set);
    if (!sample_in(set.top)) return;
    for (int i = threadIdx.x; i < kSampleBins; i += kBinT) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    const uint8_t* x = sample_row(a.P, row);
    for (int q = 4 * s0 + wave; q < 4 * s1; q += kBinWaves) {
        float v[kSampleU][4];
#pragma unroll
        for (int j = 0; j < kSampleU; ++j)
            sample_ld4<BF16>(x, (int64_t)q * (kSampleSeg / 4) + 4 * (lane + 64 * j), a.P.V, v[j]);
#pragma unroll 1
        for (int j = 0; j < kSampleU; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sample_in(v[0][i])) {
                    const int b = sample_bin(set, v[0][i]);
                    if (set.use_k) atomicAdd(&count[b], 1u);
                    if (set.use_p) atomicAdd(&mass[b], sample_mass(sample_w(set, v[0][i]), a.shift));
                }
            sample_next<kSampleU>(v);
        }
    }
    __syncthreads();
    SampleRow& R = a.rows[row];
    for (int i = threadIdx.x; i < kSampleBins; i += kBinT) {
        if (count[i]) atomicAdd(&R.count[i], count[i]);
        if (mass[i]) atomicAdd(&R.mass[i], mass[i]);
    }
}

/* p's share of a mass, one at least. */
__device__ __forceinline__ u64 sample_share(double p, u64 mass) {
    const double t = __builtin_ceil(p * (double)mass);
    return t >= 1.0 ? (u64)t : 1;
}

/* From the bins' sums, a workgroup of T lanes. */
template <int T>
__device__ __forceinline__ void sample_cut(const SampleSet& set, const unsigned int* count, const u64* mass,
                                           u64* su, SampleCut* C) {
    constexpr int B = kSampleBins / T;             /* bins a lane */
    u64 c[B], m[B], cs = 0, ms = 0, all, total;
#pragma unroll
    for (int i = 0; i < B; ++i) {
        c[i] = count[B * threadIdx.x + i];
        m[i] = mass[B * threadIdx.x + i];
        cs += c[i];
        ms += m[i];
    }
    u64 c0 = sample_block_scan<T>(cs, su, &all);
    const u64 m0 = sample_block_scan<T>(ms, su, &total);
    if (threadIdx.x == 0) {
        C->kb = C->pb_lo = C->pb_hi = kSampleBins;
        C->count_k = 0;
        C->mass_k = C->mass_p = C->mass_kb = 0;
        C->total = total;
    }
    __syncthreads();
    u64 mm = m0;
    if (set.use_k && (u64)set.k <= all) {          /* (k of k listed ones are a cut of the row) */
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (c0 < (u64)set.k && c0 + c[i] >= (u64)set.k) {
                C->kb = B * threadIdx.x + i;
                C->mass_k = mm;
                C->mass_kb = m[i];
                C->count_k = (int)c0;
            }
            c0 += c[i];
            mm += m[i];
        }
    }
    __syncthreads();
    if (set.use_p) {
        /* the kept tokens' mass is known to within bin kb: the border of top-p to within these */
        const u64 lo = sample_share(set.p, C->kb < kSampleBins ? C->mass_k : total);
        const u64 hi = sample_share(set.p, C->kb < kSampleBins ? C->mass_k + C->mass_kb : total);
        mm = m0;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (mm < lo && mm + m[i] >= lo) {
                C->pb_lo = B * threadIdx.x + i;
                C->mass_p = mm;
            }
            if (mm < hi && mm + m[i] >= hi) C->pb_hi = B * threadIdx.x + i;
            mm += m[i];
        }
    }
    __syncthreads();
}
/* Bins below this one are kept whole. */
__device__ __forceinline__ int sample_whole(const SampleCut& C) { return C.kb < C.pb_lo ? C.kb : C.pb_lo; }
/* Tokens of a border bin are listed. */
__device__ __forceinline__ bool sample_border(const SampleCut& C, int b) {
    return b == C.kb || (b >= C.pb_lo && b <= C.pb_hi);
}
/* Places for this lane's c entries (BITS bits) of a list: the first.  By the bits' ballots: no lane waits
 * for another. */
template <int BITS>
__device__ __forceinline__ unsigned int sample_slots(unsigned int c, unsigned int* counter) {
    unsigned int before = 0, all = 0;
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const u64 m = __ballot(c >> b & 1);
        before += __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0)) << b;
        all += (unsigned)__builtin_popcountll(m) << b;
    }
    if (!all) return 0;
    unsigned int at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(counter, all);
    return __builtin_amdgcn_readfirstlane(at) + before;
}
__device__ __forceinline__ u64 sample_entry_of(float x, int64_t i) { return (u64)~sample_key(x) << 32 | (u64)i; }

template <bool BF16>
__global__ __launch_bounds__(kBinT) void sample_gather_kernel(SampleArgs a) {
    __shared__ u64 su[kBinT / 64];
    __shared__ float s[kBinT / 64];
    __shared__ SampleCut cut;
    __shared__ u64 sums[kSampleMaxSegs];
    __shared__ u64 part[kBinList];                 /* listed by this workgroup: one atomic for them all */
    __shared__ unsigned int n_part, part_at;
    const SampleShare share = sample_share_out(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= share.items) return;
    const int64_t row = a.rows[blockIdx.x / share.parts].binned;
    const int s0 = (int)blockIdx.x % share.parts * share.per;
    const int s1 = s0 + share.per < a.segs ? s0 + share.per : a.segs;
    SampleSet set = sample_set(a, row);
    sample_range<kBinT>(a, row, s, &set);
    if (!sample_in(set.top)) return;
    SampleRow& R = a.rows[row];
    if (threadIdx.x == 0) n_part = 0;
    for (int i = threadIdx.x; i < s1 - s0; i += kBinT) sums[i] = 0;
    sample_cut<kBinT>(set, R.count, R.mass, su, &cut);
    const SampleCut C = cut;
    if (s0 == 0 && threadIdx.x == 0) R.cut = C;
    const int whole = sample_whole(C);
    /* no token past bin `most` is kept or listed: a chunk whose largest logit lies there is not read */
    const int most = C.kb < kSampleBins ? C.kb : C.pb_hi < kSampleBins ? C.pb_hi : kSampleBins - 1;
    const uint8_t* x = sample_row(a.P, row);
    for (int q = 4 * s0 + wave; q < 4 * s1; q += kBinWaves) {
        const float* const cm = a.chunk_max + (row * 4 * a.segs + q) * (kSampleSegChunks / 4);
        float v[kSampleU][4];
#pragma unroll
        for (int j = 0; j < kSampleU; ++j) {
            const float m = cm[lane / 16 + 4 * j];
            if (sample_in(m) && sample_bin(set, m) <= most) {
                sample_ld4<BF16>(x, (int64_t)q * (kSampleSeg / 4) + 4 * (lane + 64 * j), a.P.V, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j][i] = -__builtin_inff();
            }
        }
        u64 sum = 0;
#pragma unroll 1
        for (int j = 0; j < kSampleU; ++j) {
            unsigned int border = 0;       /* a bit a token */
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!sample_in(v[0][i])) continue;
                const int b = sample_bin(set, v[0][i]);
                if (b < whole) {
                    const double w = sample_w(set, v[0][i]);
                    if (w >= set.min_p) sum += sample_mass(w, a.shift);
                } else if (sample_border(C, b)) {
                    border |= 1u << i;
                }
            }
            unsigned int at = sample_slots<3>(__builtin_popcount(border), &n_part);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (border >> i & 1) {
                    const u64 e = sample_entry_of(v[0][i], (int64_t)q * (kSampleSeg / 4) + 4 * (lane + 64 * j) + i);
                    if (at < kBinList) {
                        part[at] = e;
                    } else {               /* many equal logits */
                        const unsigned int g = atomicAdd(&R.n_list, 1u);
                        if (g < kSampleList) R.list[g] = e;
                    }
                    ++at;
                }
            sample_next<kSampleU>(v);
        }
        sum = r3d_wave_scan(sum);
        if (lane == 63 && sum) atomicAdd(&sums[q / 4 - s0], sum);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s1 - s0; i += kBinT) a.seg_mass[row * a.segs + s0 + i] = sums[i];
    const unsigned int n = n_part < kBinList ? n_part : kBinList;
    if (threadIdx.x == 0 && n) part_at = atomicAdd(&R.n_list, n);
    __syncthreads();
    for (unsigned int i = threadIdx.x; i < n; i += kBinT)
        if (part_at + i < kSampleList) R.list[part_at + i] = part[i];
}

constexpr int kPickT = 1024;
/* Pass 4's LDS, in 8 bytes: the list [8192], the segments' masses [1024], the bins' masses [2048] and counters
 * [2048 / 2] (or a radix pass's), the listed chunks' numbers [8192 / 2] */
constexpr int kPickSeg = kSampleList, kPickMass = kPickSeg + kSampleMaxSegs, kPickCount = kPickMass + kSampleBins;
constexpr int kPickWhich = kPickCount + kSampleBins / 2, kPickWords = kPickWhich + kSampleList / 2;

template <bool BF16>
__global__ __launch_bounds__(kPickT) void sample_pick_kernel(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) u64 smem[];
    u64* const list = smem;
    u64* const segm = smem + kPickSeg;
    u64* const hmass = smem + kPickMass;                          /* [bins], or [256] of a radix pass */
    unsigned int* const hcount = reinterpret_cast<unsigned int*>(smem + kPickCount);
    __shared__ u64 su[kPickT / 64];
    __shared__ float sf[kPickT / 64];
    __shared__ SampleCut s_cut;
    __shared__ u64 s_a, s_b;
    __shared__ int s_i, s_j;
    __shared__ unsigned int s_n, s_key;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x, V = a.P.V;
    const uint8_t* x = sample_row(a.P, row);
    int* const token = a.P.token + row * a.P.token_stride;
    float* const prob = a.P.prob ? a.P.prob + row * a.P.prob_stride : nullptr;
    /* the listed rows' chunk maxima, the first 4096 of them on their way before they are asked for */
    const float* const cm = a.chunk_max + row * a.segs * kSampleSegChunks;
    const int chunks = a.segs * kSampleSegChunks;
    float cv[4];
    auto load_chunks = [&](int i0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            cv[j] = i0 + t + kPickT * j < chunks ? cm[i0 + t + kPickT * j] : -__builtin_inff();
    };
    load_chunks(0);
    SampleSet set = sample_set(a, row);
    const float u = a.P.u[row * a.P.u_stride];
    sample_range<kPickT>(a, row, sf, &set);
    const float top = set.top;
    const float* const q_max = a.q_max + row * 4 * a.segs;
    if (!sample_in(top)) {
        if (t == 0) {
            *token = -1;
            if (prob) *prob = 0.0f;
        }
        return;
    }
    if (set.greedy) {
        if (t == 0) s_i = a.segs;
        __syncthreads();
        for (int i = t; i < 4 * a.segs; i += kPickT)
            if (q_max[i] == top) atomicMin(&s_i, i / 4);
        if (t == 0) s_j = kSampleSeg;
        __syncthreads();
        float v[4];
        sample_ld4<BF16>(x, (int64_t)s_i * kSampleSeg + 4 * t, V, v);
#pragma unroll
        for (int i = 3; i >= 0; --i)
            if (v[i] == top) atomicMin(&s_j, 4 * t + i);
        __syncthreads();
        if (t == 0) {
            *token = s_i * kSampleSeg + s_j;
            if (prob) *prob = 1.0f;
        }
        return;
    }
    const SampleRow& R = a.rows[row];
    /* top-k's border is in bins [kb_lo, C.kb] */
    SampleCut C = {kSampleBins, kSampleBins, kSampleBins, 0, 0, 0, 0, 0};
    int kb_lo = kSampleBins;
    unsigned int n = 0;                            /* listed tokens */
    if (set.plain) {
        for (int i = t; i < a.segs; i += kPickT) {
            double w = 0.0;
#pragma unroll
            for (int j = 4 * i; j < 4 * i + 4; ++j)
                if (sample_in(q_max[j])) w += a.q_sum[row * 4 * a.segs + j] * sample_w(set, q_max[j]);
            segm[i] = sample_mass_sum(w, a.shift);
        }
    } else if (set.listed) {
        /* top-k: k chunks have their largest logit in bins 0 .. last, so no token under the least of those
         * is among the k.  min-p: none under max + T log(min_p) has w >= min_p (the logarithm a millionth
         * and 1e-14 less, for its rounding and those of exp, which makes a 1 of everything above -2^-54). */
        int last = kSampleBins;
        float least = -3.4028235e38f;              /* and no token under this one can be kept */
        for (int i = t; i < a.segs; i += kPickT) segm[i] = 0;
        for (int i = t; i < kSampleBins; i += kPickT) hcount[i] = 0;
        if (t == 0) {
            s_i = kSampleBins;                     /* fewer than k chunks */
            s_j = 0;                               /* chunks */
            s_n = 0;                               /* tokens */
            s_key = 0xFFFFFFFFu;
        }
        __syncthreads();
        if (set.use_k) {
            for (int i0 = 0; i0 < chunks; i0 += 4 * kPickT) {
                if (i0) load_chunks(i0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (sample_in(cv[j])) atomicAdd(&hcount[sample_bin(set, cv[j])], 1u);
            }
            if (chunks > 4 * kPickT) load_chunks(0);
            __syncthreads();
            const unsigned int c0 = hcount[2 * t], c1 = hcount[2 * t + 1];
            u64 all;
            const u64 c = sample_block_scan<kPickT>((u64)(c0 + c1), su, &all);
            if (c < (u64)set.k && c + c0 + c1 >= (u64)set.k) s_i = c + c0 >= (u64)set.k ? 2 * t : 2 * t + 1;
            hcount[2 * t] = hcount[2 * t + 1] = 0;
            hmass[2 * t] = hmass[2 * t + 1] = 0;
            __syncthreads();
            last = s_i;
        } else {
            const double l = (double)top + (log(set.min_p) * 1.000001 - 1e-14) / set.inv_t;
            least = l > -3.4028234e38 ? (float)l : least;
        }
        /* the chunks, then their tokens, 16 lanes a chunk */
        unsigned int* const which = reinterpret_cast<unsigned int*>(smem + kPickWhich);
        uint32_t low = 0xFFFFFFFFu;                /* as a key */
        for (int i0 = 0; i0 < chunks; i0 += 4 * kPickT) {
            unsigned int in = 0;
            if (i0) load_chunks(i0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (cv[j] >= least && sample_bin(set, cv[j]) <= last) {
                    in |= 1u << j;
                    low = min(low, sample_key(cv[j]));
                }
            unsigned int at = sample_slots<3>(__builtin_popcount(in), reinterpret_cast<unsigned int*>(&s_j));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (in >> j & 1) {
                    if (at < kSampleList) which[at] = (unsigned int)(i0 + t + kPickT * j);
                    ++at;
                }
        }
        if (last < kSampleBins) {
            low = ~r3d_wave_max(~low);
            if ((t & 63) == 0) atomicMin(&s_key, low);
        }
        __syncthreads();
        if (last < kSampleBins) least = sample_value(s_key);
        const int nc = s_j;
        if (nc <= kSampleList) {
            constexpr int U = 8;                   /* loads in flight a lane: 32 tokens, a bit each */
            for (int c0 = t / 16; c0 - t / 16 < nc; c0 += kPickT / 16 * U) {
                float v[U][4];
                unsigned int in = 0;
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int c = c0 + kPickT / 16 * j;
                    if (c < nc) {
                        sample_ld4<BF16>(x, (int64_t)which[c] * kSampleChunk + 4 * (t & 15), V, v[j]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[j][i] = -__builtin_inff();
                    }
                }
#pragma unroll
                for (int j = 0; j < U; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) in = 2 * in + (v[j][i] >= least);       /* the first token in bit 31 */
                unsigned int at = sample_slots<6>(__builtin_popcount(in), &s_n);
                while (in) {
                    const int k = __builtin_clz(in);
                    in &= ~(0x80000000u >> k);
                    if (at < kSampleList)
                        list[at] = which[c0 + kPickT / 16 * (k >> 2)] * kSampleChunk + 4 * (t & 15) + (k & 3);
                    ++at;
                }
            }
            __syncthreads();
            n = s_n;
            /* (entries only now, a lane each: made where a token is found they would take as many steps of a
             * wave as it has tokens in flight) */
            if (n <= kSampleList)
                for (int i = t; i < (int)n; i += kPickT) {
                    const int64_t at = (int64_t)list[i];
                    list[i] = sample_entry_of(sample_ld1<BF16>(x, at), at);
                }
            __syncthreads();
        } else {
            n = kSampleList + 1;
        }
        /* few tokens are all sorted (50: 1.3 us for the bins' 4.3; 205: 3.8 and twice the exps); of more, or
         * with min-p alone, only those that lie at a cut */
        if (n <= kSampleList && !(set.use_k && n <= 128)) {
            /* the same cuts as from a whole row's bins, of the listed: what lies above the border bins
             * is kept, the list is left with what lies in them */
            if (set.use_k) {
                for (int i = t; i < (int)n; i += kPickT) {
                    const float v = sample_value(~(uint32_t)(list[i] >> 32));
                    const int b = sample_bin(set, v);
                    atomicAdd(&hcount[b], 1u);
                    if (set.use_p) atomicAdd(&hmass[b], sample_mass(sample_w(set, v), a.shift));
                }
                __syncthreads();
                sample_cut<kPickT>(set, hcount, hmass, su, &s_cut);
                C = s_cut;
            }
            if (t == 0) s_n = 0;
            const int whole = sample_whole(C);
            for (int i0 = 0; i0 < (int)n; i0 += kPickT) {
                const int i = i0 + t;
                bool in = false;
                u64 e = 0;
                if (i < (int)n) {
                    e = list[i];
                    const float v = sample_value(~(uint32_t)(e >> 32));
                    const int b = sample_bin(set, v);
                    if (b < whole) {
                        const double w = sample_w(set, v);
                        if (w >= set.min_p) atomicAdd(&segm[(int)(uint32_t)e / kSampleSeg], sample_mass(w, a.shift));
                    } else {
                        in = sample_border(C, b);
                    }
                }
                __syncthreads();                   /* the list is read up to here, and written up to here at most */
                const unsigned int at = sample_slots<1>(in, &s_n);
                if (in) list[at] = e;
            }
            __syncthreads();
            n = s_n;
            kb_lo = C.kb;
        } else {
            kb_lo = 0;
            if (set.use_k) C.kb = kSampleBins - 1;
            if (set.use_p) {
                C.pb_lo = 0;
                C.pb_hi = kSampleBins - 1;
            }
        }
    } else {
        for (int i = t; i < a.segs; i += kPickT) segm[i] = a.seg_mass[row * a.segs + i];
        C = R.cut;
        kb_lo = C.kb;
        n = R.n_list;
        for (int i = t; i < (int)n && i < kSampleList; i += kPickT) list[i] = R.list[i];
    }
    const bool cut_k = C.kb < kSampleBins, cut_p = C.pb_lo < kSampleBins;
    /* the last kept token: its key, and its index among equal keys */
    uint32_t last_key = 0;
    int64_t last_idx = V;
    if (cut_k || cut_p || n > kSampleList) {
        if (n <= kSampleList) {
            int size = 2;
            while (size < (int)n) size *= 2;
            /* Rising.  Up to 256 tokens each counts those before it (a lane a token, the list read by all
             * lanes alike: 88 take 1.2 us less than bitonic steps do, 205 in all 3.8 us).  Past that
             * bitonic: up to a token a lane in registers, by way of LDS only to another wave; past that in
             * LDS, where a wave's 64 pairs at distance 64 or less are 128 tokens of its own and only wider
             * steps need the barrier (480 tokens 7.5 us by barriers alone, 5 so). */
            if (n <= 256) {
                __syncthreads();
                const u64 e = list[t & 255];
                int before = 0;
                if ((t & ~63) < (int)n) {
                    int i = 0;
                    for (; i + 8 <= (int)n; i += 8)
#pragma unroll
                        for (int j = 0; j < 8; ++j) before += list[i + j] < e;
                    for (; i < (int)n; ++i) before += list[i] < e;
                }
                __syncthreads();
                if (t < (int)n) list[before] = e;
            } else if (size <= kPickT) {
                __syncthreads();
                u64 e = t < (int)n ? list[t] : ~(u64)0;
                for (int k = 2; k <= size; k *= 2)
                    for (int j = k / 2; j > 0; j /= 2) {
                        u64 o;
                        if (j < 64) {
                            o = __shfl_xor(e, j, 64);
                        } else {
                            __syncthreads();
                            list[t] = e;
                            __syncthreads();
                            o = list[t ^ j];
                        }
                        const bool low = ((t & j) == 0) == ((t & k) == 0);
                        e = (o < e) == low ? o : e;
                    }
                __syncthreads();
                list[t] = e;
            } else {
                for (int i = (int)n + t; i < size; i += kPickT) list[i] = ~(u64)0;
                __syncthreads();
                for (int k = 2; k <= size; k *= 2)
                    for (int j = k / 2; j > 0; j /= 2) {
                        for (int i = t; i < size / 2; i += kPickT) {
                            const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                            const u64 p = list[lo], q = list[hi];
                            if ((p > q) == ((lo & k) == 0)) {
                                list[lo] = q;
                                list[hi] = p;
                            }
                        }
                        if (j > 64 || (j == 1 && k > 64)) {
                            __syncthreads();
                        } else {
                            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                            __builtin_amdgcn_wave_barrier();
                        }
                    }
            }
            __syncthreads();
            /* a lane has `each` tokens in a row of the sorted list */
            const int each = (size + kPickT - 1) / kPickT, e0 = t * each;
            int in_p = 0;                                         /* listed tokens of top-p's bins */
            u64 wk = 0, wp = 0;
            auto value = [&](int i) { return sample_value(~(uint32_t)(list[i] >> 32)); };
            const double w0 = e0 < (int)n ? sample_w(set, value(e0)) : 0.0;
            auto weight = [&](int i) { return i == e0 ? w0 : sample_w(set, value(i)); };
            /* tokens of bin C.kb among the k; their positions start behind top-p's own bins */
            const int need = cut_k ? set.k - C.count_k : 0;
            int before_kb = 0;
            for (int i = e0; i < e0 + each && i < (int)n; ++i) {
                const int b = sample_bin(set, value(i));
                if (cut_p && b <= C.pb_hi) ++in_p;
                if (cut_k && b < kb_lo) ++before_kb;
            }
            u64 tmp;
            sample_block_scan<kPickT>((u64)in_p << 32 | (u64)before_kb, su, &tmp);
            in_p = (int)(tmp >> 32);
            before_kb = (int)(tmp & 0xFFFFFFFFu);
            const int end_k = cut_k && before_kb + need < (int)n ? before_kb + need : (int)n;
            int end = end_k;
            if (cut_p) {
                for (int i = e0; i < e0 + each && i < (int)n; ++i) {
                    const u64 w = sample_mass(weight(i), a.shift);
                    if (cut_k && i >= before_kb && i < end_k) wk += w;
                    if (i < in_p) wp += w;
                }
                u64 mass_k, all_p;
                mass_k = sample_block_sum<kPickT>(wk, su);
                u64 run = sample_block_scan<kPickT>(wp, su, &all_p);
                /* the mass that p is a share of: top-k's, or all */
                const u64 of = cut_k ? C.mass_k + mass_k : C.total;
                const u64 want = sample_share(set.p, of);
                if (t == 0) s_i = in_p < end_k ? in_p : end_k;
                __syncthreads();
                run += C.mass_p;
                for (int i = e0; i < e0 + each && i < in_p; ++i) {
                    if (run >= want) {                            /* enough before this one */
                        atomicMin(&s_i, i);
                        break;
                    }
                    run += sample_mass(weight(i), a.shift);
                }
                __syncthreads();
                end = s_i;
            }
            for (int i = e0; i < e0 + each && i < end; ++i) {
                const double w = weight(i);
                if (w >= set.min_p) atomicAdd(&segm[(int)(uint32_t)list[i] / kSampleSeg], sample_mass(w, a.shift));
            }
            last_key = ~(uint32_t)(list[end - 1] >> 32);
            last_idx = (int64_t)(uint32_t)list[end - 1];
        } else {
            /* Radix selection over the row.  select(lo, hi, by mass, goal): among the tokens of bins
             * [lo, hi], in order, the one that brings the count (or mass) to the goal: its key to
             * *key, what lies above it to *above, how many share it to *same. */
            auto select = [&](int lo, int hi, bool by_mass, u64 goal, uint32_t* key, u64* above, u64* over,
                              unsigned int* same) {
                uint32_t pre = 0;
                u64 done = 0, done_m = 0;
                for (int sh = 24; sh >= 0; sh -= 8) {
                    for (int i = t; i < 256; i += kPickT) {
                        hmass[i] = 0;
                        hcount[i] = 0;
                    }
                    __syncthreads();
                    for (int64_t i = 4 * t; i < V; i += 4 * kPickT) {
                        float v[4];
                        sample_ld4<BF16>(x, i, V, v);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (!sample_in(v[j])) continue;
                            const int b = sample_bin(set, v[j]);
                            const uint32_t kk = sample_key(v[j]);
                            if (b < lo || b > hi || (sh < 24 && (kk ^ pre) >> (sh + 8))) continue;
                            atomicAdd(&hcount[kk >> sh & 255], 1u);
                            atomicAdd(&hmass[kk >> sh & 255], sample_mass(sample_w(set, v[j]), a.shift));
                        }
                    }
                    __syncthreads();
                    if (t == 0) {
                        u64 c = done, m = done_m;
                        int d = 255;
                        for (; d > 0; --d) {
                            if ((by_mass ? m + hmass[d] : c + hcount[d]) >= goal) break;
                            c += hcount[d];
                            m += hmass[d];
                        }
                        s_i = d;
                        s_a = c;
                        s_b = m;
                    }
                    __syncthreads();
                    pre |= (uint32_t)s_i << sh;
                    done = s_a;
                    done_m = s_b;
                    *same = hcount[s_i];
                    __syncthreads();
                }
                *key = pre;
                *above = done;
                *over = done_m;
            };
            /* the index of the r-th token (from 1) of a key */
            auto nth = [&](uint32_t key, u64 r) -> int64_t {
                uint32_t pre = 0;
                u64 done = 0;
                for (int sh = 16; sh >= 0; sh -= 8) {
                    for (int i = t; i < 256; i += kPickT) hcount[i] = 0;
                    __syncthreads();
                    for (int64_t i = 4 * t; i < V; i += 4 * kPickT) {
                        float v[4];
                        sample_ld4<BF16>(x, i, V, v);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (sample_in(v[j]) && sample_key(v[j]) == key &&
                                (sh == 16 || ((uint32_t)(i + j) ^ pre) >> (sh + 8) == 0))
                                atomicAdd(&hcount[(uint32_t)(i + j) >> sh & 255], 1u);
                    }
                    __syncthreads();
                    if (t == 0) {
                        u64 c = done;
                        int d = 0;
                        for (; d < 255; ++d) {
                            if (c + hcount[d] >= r) break;
                            c += hcount[d];
                        }
                        s_i = d;
                        s_a = c;
                    }
                    __syncthreads();
                    pre |= (uint32_t)s_i << sh;
                    done = s_a;
                    __syncthreads();
                }
                return pre;
            };
            u64 above, over, keep = 0, of = 0;
            unsigned int same;
            uint32_t key_k = 0;
            u64 keep_k = 0;
            if (cut_k) {
                select(kb_lo, C.kb, false, (u64)(set.k - C.count_k), &key_k, &above, &over, &same);
                keep_k = (u64)(set.k - C.count_k) - above;
                if (keep_k > same) keep_k = same;  /* fewer than k tokens */
                last_key = key_k;
                keep = keep_k;
                of = C.mass_k + over + keep * sample_mass(sample_w(set, sample_value(key_k)), a.shift);
            }
            if (cut_p) {
                if (!cut_k) of = C.total;
                const u64 want = sample_share(set.p, of) - C.mass_p;
                select(C.pb_lo, C.pb_hi, true, want, &last_key, &above, &over, &same);
                const u64 w = sample_mass(sample_w(set, sample_value(last_key)), a.shift);
                keep = w ? (want - over + w - 1) / w : same;
                if (keep > same) keep = same;
                if (cut_k && last_key == key_k && keep > keep_k) keep = keep_k;
            }
            if (cut_k || cut_p) last_idx = nth(last_key, keep);
            const int whole = cut_p && C.pb_lo < kb_lo ? C.pb_lo : kb_lo;
            __syncthreads();
            for (int64_t i = 4 * t; i < V; i += 4 * kPickT) {
                float v[4];
                sample_ld4<BF16>(x, i, V, v);
                u64 sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!sample_in(v[j]) || sample_bin(set, v[j]) < whole) continue;
                    const uint32_t kk = sample_key(v[j]);
                    if (kk < last_key || (kk == last_key && i + j > last_idx)) continue;
                    const double w = sample_w(set, v[j]);
                    if (w >= set.min_p) sum += sample_mass(w, a.shift);
                }
                if (sum) atomicAdd(&segm[i / kSampleSeg], sum);
            }
        }
    }
    __syncthreads();
    /* u's share of the kept mass, the segment that holds it, the token */
    u64 total;
    const u64 mine = t < a.segs ? segm[t] : 0;
    const u64 before = sample_block_scan<kPickT>(mine, su, &total);
    const double goal = __builtin_floor((u > 0.0f ? (double)u : 0.0) * (double)total);
    const u64 at = goal < (double)total ? (u64)goal : total - 1;
    const u64 r = at < total ? at : total - 1;
    if (before <= r && r < before + mine) {
        s_i = t;
        s_a = r - before;
    }
    __syncthreads();
    /* Within the segment in f64: its kept tokens in order until their sum passes what is left of u's
     * share, or the last one should a rounding leave none.  With u at 0 or next to it masses under half
     * of 2^-s decide: from the first segment on, up to the first token that has a mass at the latest. */
    const double unit = __longlong_as_double((long long)(1023 - a.shift) << 52);
    const double whole_mass = (double)total * unit;
    const bool first = r == 0;
    const double rest = first ? (u > 0.0f ? (double)u : 0.0) * whole_mass : (double)s_a * unit;
    double done = 0.0;
    for (int seg = first ? 0 : s_i;; ++seg) {
        const int64_t i0 = (int64_t)seg * kSampleSeg + 4 * t;
        float v[4];
        double w[4] = {0.0, 0.0, 0.0, 0.0}, sum = 0.0;
        int any = -1;
        sample_ld4<BF16>(x, i0, V, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t kk = sample_key(v[i]);
            if (!sample_in(v[i]) || kk < last_key || (kk == last_key && i0 + i > last_idx)) continue;
            w[i] = sample_w(set, v[i]);
            if (!(w[i] >= set.min_p)) w[i] = 0.0;
            if (w[i] > 0.0) any = 4 * t + i;
            sum += w[i];
        }
        __syncthreads();                           /* s_i and s_a are read, and the last segment's */
        if (t == 0) {
            s_i = kSampleSeg;
            s_j = -1;
        }
        double all;
        double run = done + sample_block_scan<kPickT>(sum, reinterpret_cast<double*>(su), &all);
        done += all;
        int over = -1;                             /* the first past u's share: lanes are in index order */
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            run += w[i];
            if (over < 0 && w[i] > 0.0 && run > rest) over = 4 * t + i;
        }
        const u64 m_over = __ballot(over >= 0), m_any = __ballot(any >= 0);
        if (m_over && (t & 63) == __builtin_ctzll(m_over)) atomicMin(&s_i, over);
        if (m_any && (t & 63) == 63 - __builtin_clzll(m_any)) atomicMax(&s_j, any);
        __syncthreads();
        if (first && s_i == kSampleSeg && seg + 1 < a.segs) continue;
        const int pick = s_i < kSampleSeg ? s_i : s_j;
        if (pick >= 0 && t == pick >> 2) {
            *token = seg * kSampleSeg + pick;
            const double wp = (pick & 3) == 0 ? w[0] : (pick & 3) == 1 ? w[1] : (pick & 3) == 2 ? w[2] : w[3];
            if (prob) *prob = (float)(wp / whole_mass);
        }
        return;
    }
}

static int sample_entry(const RadArgs* ra, RadStream s) {
    if (env_no_sample()) return RAD_E_UNSUPPORTED;
    SampleArgs a{};
    const int rc = plan_sample(ra, &a.P);
    if (rc) return rc;
    const int64_t M = a.P.M, V = a.P.V;
    if (!ra->scratch || ((uintptr_t)ra->scratch & 15) || ra->scratch_bytes < sample_scratch_bytes(M, V))
        return RAD_E_UNSUPPORTED;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    a.segs = (int)((V + kSampleSeg - 1) / kSampleSeg);
    a.rows = (SampleRow*)ra->scratch;
    a.seg_mass = (u64*)(a.rows + M);
    a.q_sum = (double*)(a.seg_mass + M * a.segs);
    a.q_max = (float*)(a.q_sum + 4 * M * a.segs);
    a.q_min = a.q_max + 4 * M * a.segs;
    a.chunk_max = a.q_min + 4 * M * a.segs;
    int bits = 0;                                  /* V <= 2^bits: V 2^(62 - bits) <= 2^62 */
    while (((int64_t)1 << bits) < V) ++bits;
    a.shift = 62 - bits < 51 ? 62 - bits : 51;
    /* a workgroup a segment while that makes 16384 at most (128 rows of 64: 29 us; four a workgroup, which
     * leaves a last round of few workgroups, 36) */
    a.per = (int)((a.segs * M + 16383) / 16384);
    if (a.per > a.segs) a.per = a.segs;
    const dim3 grid((unsigned)((a.segs + a.per - 1) / a.per), (unsigned)M);
    const int64_t shares = (int64_t)((a.segs + kBinLeast - 1) / kBinLeast) * M;
    const dim3 bgrid((unsigned)(shares < kBinGrid ? shares : M > kBinGrid ? M : kBinGrid));
    const size_t lds = kPickWords * 8;
    hipStream_t stream = (hipStream_t)s;
#define R3D_SAMPLE(B_)                                                                          \
    hipLaunchKernelGGL((sample_range_kernel<B_>), grid, dim3(kSampleT), 0, stream, a);            \
    if (a.P.top_k || a.P.top_p) {                                                                \
        hipLaunchKernelGGL((sample_hist_kernel<B_>), bgrid, dim3(kBinT), 0, stream, a);           \
        hipLaunchKernelGGL((sample_gather_kernel<B_>), bgrid, dim3(kBinT), 0, stream, a);         \
    }                                                                                            \
    hipLaunchKernelGGL((sample_pick_kernel<B_>), dim3((unsigned)M), dim3(kPickT), lds, stream, a)
    if (a.P.bf16) { R3D_SAMPLE(true); } else { R3D_SAMPLE(false); }
#undef R3D_SAMPLE
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        fprintf(stderr, "libr3d_gfx950: sample_logits launch FAILED (%s)\n", hipGetErrorName(e));
        return RAD_E_DEVICE;
    }
    return RAD_OK;
}

}  // namespace r3d

extern "C" {

int r3d_rad_sample_logits(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("sample_logits", a, s, r3d::sample_entry);
}
int64_t r3d_rad_sample_logits_scratch(const RadArgs* a) { return r3d::sample_hook_bytes(a); }

}  /* extern "C" */
