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
 * Masses are 64-bit integers, w * 2^s to nearest with V 2^s < 2^63 (s = 44 at V = 262144), from an
 * exp in f64: integer sums do not depend on their order, so atomics may make them, a cut and the
 * search see the same numbers, and a run repeats bit for bit.  A border moves by about
 * 2^-s sqrt(V) / mass, 2^-35 at V = 262144, where f32 sums would move it by 2^-20 and pick a
 * neighbour now and then.
 *
 * Three passes over the logits and one over a segment, four launches:
 *   1 largest and least logit of every segment (4096 tokens); the row's scratch is cleared
 *   2 rows with top-k or top-p: count and mass in 2048 bins, of equal width in x over the row's range
 *     (at most 32 T: below that w is 0); bins are in the order of x, so a cut falls into one bin
 *   3 the border bins are found from the 2048 sums; the tokens above them are added up a segment at a
 *     time, the tokens in them are listed
 *   4 a workgroup a row: the listed tokens are sorted, the cuts placed, the segment that holds
 *     u * mass found, and the token in it.  Past 8192 tokens in the border bins (many equal
 *     logits) the cuts are placed by radix selection over the row instead.
 * The row is read from L2 and the last-level cache after pass 1 where it fits. */
#include <hip/hip_runtime.h>

#include <stdio.h>

#include "r3d_device.h"
#include "r3d_dump.h"
#include "r3d_plan.h"
#include "r3d_sample.h"

namespace r3d {

bool chip_ok();                  /* r3d_gemm.hip */

typedef unsigned long long u64;

struct SampleArgs {
    SamplePlan P;
    SampleRow* rows;
    float* seg_max;              /* [M][segs] */
    float* seg_min;
    u64* seg_mass;
    int segs, per, shift;        /* per: segments a workgroup; shift: s of the masses */
};

/* A row's settings, and what its tokens are measured against. */
struct SampleSet {
    float top;                   /* the largest logit; -inf: the row is empty */
    float bin;                   /* bins a unit of x */
    double inv_t, p, min_p;
    int k;
    bool greedy, use_k, use_p;
};

__device__ __forceinline__ SampleSet sample_set(const SampleArgs& a, int64_t row, float top, float low) {
    const SamplePlan& P = a.P;
    SampleSet s;
    const float T = P.temperature ? P.temperature[row * P.t_stride] : 1.0f;
    const int k = P.top_k ? P.top_k[row * P.k_stride] : 0;
    const float p = P.top_p ? P.top_p[row * P.p_stride] : 1.0f;
    const float m = P.min_p ? P.min_p[row * P.m_stride] : 0.0f;
    s.top = top;
    s.greedy = !(T > 0.0f);
    s.inv_t = 1.0 / (double)T;
    s.k = k;
    s.use_k = k > 0 && k < P.V;
    s.p = (double)p;
    s.use_p = p < 1.0f;
    s.min_p = m > 0.0f ? (m < 1.0f ? (double)m : 1.0) : 0.0;
    s.bin = (float)(kSampleBins - 1) / __builtin_fminf(top - low, 32.0f * T);
    return s;
}

/* exp(z) for z <= 0, within 2^-50: z = n ln 2 + r, |r| <= ln 2 / 2, the series of exp(r) to r^12
 * (r^13 / 13! < 2^-52), times 2^n.  Past the least f64 (and for NaN) 0. */
__device__ __forceinline__ double sample_exp(double z) {
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
    if (!(z > -746.0)) return 0.0;
    return __builtin_amdgcn_ldexp(e, (int)n);
}

__device__ __forceinline__ bool sample_in(float x) { return x > -__builtin_inff(); }   /* NaN: no */

__device__ __forceinline__ double sample_w(const SampleSet& s, float x) {
    return x == s.top ? 1.0 : sample_exp(((double)x - (double)s.top) * s.inv_t);
}
__device__ __forceinline__ u64 sample_mass(double w, int shift) {
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
            if (i + j < V)
                v[j] = BF16 ? r3d_bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i + j])
                            : reinterpret_cast<const float*>(x)[i + j];
        }
    }
}

constexpr int kSampleT = 256;                      /* lanes of passes 1 to 3 */
constexpr int kSampleU = kSampleSeg / kSampleT / 4; /* loads a lane and segment */

/* Segments [g per, min(segs, (g + 1) per)) of row blockIdx.y: f(segment, index, four logits). */
template <bool BF16, typename F>
__device__ __forceinline__ void sample_walk(const SampleArgs& a, F f) {
    const uint8_t* x = sample_row(a.P, blockIdx.y);
    const int s1 = ((int)blockIdx.x + 1) * a.per < a.segs ? ((int)blockIdx.x + 1) * a.per : a.segs;
    for (int s = blockIdx.x * a.per; s < s1; ++s) {
        float v[kSampleU][4];
#pragma unroll
        for (int j = 0; j < kSampleU; ++j)
            sample_ld4<BF16>(x, (int64_t)s * kSampleSeg + 4 * (threadIdx.x + kSampleT * j), a.P.V, v[j]);
        f(s, (int64_t)s * kSampleSeg + 4 * threadIdx.x, v);
    }
}

template <int T>
__device__ __forceinline__ float sample_block_max(float v, float* s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v = __builtin_fmaxf(v, s[i]);
    return v;
}
template <int T>
__device__ __forceinline__ u64 sample_block_sum(u64 v, u64* s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += s[i];
    return v;
}
/* The sum over the lanes before this one; *total over all. */
template <int T>
__device__ __forceinline__ u64 sample_block_scan(u64 v, u64* s, u64* total) {
    u64 in = v;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 o = __shfl_up(in, off, 64);
        if (lane >= off) in += o;
    }
    __syncthreads();
    if (lane == 63) s[wave] = in;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) {
        if (i < wave) before += s[i];
        all += s[i];
    }
    *total = all;
    return before + in - v;
}

/* The row's largest and least logit from its segments'. */
template <int T>
__device__ __forceinline__ void sample_range(const SampleArgs& a, int64_t row, float* s, float* top, float* low) {
    float hi = -__builtin_inff(), lo = __builtin_inff();
    for (int i = threadIdx.x; i < a.segs; i += T) {
        hi = __builtin_fmaxf(hi, a.seg_max[row * a.segs + i]);
        lo = __builtin_fminf(lo, a.seg_min[row * a.segs + i]);
    }
    *top = sample_block_max<T>(hi, s);
    *low = -sample_block_max<T>(-lo, s);
}

template <bool BF16>
__global__ __launch_bounds__(kSampleT) void sample_range_kernel(SampleArgs a) {
    __shared__ float s[kSampleT / 64];
    const int64_t row = blockIdx.y;
    SampleRow& R = a.rows[row];
    for (int i = blockIdx.x * kSampleT + threadIdx.x; i < kSampleBins; i += gridDim.x * kSampleT) {
        R.mass[i] = 0;
        R.count[i] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) R.n_list = 0;
    sample_walk<BF16>(a, [&](int seg, int64_t, float (*v)[4]) {
        float hi = -__builtin_inff(), lo = __builtin_inff();
#pragma unroll
        for (int j = 0; j < kSampleU; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sample_in(v[j][i])) {
                    hi = __builtin_fmaxf(hi, v[j][i]);
                    lo = __builtin_fminf(lo, v[j][i]);
                }
        hi = sample_block_max<kSampleT>(hi, s);
        lo = -sample_block_max<kSampleT>(-lo, s);
        if (threadIdx.x == 0) {
            a.seg_max[row * a.segs + seg] = hi;
            a.seg_min[row * a.segs + seg] = lo;
        }
    });
}

template <bool BF16>
__global__ __launch_bounds__(kSampleT) void sample_hist_kernel(SampleArgs a) {
    __shared__ u64 mass[kSampleBins];
    __shared__ unsigned int count[kSampleBins];
    __shared__ float s[kSampleT / 64];
    const int64_t row = blockIdx.y;
    float top, low;
    sample_range<kSampleT>(a, row, s, &top, &low);
    const SampleSet set = sample_set(a, row, top, low);
    if (set.greedy || !sample_in(top) || !(set.use_k || set.use_p)) return;      /* the whole workgroup */
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleT) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    sample_walk<BF16>(a, [&](int, int64_t, float (*v)[4]) {
#pragma unroll
        for (int j = 0; j < kSampleU; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sample_in(v[j][i])) {
                    const int b = sample_bin(set, v[j][i]);
                    atomicAdd(&count[b], 1u);
                    if (set.use_p) atomicAdd(&mass[b], sample_mass(sample_w(set, v[j][i]), a.shift));
                }
    });
    __syncthreads();
    SampleRow& R = a.rows[row];
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleT)
        if (count[i]) {
            atomicAdd(&R.count[i], count[i]);
            if (mass[i]) atomicAdd(&R.mass[i], mass[i]);
        }
}

/* p's share of a mass, one at least. */
__device__ __forceinline__ u64 sample_share(double p, u64 mass) {
    const double t = __builtin_ceil(p * (double)mass);
    return t >= 1.0 ? (u64)t : 1;
}

template <bool BF16>
__global__ __launch_bounds__(kSampleT) void sample_gather_kernel(SampleArgs a) {
    constexpr int B = kSampleBins / kSampleT;      /* bins a lane */
    __shared__ u64 su[kSampleT / 64];
    __shared__ float s[kSampleT / 64];
    __shared__ int kb, pb[2];
    __shared__ u64 edge[2];                        /* mass above kb, above pb_lo */
    __shared__ int count_k;
    __shared__ u64 mass_kb;
    const int64_t row = blockIdx.y;
    float top, low;
    sample_range<kSampleT>(a, row, s, &top, &low);
    const SampleSet set = sample_set(a, row, top, low);
    if (set.greedy || !sample_in(top)) return;
    SampleRow& R = a.rows[row];
    if (threadIdx.x == 0) {
        kb = pb[0] = pb[1] = kSampleBins;
        edge[0] = edge[1] = mass_kb = 0;
        count_k = 0;
    }
    if (set.use_k || set.use_p) {
        u64 c[B], m[B], cs = 0, ms = 0, all, total;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            c[i] = R.count[B * threadIdx.x + i];
            m[i] = R.mass[B * threadIdx.x + i];
            cs += c[i];
            ms += m[i];
        }
        u64 c0 = sample_block_scan<kSampleT>(cs, su, &all);
        const u64 m0 = sample_block_scan<kSampleT>(ms, su, &total);
        u64 mm = m0;
        if (set.use_k && (u64)set.k < all) {
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (c0 < (u64)set.k && c0 + c[i] >= (u64)set.k) {
                    kb = B * threadIdx.x + i;
                    edge[0] = mm;
                    mass_kb = m[i];
                    count_k = (int)c0;
                }
                c0 += c[i];
                mm += m[i];
            }
        }
        __syncthreads();
        if (set.use_p) {
            /* the kept tokens' mass is known to within bin kb: the border of top-p to within these */
            const u64 lo = sample_share(set.p, kb < kSampleBins ? edge[0] : total);
            const u64 hi = sample_share(set.p, kb < kSampleBins ? edge[0] + mass_kb : total);
            mm = m0;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (mm < lo && mm + m[i] >= lo) {
                    pb[0] = B * threadIdx.x + i;
                    edge[1] = mm;
                }
                if (mm < hi && mm + m[i] >= hi) pb[1] = B * threadIdx.x + i;
                mm += m[i];
            }
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        R.kb = kb;
        R.pb_lo = pb[0];
        R.pb_hi = pb[1];
        R.mass_k = edge[0];
        R.mass_p = edge[1];
        R.count_k = count_k;
    }
    __syncthreads();
    const int lk = kb, p0 = pb[0], p1 = pb[1], whole = lk < p0 ? lk : p0;   /* bins below `whole`: kept */
    sample_walk<BF16>(a, [&](int seg, int64_t i0, float (*v)[4]) {
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < kSampleU; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[j][i];
                if (!sample_in(x)) continue;
                const int b = sample_bin(set, x);
                if (b < whole) {
                    const double w = sample_w(set, x);
                    if (w >= set.min_p) sum += sample_mass(w, a.shift);
                } else if (b == lk || (b >= p0 && b <= p1)) {
                    const unsigned int at = atomicAdd(&R.n_list, 1u);
                    if (at < kSampleList)
                        R.list[at] = (u64)~sample_key(x) << 32 | (u64)(i0 + 4 * kSampleT * j + i);
                }
            }
        sum = sample_block_sum<kSampleT>(sum, su);
        if (threadIdx.x == 0) a.seg_mass[row * a.segs + seg] = sum;
    });
}

constexpr int kPickT = 1024;

/* Pass 4.  LDS: the list [8192], the segments' masses [1024], 256 counters and masses. */
template <bool BF16>
__global__ __launch_bounds__(kPickT) void sample_pick_kernel(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) u64 smem[];
    u64* const list = smem;
    u64* const segm = smem + kSampleList;
    u64* const hmass = segm + kSampleMaxSegs;                     /* [256] */
    unsigned int* const hcount = reinterpret_cast<unsigned int*>(hmass + 256);   /* [256] */
    __shared__ u64 su[kPickT / 64];
    __shared__ float sf[kPickT / 64];
    __shared__ u64 s_a, s_b;
    __shared__ int s_i, s_j;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x, V = a.P.V;
    const uint8_t* x = sample_row(a.P, row);
    int* const token = a.P.token + row * a.P.token_stride;
    float* const prob = a.P.prob ? a.P.prob + row * a.P.prob_stride : nullptr;
    float top, low;
    sample_range<kPickT>(a, row, sf, &top, &low);
    const SampleSet set = sample_set(a, row, top, low);
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
        for (int i = t; i < a.segs; i += kPickT)
            if (a.seg_max[row * a.segs + i] == top) atomicMin(&s_i, i);
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
    for (int i = t; i < a.segs; i += kPickT) segm[i] = a.seg_mass[row * a.segs + i];
    const SampleRow& R = a.rows[row];
    const int kb = R.kb, pb_lo = R.pb_lo, pb_hi = R.pb_hi;
    const bool cut_k = kb < kSampleBins, cut_p = pb_lo < kSampleBins;
    /* the last kept token: its key, and its index among equal keys */
    uint32_t last_key = 0;
    int64_t last_idx = V;
    if (cut_k || cut_p) {
        const unsigned int n = R.n_list;
        if (n <= kSampleList) {
            int size = 2;
            while (size < (int)n) size *= 2;
            for (int i = t; i < size; i += kPickT) list[i] = i < (int)n ? R.list[i] : ~(u64)0;
            __syncthreads();
            for (int k = 2; k <= size; k *= 2)                    /* bitonic, rising */
                for (int j = k / 2; j > 0; j /= 2) {
                    for (int i = t; i < size / 2; i += kPickT) {
                        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                        const u64 p = list[lo], q = list[hi];
                        if ((p > q) == ((lo & k) == 0)) {
                            list[lo] = q;
                            list[hi] = p;
                        }
                    }
                    __syncthreads();
                }
            /* a lane has `each` tokens in a row of the sorted list */
            const int each = (size + kPickT - 1) / kPickT, e0 = t * each;
            int in_p = 0;                                         /* listed tokens of top-p's bins */
            u64 wk = 0, wp = 0;
            auto value = [&](int i) { return sample_value(~(uint32_t)(list[i] >> 32)); };
            /* tokens of bin kb among the k; their positions start behind top-p's own bins */
            const int need = cut_k ? set.k - R.count_k : 0;
            int before_kb = 0;
            for (int i = e0; i < e0 + each && i < (int)n; ++i) {
                const int b = sample_bin(set, value(i));
                if (cut_p && b <= pb_hi) ++in_p;
                if (cut_k && b < kb) ++before_kb;
            }
            u64 tmp;
            sample_block_scan<kPickT>((u64)in_p << 32 | (u64)before_kb, su, &tmp);
            in_p = (int)(tmp >> 32);
            before_kb = (int)(tmp & 0xFFFFFFFFu);
            const int end_k = cut_k ? before_kb + need : (int)n;
            int end = end_k;
            if (cut_p) {
                for (int i = e0; i < e0 + each && i < (int)n; ++i) {
                    const u64 w = sample_mass(sample_w(set, value(i)), a.shift);
                    if (cut_k && i >= before_kb && i < end_k) wk += w;
                    if (i < in_p) wp += w;
                }
                u64 mass_k, all_p;
                mass_k = sample_block_sum<kPickT>(wk, su);
                u64 run = sample_block_scan<kPickT>(wp, su, &all_p);
                /* the mass that p is a share of: top-k's, or all */
                u64 of = R.mass_k + mass_k;
                if (!cut_k) {
                    u64 m = 0;
                    for (int i = t; i < kSampleBins; i += kPickT) m += R.mass[i];
                    of = sample_block_sum<kPickT>(m, su);
                }
                const u64 want = sample_share(set.p, of);
                if (t == 0) s_i = in_p < end_k ? in_p : end_k;
                __syncthreads();
                run += R.mass_p;
                for (int i = e0; i < e0 + each && i < in_p; ++i) {
                    if (run >= want) {                            /* enough before this one */
                        atomicMin(&s_i, i);
                        break;
                    }
                    run += sample_mass(sample_w(set, value(i)), a.shift);
                }
                __syncthreads();
                end = s_i;
            }
            for (int i = e0; i < e0 + each && i < end; ++i) {
                const double w = sample_w(set, value(i));
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
                select(kb, kb, false, (u64)(set.k - R.count_k), &key_k, &above, &over, &same);
                keep_k = (u64)(set.k - R.count_k) - above;
                last_key = key_k;
                keep = keep_k;
                of = R.mass_k + over + keep * sample_mass(sample_w(set, sample_value(key_k)), a.shift);
            }
            if (cut_p) {
                if (!cut_k) {
                    u64 m = 0;
                    for (int i = t; i < kSampleBins; i += kPickT) m += R.mass[i];
                    of = sample_block_sum<kPickT>(m, su);
                }
                const u64 want = sample_share(set.p, of) - R.mass_p;
                select(pb_lo, pb_hi, true, want, &last_key, &above, &over, &same);
                const u64 w = sample_mass(sample_w(set, sample_value(last_key)), a.shift);
                keep = w ? (want - over + w - 1) / w : same;
                if (keep > same) keep = same;
                if (cut_k && last_key == key_k && keep > keep_k) keep = keep_k;
            }
            last_idx = nth(last_key, keep);
            const int whole = cut_p && pb_lo < kb ? pb_lo : kb;
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
    const float u = a.P.u[row * a.P.u_stride];
    const double goal = __builtin_floor((u > 0.0f ? (double)u : 0.0) * (double)total);
    const u64 at = goal < (double)total ? (u64)goal : total - 1;
    const u64 r = at < total ? at : total - 1;
    if (before <= r && r < before + mine) {
        s_i = t;
        s_a = r - before;
    }
    __syncthreads();
    float v[4];
    const double whole_mass = (double)total * __longlong_as_double((long long)(1023 - a.shift) << 52);
    if (r == 0) {
        /* u at 0 or next to it, where masses under half of 2^-s decide: the running sum in f64, from
         * the first token on (up to the first one that has a mass, at the latest) */
        const double want = (u > 0.0f ? (double)u : 0.0) * whole_mass;
        double done = 0.0;
        for (int seg = 0; seg < a.segs; ++seg) {
            const int64_t i1 = (int64_t)seg * kSampleSeg + 4 * t;
            double wv[4], mine_d = 0.0;
            sample_ld4<BF16>(x, i1, V, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t kk = sample_key(v[i]);
                wv[i] = 0.0;
                if (sample_in(v[i]) && (kk > last_key || (kk == last_key && i1 + i <= last_idx))) {
                    wv[i] = sample_w(set, v[i]);
                    if (!(wv[i] >= set.min_p)) wv[i] = 0.0;
                }
                mine_d += wv[i];
            }
            double in = mine_d;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const double o = __shfl_up(in, off, 64);
                if ((t & 63) >= off) in += o;
            }
            __syncthreads();
            if ((t & 63) == 63) su[t >> 6] = (u64)__double_as_longlong(in);
            if (t == 0) s_j = kSampleSeg;
            __syncthreads();
            double run = done, seg_all = done;
            for (int i = 0; i < kPickT / 64; ++i) {
                if (i < t >> 6) run += __longlong_as_double((long long)su[i]);
                seg_all += __longlong_as_double((long long)su[i]);
            }
            run += in - mine_d;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                run += wv[i];
                if (wv[i] > 0.0 && run > want) {
                    atomicMin(&s_j, 4 * t + i);
                    break;
                }
            }
            __syncthreads();
            if (s_j < kSampleSeg) {
                const int at_t = s_j >> 2, at_i = s_j & 3;
                if (t == at_t) {
                    *token = seg * kSampleSeg + s_j;
                    if (prob) *prob = (float)((at_i == 0 ? wv[0] : at_i == 1 ? wv[1] : at_i == 2 ? wv[2] : wv[3]) / whole_mass);
                }
                return;
            }
            done = seg_all;
        }
        return;
    }
    const int64_t i0 = (int64_t)s_i * kSampleSeg + 4 * t;
    const u64 rest = s_a;
    u64 w[4], sum = 0, all;
    double wd[4] = {0.0, 0.0, 0.0, 0.0};
    sample_ld4<BF16>(x, i0, V, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = 0;
        if (!sample_in(v[i])) continue;
        const uint32_t kk = sample_key(v[i]);
        if (kk < last_key || (kk == last_key && i0 + i > last_idx)) continue;
        wd[i] = sample_w(set, v[i]);
        if (wd[i] >= set.min_p) w[i] = sample_mass(wd[i], a.shift);
        sum += w[i];
    }
    u64 run = sample_block_scan<kPickT>(sum, su, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (run <= rest && rest < run + w[i]) {
            *token = (int)(i0 + i);
            if (prob) *prob = (float)(wd[i] / whole_mass);
        }
        run += w[i];
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
    a.seg_max = (float*)(a.seg_mass + M * a.segs);
    a.seg_min = a.seg_max + M * a.segs;
    int bits = 0;                                  /* V <= 2^bits: V 2^(62 - bits) <= 2^62 */
    while (((int64_t)1 << bits) < V) ++bits;
    a.shift = 62 - bits;
    /* a workgroup a segment while that makes no more than 2048 of them */
    a.per = (int)((a.segs * M + 2047) / 2048);
    if (a.per > a.segs) a.per = a.segs;
    const dim3 grid((unsigned)((a.segs + a.per - 1) / a.per), (unsigned)M);
    const size_t lds = (kSampleList + kSampleMaxSegs + 256) * 8 + 256 * 4;
    hipStream_t stream = (hipStream_t)s;
#define R3D_SAMPLE(B_)                                                                        \
    hipLaunchKernelGGL((sample_range_kernel<B_>), grid, dim3(kSampleT), 0, stream, a);          \
    if (a.P.top_k || a.P.top_p)                                                                \
        hipLaunchKernelGGL((sample_hist_kernel<B_>), grid, dim3(kSampleT), 0, stream, a);       \
    hipLaunchKernelGGL((sample_gather_kernel<B_>), grid, dim3(kSampleT), 0, stream, a);         \
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
