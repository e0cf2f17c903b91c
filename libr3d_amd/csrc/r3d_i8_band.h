/* r3d_i8_band.h -- the activation producers of the int8 linear layer on gfx950: quant_act_i8,
 * gated_quant_i8 and rmsnorm_quant_i8.  Each writes int8 codes with one f32 scale a row of
 *
 *   quant    h = x
 *   gated    h = act(gate) * up,  act(g) = silu ? g * sigmoid(g) : sigmoid(g),   in f32
 *   rmsnorm  r = bf16(residual + x) (written back), or x;  rs = f32(1 / sqrt(sum r^2 / n + eps)),
 *            the sum in f64;  h = (r * rs) * (w + wadd), each product rounded to f32
 *
 *   amax = max |h|,  s = amax > 0 ? max(amax * (1/127), 2^-126) : 1   (stored)
 *   q    = rint(h * (1 / s)), to nearest even, within +-127
 *
 * h is quantised as it stands in f32 (the e4m3 producers beside these narrow it to bf16 first, as
 * the kernels that they follow do; here the narrowing would only move codes).  The 2^-126 keeps 1 / s
 * finite.  The maximum is taken over the magnitudes' bits, where an infinity is above every number and
 * a NaN above that: a row whose h has a NaN has scale NaN and one with an infinity scale inf, both with codes
 * 0, so the product over the row is NaN and not a number that hides them.  (h of a norm over an infinity is NaN,
 * inf * (1 / inf); so is that of silu at -inf, -inf * 0.)
 *
 * One workgroup a row, the row in registers (C chunks of 8 elements a lane) from the load to the
 * codes: every operand is read once and every result written once, which is all the traffic there
 * is; the kernels are bound by it (us of a kernel trace, and all bytes a second: norm with its residual
 * 2048 x 5376 19.5, 4.0 TB/s; gated 2048 x 21504 44.8, 4.9; quant 2048 x 4096 6.0, 4.2; four rows, where the
 * chain of one row counts, 4.2, 6.6 and 2.4; f32 in gated 78.7, quant 8.0; the norm alone 12.5; with the two reductions over a wave by way of LDS 20.0, 46.9
 * and 6.4; 4.6, 6.8 and 2.6;
 * a large copy reaches 5.1).  Operands move in 16-byte accesses at element alignment
 * (gfx950's global memory takes them anywhere), so no pitch or base needs a kernel of its own; the
 * last n % 8 elements go one by one.  A row past the registers (C = 0) is walked twice. */
#ifndef R3D_I8_BAND_H
#define R3D_I8_BAND_H

#include "r3d_device.h"
#include "r3d_i8.h"
#include "r3d_wave.h"

namespace r3d {

struct I8BandArgs {
    const uint8_t* x;
    const uint16_t* res;
    uint16_t* res_out;
    const uint8_t* w;
    uint8_t* q;
    float* scale;
    uint8_t* ob;
    int64_t n, x_pitch, r_pitch, ro_pitch, q_pitch, s_stride, ob_pitch;
    double eps;
    float wadd;
    int silu, ob_bf16;
};

/* Eight elements of a row as they lie in memory. */
template <bool BF16>
struct I8Raw {
    r3d_i32x4 v[BF16 ? 1 : 2];
    __device__ __forceinline__ float at(int j) const {
        if (BF16) return __uint_as_float(j & 1 ? (uint32_t)v[0][j >> 1] & 0xFFFF0000u : (uint32_t)v[0][j >> 1] << 16);
        return __int_as_float(v[BF16 ? 0 : j >> 2][j & 3]);
    }
};

/* The eight from element i of a row of n on; zeros past its end. */
template <bool BF16>
__device__ __forceinline__ I8Raw<BF16> i8_ld8(const uint8_t* row, int64_t i, int64_t n) {
    I8Raw<BF16> r;
    if (i + 8 <= n) {
        r.v[0] = *reinterpret_cast<const r3d_i32x4_u2*>(row + (BF16 ? 2 : 4) * i);
        if (!BF16) r.v[BF16 ? 0 : 1] = *reinterpret_cast<const r3d_i32x4_u2*>(row + 4 * i + 16);
    } else {
#pragma unroll
        for (int k = 0; k < (BF16 ? 1 : 2); ++k) r.v[k] = r3d_i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) {
                if (BF16)
                    r.v[0][j >> 1] |= (int)((uint32_t)reinterpret_cast<const uint16_t*>(row)[i + j] << (16 * (j & 1)));
                else
                    r.v[BF16 ? 0 : j >> 2][j & 3] = reinterpret_cast<const int*>(row)[i + j];
            }
    }
    return r;
}

/* Eight f32 as bf16 (or as they are) to element i of a row of n on. */
__device__ __forceinline__ void i8_st8(uint8_t* row, int64_t i, int64_t n, const float* v, int bf16) {
    if (bf16) {
        r3d_i32x4_u2 d;
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = (int)r3d_pack_bf16x2(v[2 * j], v[2 * j + 1]);
        if (i + 8 <= n) {
            *reinterpret_cast<r3d_i32x4_u2*>(row + 2 * i) = d;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < n)
                    reinterpret_cast<uint16_t*>(row)[i + j] = (uint16_t)((uint32_t)d[j >> 1] >> (16 * (j & 1)));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) reinterpret_cast<float*>(row)[i + j] = v[j];
    }
}

/* sigmoid(g) = 1 / (1 + exp(-g)) in f32, within 3 ulp where that is a normal number (g over -87.3; under that
 * it may be 0, off by less than 2^-126): exp2 of the product's high part (its
 * rounding error times ln 2 is a factor on top, which keeps large |g| exact) and a reciprocal with
 * one Newton step.  Past 100 exp is inf and the result 0, as 1 / (1 + inf). */
__device__ __forceinline__ float i8_sigmoid(float g) {
    const float x = __builtin_fminf(__builtin_fmaxf(-g, -100.0f), 100.0f);
    const float t = x * 1.44269504f;
    const float lo = __builtin_fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    const float d = 1.0f + __builtin_fmaf(e, lo * 0.693147181f, e);
    float r = __builtin_amdgcn_rcpf(d);
    r = d < 3.0e38f ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) : 0.0f;
    return g != g ? g : r;
}

/* bf16(residual + x), also to element i of the row at ro on. */
__device__ __forceinline__ I8Raw<true> i8_add8(const I8Raw<true>& x, const I8Raw<true>& a, uint8_t* ro, int64_t i,
                                               int64_t n) {
    I8Raw<true> r;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        r.v[0][j] = (int)r3d_pack_bf16x2(__fadd_rn(a.at(2 * j), x.at(2 * j)), __fadd_rn(a.at(2 * j + 1), x.at(2 * j + 1)));
    if (i + 8 <= n) {
        *reinterpret_cast<r3d_i32x4_u2*>(ro + 2 * i) = r.v[0];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n)
                reinterpret_cast<uint16_t*>(ro)[i + j] = (uint16_t)((uint32_t)r.v[0][j >> 1] >> (16 * (j & 1)));
    }
    return r;
}

/* act(gate) * up */
template <bool BF16>
__device__ __forceinline__ void i8_gated8(const I8Raw<BF16>& g, const I8Raw<BF16>& u, int silu, float* h) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float gv = g.at(j), s = i8_sigmoid(gv);
        h[j] = (silu ? gv * s : s) * u.at(j);
    }
}

/* The largest of a workgroup's values, or their sum, on every lane; `s` holds one a wave. */
__device__ __forceinline__ uint32_t i8_block_max(uint32_t v, uint32_t* s) {
    v = r3d_wave_max(v);
    const int nw = blockDim.x >> 6;
    if (nw == 1) return v;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t r = s[0];
    for (int i = 1; i < nw; ++i) r = r > s[i] ? r : s[i];
    return r;
}
__device__ __forceinline__ double i8_block_sum(double v, double* s) {
    v = r3d_wave_sum(v);
    const int nw = blockDim.x >> 6;
    if (nw == 1) return v;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = s[0];
    for (int i = 1; i < nw; ++i) r += s[i];
    return r;
}

__device__ __forceinline__ uint32_t i8_amax8(const float* h, uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(h[j]) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    return m;
}

/* h = (r * rs) * (w + wadd) over a chunk. */
template <bool WBF16>
__device__ __forceinline__ void i8_norm8(const I8Raw<true>& r, const I8Raw<WBF16>& w, float wadd, float rs, float* h) {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = __fmul_rn(__fmul_rn(r.at(j), rs), __fadd_rn(w.at(j), wadd));
}

/* A row's scale from its largest magnitude's bits, and whether that is a number. */
__device__ __forceinline__ float i8_scale(uint32_t m, bool* fin) {
    const float amax = __uint_as_float(m);
    *fin = m < 0x7F800000u;
    return m == 0 ? 1.0f : *fin ? __builtin_fmaxf(amax * (1.0f / 127.0f), 0x1p-126f) : amax;
}

/* The codes of chunk i, four to a dword; 0 on a row whose scale is no number.  |h * inv| is 127 up
 * to a few roundings; added to 1.5 * 2^23 it is rounded to a whole number, to nearest even, whose two's
 * complement is the low byte of the sum. */
__device__ __forceinline__ void i8_codes8(uint8_t* qr, int64_t i, int64_t n, float inv, bool fin,
                                          const float* h) {
#pragma clang fp contract(off)                   /* the product is rounded before the sum */
    uint32_t c[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            d[j] = __float_as_uint(h[4 * k + j] * inv + 12582912.0f);
        const uint32_t lo = __builtin_amdgcn_perm(d[1], d[0], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(d[3], d[2], 0x04000c0cu);
        c[k] = fin ? lo | hi : 0u;
    }
    if (i + 8 <= n) {
        typedef uint32_t u32x2_u1 __attribute__((ext_vector_type(2), aligned(1)));
        *reinterpret_cast<u32x2_u1*>(qr + i) = u32x2_u1{c[0], c[1]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) qr[i + j] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
    }
}

template <int OP, bool XBF16, bool WBF16, int C>
__global__ __launch_bounds__(1024) void i8_band_kernel(I8BandArgs P) {
    __shared__ double s_sum[16];
    __shared__ uint32_t s_max[16];
    const int64_t row = blockIdx.x;
    const uint8_t* xr = P.x + row * P.x_pitch * (XBF16 ? 2 : 4);
    const uint8_t* rr = P.res ? reinterpret_cast<const uint8_t*>(P.res + row * P.r_pitch) : nullptr;
    uint8_t* ro = P.res ? reinterpret_cast<uint8_t*>(P.res_out + row * P.ro_pitch) : nullptr;
    uint8_t* qr = P.q + row * P.q_pitch;
    uint8_t* obr = P.ob ? P.ob + row * P.ob_pitch * (P.ob_bf16 ? 2 : 4) : nullptr;
    const int64_t n = P.n, step = 8 * (int64_t)blockDim.x, i0 = 8 * (int64_t)threadIdx.x;
    float rs = 1.0f;
    uint32_t m = 0;
    if constexpr (C > 0) {
        /* every load of the row before the first use of one; a lane past the row's end has zeros */
        float h[C][8];
        I8Raw<XBF16> x[C], y[C];                 /* y: up, or the residual */
#pragma unroll
        for (int c = 0; c < C; ++c) x[c] = i8_ld8<XBF16>(xr, i0 + c * step, n);
        if (OP == I8_GATED || (OP == I8_NORM && rr)) {
            const uint8_t* yr = OP == I8_GATED ? xr + (XBF16 ? 2 : 4) * n : rr;
#pragma unroll
            for (int c = 0; c < C; ++c) y[c] = i8_ld8<XBF16>(yr, i0 + c * step, n);
        }
        if constexpr (OP == I8_NORM) {
            I8Raw<WBF16> w[C];
#pragma unroll
            for (int c = 0; c < C; ++c) w[c] = i8_ld8<WBF16>(P.w, i0 + c * step, n);
            double ss = 0.0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (rr) x[c] = i8_add8(x[c], y[c], ro, i0 + c * step, n);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)x[c].at(j), (double)x[c].at(j), ss);
            }
            rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum) / (double)n + P.eps));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                i8_norm8<WBF16>(x[c], w[c], P.wadd, rs, h[c]);
                if (i0 + c * step + 8 > n) {     /* a zero past the end is no value (0 * inf) */
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (i0 + c * step + j >= n) h[c][j] = 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (OP == I8_GATED) {
                    i8_gated8<XBF16>(x[c], y[c], P.silu, h[c]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[c][j] = x[c].at(j);
                }
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) m = i8_amax8(h[c], m);
        m = i8_block_max(m, s_max);
        bool fin;
        const float s = i8_scale(m, &fin);
        const float inv = 1.0f / s;
        if (threadIdx.x == 0) P.scale[row * P.s_stride] = s;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t i = i0 + c * step;
            if (i >= n) break;
            i8_codes8(qr, i, n, inv, fin, h[c]);
            if (OP != I8_QUANT && obr) i8_st8(obr, i, n, h[c], P.ob_bf16);
        }
    } else {
        float h[8];
        if constexpr (OP == I8_NORM) {
            double ss = 0.0;
            for (int64_t i = i0; i < n; i += step) {
                I8Raw<true> x = i8_ld8<true>(xr, i, n);
                if (rr) x = i8_add8(x, i8_ld8<true>(rr, i, n), ro, i, n);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)x.at(j), (double)x.at(j), ss);
            }
            rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum) / (double)n + P.eps));
        }
        /* the norm's later walks read r where the first one wrote it: the same lane's own chunks */
        auto value = [&](int64_t i) {
            if constexpr (OP == I8_NORM) {
                i8_norm8<WBF16>(i8_ld8<true>(rr ? ro : xr, i, n), i8_ld8<WBF16>(P.w, i, n), P.wadd, rs, h);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j >= n) h[j] = 0.0f;
            } else {
                const I8Raw<XBF16> x = i8_ld8<XBF16>(xr, i, n);
                if (OP == I8_GATED) {
                    i8_gated8<XBF16>(x, i8_ld8<XBF16>(xr + (XBF16 ? 2 : 4) * n, i, n), P.silu, h);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = x.at(j);
                }
            }
        };
        for (int64_t i = i0; i < n; i += step) {
            value(i);
            m = i8_amax8(h, m);
        }
        m = i8_block_max(m, s_max);
        bool fin;
        const float s = i8_scale(m, &fin);
        const float inv = 1.0f / s;
        if (threadIdx.x == 0) P.scale[row * P.s_stride] = s;
        for (int64_t i = i0; i < n; i += step) {
            value(i);
            i8_codes8(qr, i, n, inv, fin, h);
            if (OP != I8_QUANT && obr) i8_st8(obr, i, n, h, P.ob_bf16);
        }
    }
}

}  // namespace r3d

#endif /* R3D_I8_BAND_H */
