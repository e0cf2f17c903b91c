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
 * the kernels that they follow do; here the narrowing would only move codes).  The 2^-126 keeps 1 / s finite.  The maximum is taken
 * over the magnitudes' bits, where an infinity is above every number and a NaN above that: a row
 * with a NaN has scale NaN and one with an infinity scale inf, both with codes 0, so the product
 * over the row is NaN and not a number that hides them.
 *
 * One workgroup a row, the row in registers (C chunks of 8 elements a lane) from the load to the
 * codes: every operand is read once and every result written once, which is all the traffic there
 * is; the kernels are bound by it.  Operands move in 16-byte accesses at element alignment
 * (gfx950's global memory takes them anywhere), so no pitch or base needs a kernel of its own; the
 * last n % 8 elements go one by one.  A row past the registers (C = 0) is walked twice. */
#ifndef R3D_I8_BAND_H
#define R3D_I8_BAND_H

#include "r3d_device.h"
#include "r3d_i8.h"

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

__device__ __forceinline__ float i8_bf(uint32_t b) { return __uint_as_float(b << 16); }

/* Eight elements from element i of a row of n on; zeros past its end. */
template <bool BF16>
__device__ __forceinline__ void i8_ld8(const uint8_t* row, int64_t i, int64_t n, float* v) {
    if (i + 8 <= n) {
        if (BF16) {
            const r3d_i32x4_u2 d = *reinterpret_cast<const r3d_i32x4_u2*>(row + 2 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float((uint32_t)d[j] << 16);
                v[2 * j + 1] = __uint_as_float((uint32_t)d[j] & 0xFFFF0000u);
            }
        } else {
            const r3d_f32x4_u4 lo = *reinterpret_cast<const r3d_f32x4_u4*>(row + 4 * i);
            const r3d_f32x4_u4 hi = *reinterpret_cast<const r3d_f32x4_u4*>(row + 4 * i + 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = lo[j];
                v[4 + j] = hi[j];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.0f;
            if (i + j < n)
                v[j] = BF16 ? i8_bf(reinterpret_cast<const uint16_t*>(row)[i + j])
                            : reinterpret_cast<const float*>(row)[i + j];
        }
    }
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

/* sigmoid(g) = 1 / (1 + exp(-g)) in f32, within 3 ulp: exp2 of the product's high part (its
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

/* The eight values h of chunk i (before the norm's scale: r). */
template <int OP, bool XBF16>
__device__ __forceinline__ void i8_values(const I8BandArgs& P, const uint8_t* xr, const uint8_t* rr,
                                          uint8_t* ro, int64_t i, float* h) {
    i8_ld8<XBF16>(xr, i, P.n, h);
    if (OP == I8_GATED) {
        float up[8];
        i8_ld8<XBF16>(xr + (XBF16 ? 2 : 4) * P.n, i, P.n, up);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float s = i8_sigmoid(h[j]);
            h[j] = (P.silu ? h[j] * s : s) * up[j];
        }
    }
    if (OP == I8_NORM && rr) {
        float a[8];
        i8_ld8<true>(rr, i, P.n, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = r3d_bf16_to_f32(r3d_bf16_rne(__fadd_rn(a[j], h[j])));
        i8_st8(ro, i, P.n, h, 1);
    }
}

/* The largest of a workgroup's values, or their sum, on every lane; `s` holds one a wave. */
__device__ __forceinline__ uint32_t i8_block_max(uint32_t v, uint32_t* s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = __shfl_xor(v, off, 64);
        v = v > o ? v : o;
    }
    const int nw = blockDim.x >> 6;
    if (nw == 1) return v;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t r = s[0];
    for (int i = 1; i < nw; ++i) r = r > s[i] ? r : s[i];
    return r;
}
__device__ __forceinline__ double i8_block_sum(double v, double* s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
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
__device__ __forceinline__ void i8_norm8(const float* w, float wadd, float rs, float* h) {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = __fmul_rn(__fmul_rn(h[j], rs), __fadd_rn(w[j], wadd));
}

/* A row's scale from its largest magnitude's bits, and whether that is a number. */
__device__ __forceinline__ float i8_scale(uint32_t m, bool* fin) {
    const float amax = __uint_as_float(m);
    *fin = m < 0x7F800000u;
    return m == 0 ? 1.0f : *fin ? __builtin_fmaxf(amax * (1.0f / 127.0f), 0x1p-126f) : amax;
}

/* The codes of chunk i, four to a dword; 0 on a row whose scale is no number.  |h * inv| is 127 up
 * to a few roundings, so rint gives at most 127. */
__device__ __forceinline__ void i8_codes8(uint8_t* qr, int64_t i, int64_t n, float inv, bool fin,
                                          const float* h) {
    uint32_t c[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = fin ? (int)__builtin_rintf(__fmul_rn(h[4 * k + j], inv)) : 0;
        c[k] = (uint32_t)(d[0] & 255) | (uint32_t)(d[1] & 255) << 8 | (uint32_t)(d[2] & 255) << 16 |
               (uint32_t)d[3] << 24;
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
        float h[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t i = i0 + c * step;
            if (i < n) {
                i8_values<OP, XBF16>(P, xr, rr, ro, i, h[c]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[c][j] = 0.0f;
            }
        }
        if (OP == I8_NORM) {
            float w[C][8];                       /* on its way while the sum is taken */
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (i0 + c * step < n) i8_ld8<WBF16>(P.w, i0 + c * step, n, w[c]);
            double ss = 0.0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)h[c][j], (double)h[c][j], ss);
            rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum) / (double)n + P.eps));
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (i0 + c * step < n) i8_norm8(w[c], P.wadd, rs, h[c]);
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
        if (OP == I8_NORM) {
            double ss = 0.0;
            for (int64_t i = i0; i < n; i += step) {
                i8_values<OP, XBF16>(P, xr, rr, ro, i, h);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)h[j], (double)h[j], ss);
            }
            rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum) / (double)n + P.eps));
        }
        /* the norm's later walks read r where the first one wrote it: the same lane's own chunks */
        auto value = [&](int64_t i) {
            if (OP == I8_NORM) {
                i8_ld8<true>(rr ? ro : xr, i, n, h);
                float w[8];
                i8_ld8<WBF16>(P.w, i, n, w);
                i8_norm8(w, P.wadd, rs, h);
            } else {
                i8_values<OP, XBF16>(P, xr, nullptr, nullptr, i, h);
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
