/* r3d_block.hip -- rmsnorm_block on gfx950 (r3d_block.h has the formulas): kernel and entry.
 *
 * A workgroup a row, the row in registers (C chunks of 8 elements a lane) from its loads to the last store, so
 * that x, the residual and the gate are read once and every result is written once; that traffic is what bounds
 * it over many rows, and over few the chain of a load and two or three reductions over the workgroup.  All
 * arithmetic is in f32, the two sums of squares in f64; h goes on into the second norm as it stands in f32 and
 * is rounded to bf16 for residual_out alone, v is rounded (or quantised) once.
 *
 * Measured on MI355X (a 1 GiB copy 5.05 TB/s): 2048 x 5376 with post norm, residual and both results 18.4 us, 4.8
 * TB/s (20.7 with operands that come from HBM alone); 333 x 5376 with a gate and int8 codes 7.4 to 8.6; 1 x 5376 4.6 to 5.1. */
#include <hip/hip_runtime.h>

#include <stdio.h>

#include "r3d_band.h"
#include "r3d_block.h"
#include "r3d_dump.h"
#include "r3d_i8_band.h"
#include "r3d_i8_launch.h"

namespace r3d {

struct BlockArgs {
    const uint8_t* x;
    const uint8_t* res;
    const uint8_t* w_post;
    const uint8_t* gate;
    const uint8_t* w_pre;
    uint8_t* res_out;
    uint8_t* out;
    uint8_t* q;
    float* scale;
    int64_t n, x_pitch, r_pitch, g_pitch, ro_pitch, o_pitch, q_pitch, s_pitch;
    double eps;
    float wadd, res_scale;
    int gate_kind, codes, out_bf16, past;
};

/* Eight results to element i of a row of n on; past: not to be kept in the caches. */
__device__ __forceinline__ void block_st8(uint8_t* row, int64_t i, int64_t n, const float* v, int bf16, int past) {
    if (bf16) {
        r3d_i32x4_u2 d;
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = (int)r3d_pack_bf16x2(v[2 * j], v[2 * j + 1]);
        r3d_i32x4_u2* const to = reinterpret_cast<r3d_i32x4_u2*>(row + 2 * i);
        if (i + 8 <= n && past) {
            __builtin_nontemporal_store(d, to);
        } else if (i + 8 <= n) {
            *to = d;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < n) reinterpret_cast<uint16_t*>(row)[i + j] = (uint16_t)((uint32_t)d[j >> 1] >> (16 * (j & 1)));
        }
    } else {
        r3d_f32x4_u4* const to = reinterpret_cast<r3d_f32x4_u4*>(row + 4 * i);
        const r3d_f32x4_u4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
        if (i + 8 <= n && past) {
            __builtin_nontemporal_store(lo, to);
            __builtin_nontemporal_store(hi, to + 1);
        } else if (i + 8 <= n) {
            to[0] = lo;
            to[1] = hi;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < n) reinterpret_cast<float*>(row)[i + j] = v[j];
        }
    }
}

/* e4m3 codes of a chunk of 8: quant_act_fp8's arithmetic (r3d_band.h), a group of 128 in 16 lanes.  Every lane
 * takes part in the maximum; a lane past the row's end has zeros. */
__device__ __forceinline__ void block_e4m3(const float* v, uint8_t* qr, float* sr, int64_t i, int64_t n) {
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
    amax = r3d_max16(amax);
    /* a normal number, as quant_act_i8's: 1 / s of a smaller one is infinite, and 0 times that no code */
    const float s = amax > 0.0f ? fmaxf(amax * (1.0f / 448.0f), 0x1p-126f) : 1.0f;
    const float inv = 1.0f / s;
    if (i >= n) return;
    if ((threadIdx.x & 15) == 0) sr[i >> 7] = s;
    float c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = r3d_band_clamp448(v[j] * inv);
    const uint32_t lo = r3d_e4m3x4_rne(c[0], c[1], c[2], c[3]), hi = r3d_e4m3x4_rne(c[4], c[5], c[6], c[7]);
    if (i + 8 <= n) {
        typedef uint32_t u32x2_u1 __attribute__((ext_vector_type(2), aligned(1)));
        *reinterpret_cast<u32x2_u1*>(qr + i) = u32x2_u1{lo, hi};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) qr[i + j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
}

template <bool XBF16, bool WBF16, int C>
__global__ __launch_bounds__(1024) void block_kernel(BlockArgs P) {
    __shared__ double s_sum[2][16];
    __shared__ uint32_t s_max[16];
    constexpr int XB = XBF16 ? 2 : 4, WB = WBF16 ? 2 : 4;
    const int64_t row = blockIdx.x, n = P.n, step = 8 * (int64_t)blockDim.x, i0 = 8 * (int64_t)threadIdx.x;
    const uint8_t* const xr = P.x + row * P.x_pitch * XB;
    const uint8_t* const gr = P.gate ? P.gate + row * P.g_pitch * WB : nullptr;
    /* every load before the first use of one (the last weights too where registers allow) */
    I8Raw<XBF16> x[C];
    I8Raw<true> r[C];
    I8Raw<WBF16> wp[C], g[C], wn[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = i8_ld8<XBF16>(xr, i0 + c * step, n);
    if (P.w_post) {
#pragma unroll
        for (int c = 0; c < C; ++c) wp[c] = i8_ld8<WBF16>(P.w_post, i0 + c * step, n);
    }
    if (P.res) {
        const uint8_t* const rr = P.res + row * P.r_pitch * 2;
#pragma unroll
        for (int c = 0; c < C; ++c) r[c] = i8_ld8<true>(rr, i0 + c * step, n);
    }
    /* f32 weights are twice the registers: past two chunks their gate waits for the first sum (with every load before it four
     * chunks spilled 17 to 25 registers: 2048 x 8192 41.7 us for 24.6, with a gate an element 51.3 for 38.4) */
    constexpr bool EARLY_GATE = WBF16 || C <= 2, EARLY = C <= (WBF16 ? 2 : 1);
    if (EARLY_GATE && P.gate_kind == BLOCK_GATE_ROWS) {
#pragma unroll
        for (int c = 0; c < C; ++c) g[c] = i8_ld8<WBF16>(gr, i0 + c * step, n);
    }
    float gt = 1.0f;
    if (P.gate_kind == BLOCK_GATE_TOKEN)
        gt = WBF16 ? r3d_bf16_to_f32(*reinterpret_cast<const uint16_t*>(gr)) : *reinterpret_cast<const float*>(gr);
    if (EARLY && P.w_pre) {
#pragma unroll
        for (int c = 0; c < C; ++c) wn[c] = i8_ld8<WBF16>(P.w_pre, i0 + c * step, n);
    }
    float h[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) h[c][j] = x[c].at(j);
    if (P.w_post) {
        double ss = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)h[c][j], (double)h[c][j], ss);
        const float rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum[0]) / (double)n + P.eps));
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[c][j] = __fmul_rn(__fmul_rn(h[c][j], rs), __fadd_rn(wp[c].at(j), P.wadd));
    }
    if (!EARLY_GATE && P.gate_kind == BLOCK_GATE_ROWS) {
#pragma unroll
        for (int c = 0; c < C; ++c) g[c] = i8_ld8<WBF16>(gr, i0 + c * step, n);
    }
    if (P.gate_kind == BLOCK_GATE_ROWS) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[c][j] *= g[c].at(j);
    } else if (P.gate_kind == BLOCK_GATE_TOKEN) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[c][j] *= gt;
    }
    if (P.res) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[c][j] = __builtin_fmaf(r[c].at(j), P.res_scale, h[c][j]);
    }
    /* what lies past the row's end is no value (0 * inf) */
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (i0 + c * step + 8 > n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i0 + c * step + j >= n) h[c][j] = 0.0f;
        }
    if (!EARLY && P.w_pre) {
#pragma unroll
        for (int c = 0; c < C; ++c) wn[c] = i8_ld8<WBF16>(P.w_pre, i0 + c * step, n);
    }
    if (P.res_out) {
        uint8_t* const ro = P.res_out + row * P.ro_pitch * 2;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (i0 + c * step < n) block_st8(ro, i0 + c * step, n, h[c], 1, P.past);
    }
    if (!P.w_pre) return;
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)h[c][j], (double)h[c][j], ss);
    const float rs = (float)(1.0 / sqrt(i8_block_sum(ss, s_sum[1]) / (double)n + P.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[c][j] = __fmul_rn(__fmul_rn(h[c][j], rs), __fadd_rn(wn[c].at(j), P.wadd));
        if (i0 + c * step + 8 > n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i0 + c * step + j >= n) h[c][j] = 0.0f;
        }
    }
    if (P.out) {
        uint8_t* const o = P.out + row * P.o_pitch * (P.out_bf16 ? 2 : 4);
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (i0 + c * step < n) block_st8(o, i0 + c * step, n, h[c], P.out_bf16, P.past);
    }
    if (P.codes == BLOCK_I8) {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) m = i8_amax8(h[c], m);
        m = i8_block_max(m, s_max);
        bool fin;
        const float s = i8_scale(m, &fin);
        const float inv = 1.0f / s;
        if (threadIdx.x == 0) P.scale[row * P.s_pitch] = s;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (i0 + c * step < n) i8_codes8(P.q + row * P.q_pitch, i0 + c * step, n, inv, fin, h[c]);
    } else if (P.codes == BLOCK_E4M3) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            block_e4m3(h[c], P.q + row * P.q_pitch, P.scale + row * P.s_pitch, i0 + c * step, n);
    }
}

static int block_entry(const RadArgs* a, RadStream s) {
    if (env_no_block()) return RAD_E_UNSUPPORTED;
    BlockPlan P{};
    const int rc = plan_block(a, &P);
    if (rc) return rc;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    const BlockGeom g = block_geom(P.rows, P.n);
    if (g.lanes < 64 || g.lanes > 1024 || 8 * (int64_t)g.lanes * g.chunks < P.n) return RAD_E_UNSUPPORTED;
    const BlockArgs k{P.x, P.res, P.w_post, P.gate, P.w_pre, P.res_out, P.out, P.q, P.scale, P.n, P.x_pitch,
                      P.r_pitch, P.g_pitch, P.ro_pitch, P.o_pitch, P.q_pitch, P.s_pitch, P.eps, P.wadd, P.res_scale,
                      P.gate_kind, P.codes, P.out_bf16, g.past};
    const dim3 grid((unsigned)P.rows), block((unsigned)g.lanes);
    hipStream_t stream = (hipStream_t)s;
#define R3D_BLOCK_C(X_, W_)                                                                       \
    switch (g.chunks) {                                                                           \
        case 1: hipLaunchKernelGGL((block_kernel<X_, W_, 1>), grid, block, 0, stream, k); break;  \
        case 2: hipLaunchKernelGGL((block_kernel<X_, W_, 2>), grid, block, 0, stream, k); break;  \
        case 3: hipLaunchKernelGGL((block_kernel<X_, W_, 3>), grid, block, 0, stream, k); break;  \
        default: hipLaunchKernelGGL((block_kernel<X_, W_, 4>), grid, block, 0, stream, k); break; \
    }
    if (P.x_bf16) {
        if (P.w_bf16) { R3D_BLOCK_C(true, true) } else { R3D_BLOCK_C(true, false) }
    } else {
        if (P.w_bf16) { R3D_BLOCK_C(false, true) } else { R3D_BLOCK_C(false, false) }
    }
#undef R3D_BLOCK_C
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("rmsnorm_block", e);
}

}  // namespace r3d

extern "C" int r3d_rad_rmsnorm_block(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("rmsnorm_block", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::block_entry(x, t);
    });
}
