/* r3d_epi_dev.h -- gemm_nt_epi's epilogue on the device: from a product's f32 value v[m, n] (the sum, or with
 * scales (sum * a_scale[m]) * b_scale[n])
 *     y[m, n] = act(v + bias[n]) + residual[m, n]
 * in f32, rounded once, to y's type.  A lane owns some consecutive columns of a token, reads their residual
 * and writes their y, so that y may be the residual's memory. */
#ifndef R3D_EPI_DEV_H
#define R3D_EPI_DEV_H

#include "r3d_act_dev.h"
#include "r3d_device.h"

namespace r3d {

struct EpiArgs {
    const void* bias;        /* [N], or null */
    const void* res;         /* [M, N], or null; may be y */
    int64_t bias_stride, r_pitch;
    int act, bias_bf16, res_bf16, y_bf16;
};

/* Elements n .. n + W - 1 of a bf16 or f32 row as f32; those from N on are 0. */
template <int W>
__device__ __forceinline__ void epi_load(const void* row, int bf16, int64_t n, int64_t N, float* v) {
    static_assert(W == 4 || W == 8, "8 or 16 bytes of bf16");
    if (bf16) {
        const uint16_t* p = static_cast<const uint16_t*>(row) + n;
        if (n + W <= N) {
            uint32_t d[W / 2];
            if constexpr (W == 8) *reinterpret_cast<r3d_i32x4*>(d) = *reinterpret_cast<const r3d_i32x4_u2*>(p);
            else *reinterpret_cast<uint2*>(d) = __builtin_bit_cast(uint2, *reinterpret_cast<const r3d_u32x2_u2*>(p));
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = __uint_as_float(i & 1 ? d[i >> 1] & 0xFFFF0000u : d[i >> 1] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = n + i < N ? r3d_bf16_to_f32(p[i]) : 0.0f;
        }
    } else {
        const float* p = static_cast<const float*>(row) + n;
        if (n + W <= N) {
#pragma unroll
            for (int i = 0; i < W; i += 4) *reinterpret_cast<r3d_f32x4*>(v + i) = *reinterpret_cast<const r3d_f32x4_u4*>(p + i);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = n + i < N ? p[i] : 0.0f;
        }
    }
}

/* bias[n .. n + W - 1]; 0 without a bias and from N on */
template <int W>
__device__ __forceinline__ void epi_bias(const EpiArgs& E, int64_t n, int64_t N, float* b) {
#pragma unroll
    for (int i = 0; i < W; ++i) b[i] = 0.0f;
    if (!E.bias) return;
    if (E.bias_stride == 1) {
        epi_load<W>(E.bias, E.bias_bf16, n, N, b);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (n + i < N)
                b[i] = E.bias_bf16 ? r3d_bf16_to_f32(static_cast<const uint16_t*>(E.bias)[(n + i) * E.bias_stride])
                                   : static_cast<const float*>(E.bias)[(n + i) * E.bias_stride];
    }
}

/* act and residual over v + bias, in place */
template <int W>
__device__ __forceinline__ void epi_finish(const EpiArgs& E, float* v, int64_t m, int64_t n, int64_t N) {
    act_values<W>(E.act, v);
    if (E.res) {
        float r[W];
        epi_load<W>(static_cast<const uint8_t*>(E.res) + m * E.r_pitch * (E.res_bf16 ? 2 : 4), E.res_bf16, n, N, r);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += r[i];
    }
}

template <int W>
__device__ __forceinline__ void epi_store(const EpiArgs& E, void* Y, int64_t y_pitch, const float* v, int64_t m,
                                          int64_t n, int64_t N) {
    if (E.y_bf16) {
        uint16_t* y = static_cast<uint16_t*>(Y) + m * y_pitch + n;
        uint32_t d[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) d[i] = r3d_pack_bf16x2(v[2 * i], v[2 * i + 1]);
        if (n + W <= N) {
            if constexpr (W == 8) *reinterpret_cast<r3d_i32x4_u2*>(y) = *reinterpret_cast<const r3d_i32x4*>(d);
            else *reinterpret_cast<r3d_u32x2_u2*>(y) = r3d_u32x2_u2{d[0], d[1]};
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (n + i < N) y[i] = (uint16_t)(d[i >> 1] >> (16 * (i & 1)));
        }
    } else {
        float* y = static_cast<float*>(Y) + m * y_pitch + n;
        if (n + W <= N) {
#pragma unroll
            for (int i = 0; i < W; i += 4) *reinterpret_cast<r3d_f32x4_u4*>(y + i) = *reinterpret_cast<const r3d_f32x4*>(v + i);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (n + i < N) y[i] = v[i];
        }
    }
}

/* bias, act, residual over W values */
template <int W>
__device__ __forceinline__ void epi_values(const EpiArgs& E, float* v, int64_t m, int64_t n, int64_t N) {
    float b[W];
    epi_bias<W>(E, n, N, b);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += b[i];
    epi_finish<W>(E, v, m, n, N);
}

/* A token's sums in LDS, 16 bytes off a multiple of 128: 16-byte stores of 8 tokens meet no bank twice. */
constexpr int epi_row(int bn) { return 4 * bn + 16; }

/* The epilogue of ROWS tokens from m0 on and BN columns from n0 on, their sums in LDS: eight columns a lane,
 * the same ones for every token it takes, so that scales and bias are read once; y leaves and the residual
 * arrives in whole runs of a row.  One token at a time: two and four at once, for their loads' sake, spill 24
 * and 211 registers of the wide kernel, whose other half still holds its sums (2048 x 21504 x 5376 int8,
 * gelu_tanh: one 247 us, four 283). */
template <class T, int BN, int THREADS, int ROWS>
__device__ __forceinline__ void epi_tile(const typename T::TileArgs& P, const uint8_t* smem, int64_t m0, int64_t n0) {
    constexpr int CPR = BN / 8, STEP = THREADS / CPR;
    static_assert(THREADS % CPR == 0, "a lane keeps its columns");
    const int cc = threadIdx.x % CPR, r0 = threadIdx.x / CPR;
    const int64_t n = n0 + 8 * cc;
    if (n >= P.N) return;                                       /* no barrier in here */
    float b[8], sb[8];
    epi_bias<8>(P.e, n, P.N, b);
    if (T::kScaled) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sb[i] = P.SB[(n + i < P.N ? n + i : P.N - 1) * P.sb_stride];
    }
    for (int r = r0; r < ROWS; r += STEP) {
        const int64_t m = m0 + r;
        if (m >= P.M) return;
        float v[8], res[8];
        const float sa = T::kScaled ? P.SA[m * P.sa_stride] : 1.0f;
        if (P.e.res)
            epi_load<8>(static_cast<const uint8_t*>(P.e.res) + m * P.e.r_pitch * (P.e.res_bf16 ? 2 : 4), P.e.res_bf16, n, P.N, res);
        const typename T::Acc4* s = reinterpret_cast<const typename T::Acc4*>(smem + r * epi_row(BN) + 32 * cc);
        const typename T::Acc4 lo = s[0], hi = s[1];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = (float)(i < 4 ? lo[i & 3] : hi[i & 3]);
            v[i] = (T::kScaled ? f * sa * sb[i] : f) + b[i];
        }
        act_values<8>(P.e.act, v);
        if (P.e.res) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += res[i];
        }
        epi_store<8>(P.e, P.Y, P.y_pitch, v, m, n, P.N);
    }
}

}  // namespace r3d

#endif /* R3D_EPI_DEV_H */
