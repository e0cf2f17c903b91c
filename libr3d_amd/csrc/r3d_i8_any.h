/* r3d_i8_any.h -- gemm_nt_q at i8a8 for any K, base and pitch.
 *
 * A wave owns 32 weight rows x 16 TM tokens and walks K 64 at a time: one
 * v_mfma_i32_16x16x64_i8 per 16 x 16 sub-tile with the weights as source A (lane l: row l % 16,
 * K bytes [16 (l / 16), +16)) and the tokens as source B, summed exactly in i32.  Each 16-byte
 * piece is assembled from five aligned dword loads (r3d_gemm_any.h) and the weights' bytes past K
 * are set to zero, so whatever follows a row in memory meets a zero.  Result lane l holds
 * D[4 (l / 16) + i][l % 16]: four consecutive weight rows of one token.
 *
 * It is what runs where 16-byte loads cannot (K % 16, an odd base or pitch): bound by its own
 * dword loads, not by memory, and a weight is read once for every 16 TM tokens (us at N = 21504, K = 5375; beside them
 * the other kernels at K = 5376: 1 token 135, 20.9; 16 129, 23.1; 333 734, 56 to 61; 2048 3843, 215 to 222). */
#ifndef R3D_I8_ANY_H
#define R3D_I8_ANY_H

#include "r3d_gemm_any.h"

namespace r3d {

/* A value that is the same on every lane, as such: the quotient of two of them is computed on the
 * vector unit, and a buffer resource made from one of its lanes' values would be loaded in a loop
 * over the lanes. */
__device__ __forceinline__ int i8_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* (f32(sum) * a_scale) * b_scale, the epilogue of every i8a8 kernel */
__device__ __forceinline__ float i8_out(int sum, float sa, float sb) {
    return __fmul_rn(__fmul_rn((float)sum, sa), sb);
}

/* Zeros in place of the bytes of a 16-byte piece past its first `left`. */
__device__ __forceinline__ r3d_i32x4 i8_keep(r3d_i32x4 v, int left) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int b = left - 4 * j;
        v[j] = b >= 4 ? v[j] : b <= 0 ? 0 : v[j] & ((1 << (8 * b)) - 1);
    }
    return v;
}

template <int TM>
__global__ __launch_bounds__(256) void i8_any_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ SA, const uint8_t* __restrict__ B,
    const float* __restrict__ SB, uint16_t* __restrict__ Y, int M, int N, int K, int64_t a_pitch,
    int64_t b_pitch, int64_t y_pitch, int64_t sa_stride, int64_t sb_stride) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 128 + 32 * wave;
    const int64_t m0 = (int64_t)blockIdx.y * 16 * TM;
    if (n0 >= N) return;                                /* whole wave: no barrier follows */
    /* a buffer a fragment: 16 rows of any pitch the host allows stay under 2^31 bytes */
    AnyBuf bw[2], ba[TM];
    uint32_t ow[2], oa[TM];
    bool iw[2], ia[TM];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int64_t n = n0 + 16 * f;
        const int rows = N - n < 16 ? (int)(N > n ? N - n : 0) : 16;
        bw[f] = any_buf(B + (rows ? n : 0) * b_pitch, rows ? (rows - 1) * b_pitch + K : 0);
        ow[f] = (uint32_t)(r16 * b_pitch);
        iw[f] = r16 < rows;
    }
#pragma unroll
    for (int f = 0; f < TM; ++f) {
        const int64_t m = m0 + 16 * f;
        const int rows = M - m < 16 ? (int)(M > m ? M - m : 0) : 16;
        ba[f] = any_buf(A + (rows ? m : 0) * a_pitch, rows ? (rows - 1) * a_pitch + K : 0);
        oa[f] = (uint32_t)(r16 * a_pitch);
        ia[f] = r16 < rows;
    }
    r3d_i32x4 acc[2][TM];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[f][t] = r3d_i32x4{0, 0, 0, 0};
    for (int k0 = 0; k0 < K; k0 += 64) {
        const int k = k0 + 16 * q;
        r3d_i32x4 w[2], x[TM];
#pragma unroll
        for (int f = 0; f < 2; ++f)
            w[f] = i8_keep(any_ld16(bw[f], iw[f] && k < K ? ow[f] + k : kAnyOob, false), K - k);
#pragma unroll
        for (int t = 0; t < TM; ++t) x[t] = any_ld16(ba[t], ia[t] && k < K ? oa[t] + k : kAnyOob, false);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < TM; ++t)
                acc[f][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[f], x[t], acc[f][t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int64_t m = m0 + 16 * t + r16;
        if (m >= M) continue;
        const float sa = SA[m * sa_stride];
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t n = n0 + 16 * f + 4 * q + i;
                if (n < N) Y[m * y_pitch + n] = r3d_bf16_rne(i8_out(acc[f][t][i], sa, SB[n * sb_stride]));
            }
    }
}

}  // namespace r3d

#endif /* R3D_I8_ANY_H */
