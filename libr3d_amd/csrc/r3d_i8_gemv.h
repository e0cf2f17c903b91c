/* r3d_i8_gemv.h -- gemm_nt_q at i8a8 for up to eight tokens: a weight stream, bound by HBM.
 *
 * A wave owns 8 weight rows and one chunk of K, and walks it a 128-byte line at a time.  One
 * 16-byte load a lane takes the whole line of 8 rows (8 lanes a line), where the matrix core's own
 * layout of 16 rows x 64 bytes would take half lines.  The order of K inside a product is free as
 * long as both sides share it, so v_mfma_i32_16x16x64_i8 is fed as it comes: source A's row i is
 * (weight row i % 8, pieces of parity i / 8), source B's column j is (token j % 8, parity j / 8), and
 * of the 16 x 16 results those with i / 8 = j / 8 are wanted; one cross-lane add at the end joins the
 * two halves.  Half the matrix core's work is thrown away and it still idles: it takes 16 cycles for
 * 1 KB of weights, which HBM brings a compute unit in 80.
 *
 * The tokens lie in LDS (staged once, beside the first weight loads in flight): read from L2 next to
 * every weight line instead they cost 23.1 us where this takes 20.2 (M = 1, N = 21504, K = 5376).
 * Weight lines go from memory to registers, D ahead.  Rows past N are past the buffer's records and
 * columns past K are asked for there; both read 0.  The chunks of a row block are waves of one
 * workgroup, joined through LDS; the sums are integers, so no order changes a result.
 *
 * M = 1, N = 21504, K = 5376: 20.2 us, 5.7 TB/s.  Of D = 2, 3, 4, 6, 8, of 8 or 16 rows and of 4, 8
 * or 16 waves a workgroup, D = 4 with 8 rows and 4 waves is the best over 274 shapes (7 % off the
 * best of all of them at each shape; the next, D = 3 and D = 6, 9 %).
 */
#ifndef R3D_I8_GEMV_H
#define R3D_I8_GEMV_H

#include "r3d_device.h"
#include "r3d_epi_dev.h"
#include "r3d_i8_any.h"

namespace r3d {

constexpr uint32_t kI8Oob = 0x80000000u;      /* past every record count: reads 0 */

/* 16 bytes at lane offset voff and uniform offset soff; NT 2: streamed */
template <int NT>
__device__ __forceinline__ r3d_i32x4 i8_buf16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
    return __builtin_bit_cast(r3d_i32x4,
                              __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, NT));
}

/* A and B in bytes, K a row's bytes */
struct I8GemvArgs {
    const uint8_t* A;
    const uint8_t* B;
    const float* SA;
    const float* SB;
    uint16_t* Y;
    int M, N, K, a_pitch, b_pitch, kc, per;   /* kc chunks of `per` lines */
    int64_t sa_stride, sb_stride, y_pitch;
};

template <class T, int W>
__global__ __launch_bounds__(64 * W) void i8_gemv_kernel(typename T::GemvArgs P) {
    constexpr int D = 4, SB = 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_a[];   /* [M][lp]; then [W][16] i32x4 */
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bpw = i8_uniform(W / P.kc);                       /* row blocks a workgroup */
    const int rb = i8_uniform(wave / P.kc), c = wave - rb * P.kc;
    const int64_t n0 = ((int64_t)blockIdx.x * bpw + rb) * 8;
    const int r8 = lane & 7, chunk = ((lane >> 3) & 1) | ((lane >> 4) << 1);

    const int rows = P.N - n0 < 8 ? (P.N > n0 ? (int)(P.N - n0) : 0) : 8;
    const __amdgpu_buffer_rsrc_t rB =
        r3d_rsrc(P.B + (rows ? n0 : 0) * P.b_pitch, rows ? (int64_t)(rows - 1) * P.b_pitch + P.K : 0);
    const __amdgpu_buffer_rsrc_t rA = r3d_rsrc(P.A, (int64_t)(P.M - 1) * P.a_pitch + P.K);
    const uint32_t wo = (uint32_t)(r8 * P.b_pitch + 16 * chunk);
    const int l0 = c * P.per;
    const int k1 = (l0 + P.per) * 128 < P.K ? (l0 + P.per) * 128 : P.K;   /* the chunk's end in K */
    const int steps = k1 > l0 * 128 ? (k1 - l0 * 128 + 127) >> 7 : 0;

    /* the tokens on their way to LDS, rows of K rounded up to 128 and 16 more (bank groups) */
    const int lp = ((P.K + 127) & ~127) + 16, pieces = lp >> 4, total = P.M * pieces;
    auto st_load = [&](int i) __attribute__((always_inline)) {
        const int m = i / pieces, k = 16 * (i - m * pieces);
        return i8_buf16<0>(rA, i < total && k < P.K ? (uint32_t)(m * P.a_pitch + k) : kI8Oob, 0);
    };
    r3d_i32x4 st[SB];
#pragma unroll
    for (int j = 0; j < SB; ++j) st[j] = st_load(threadIdx.x + 64 * W * j);

    /* what the epilogue needs */
    const bool mine = c == 0 && lane < 32 && (lane & 8) == 0;
    const int ml = lane & 7, nl = 4 * ((lane >> 4) & 1);
    float sb[4], sa = 0.0f;
    if (T::kScaled && mine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + nl + i;
            sb[i] = n < P.N ? P.SB[n * P.sb_stride] : 0.0f;
        }
        if (ml < P.M) sa = P.SA[ml * P.sa_stride];
    }

    r3d_i32x4 w[D];
    typename T::Acc4 acc = {0, 0, 0, 0};
    auto load = [&](int s) __attribute__((always_inline)) {
        const int k = (l0 + s) * 128;
        return i8_buf16<2>(rB, 16 * chunk < k1 - k ? wo : kI8Oob, k);   /* zeros past the chunk's end */
    };
#pragma unroll
    for (int d = 0; d < D; ++d) w[d] = load(d);
#pragma unroll
    for (int j = 0; j < SB; ++j) {
        const int i = threadIdx.x + 64 * W * j;
        if (i < total) *reinterpret_cast<r3d_i32x4*>(s_a + 16 * i) = st[j];
    }
    for (int i = threadIdx.x + 64 * W * SB; i < total; i += 64 * W)
        *reinterpret_cast<r3d_i32x4*>(s_a + 16 * i) = st_load(i);
    /* the tokens are there; the weight loads stay in flight (__syncthreads would wait for them) */
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    /* a column past M repeats the last token: its results are not read */
    const uint8_t* xa = s_a + (r8 < P.M ? r8 : P.M - 1) * lp + 16 * chunk;
    for (int s = 0; s < steps; s += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int k = (l0 + s + d) * 128;                   /* past K the weights are zeros */
            r3d_i32x4 x = *reinterpret_cast<const r3d_i32x4*>(xa + (k < lp - 16 ? k : 0));
            if (T::kZeroBoth && s + d >= steps) x = r3d_i32x4{0, 0, 0, 0};
            acc = T::mfma16(w[d], x, acc);
            w[d] = load(s + D + d);
        }
    }
    /* lane l holds i = 4 (l / 16) .. + 3, j = l % 16; halves (0, 0) and (1, 1) are 40 lanes apart */
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl(acc[i], (lane + 40) & 63, 64);
    if (P.kc > 1) {
        typename T::Acc4* const s_part = reinterpret_cast<typename T::Acc4*>(s_a);
        const int slot = (lane >> 4) * 8 + ml;                  /* 16 lanes hold the results */
        __syncthreads();                                        /* the tokens are read */
        if (c > 0 && lane < 32 && (lane & 8) == 0) s_part[wave * 16 + slot] = acc;
        __syncthreads();
        if (mine)
            for (int o = 1; o < P.kc; ++o) acc += s_part[(wave + o) * 16 + slot];
    }
    const int64_t n = n0 + nl;
    if (!mine || ml >= P.M || n >= P.N) return;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = T::kScaled ? i8_out(acc[i], sa, sb[i]) : (float)acc[i];
    if constexpr (T::kEpi) {
        epi_values<4>(P.e, v, ml, n, P.N);
        epi_store<4>(P.e, P.Y, P.y_pitch, v, ml, n, P.N);
        return;
    }
    uint16_t* y = P.Y + ml * P.y_pitch + n;
    if (n + 4 <= P.N) {
        *reinterpret_cast<r3d_u32x2_u2*>(y) =
            r3d_u32x2_u2{r3d_pack_bf16x2(v[0], v[1]), r3d_pack_bf16x2(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < P.N) y[i] = r3d_bf16_rne(v[i]);
    }
}

}  // namespace r3d

#endif /* R3D_I8_GEMV_H */
