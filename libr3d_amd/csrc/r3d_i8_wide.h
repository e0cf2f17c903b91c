/* r3d_i8_wide.h -- gemm_nt_q at i8a8 on a 256 x 256 tile, for the largest products: eight waves (4
 * along N x 2 along M, two a SIMD), a wave 64 weight rows x 128 tokens in 2 x 4 results of
 * v_mfma_i32_32x32x32_i8.  Operands, units and epilogue as in r3d_i8_tile.h.
 *
 * A stage (128 of K, 64 KB) leaves room for a ring of two.  The stage's weights and the first half of
 * its tokens are in registers when its step begins, so two barriers a step free the ring in halves
 * and every load has one and a half steps to land:
 *   mid  (a fifth into the step)  weights and first halves are read: stage s + 2's go out in their
 *                                 place; this stage's second halves are here
 *   end  (five eighths)           the second halves are read and go out; stage s + 1's weights and
 *                                 first halves are here
 * Each operand piece is read right after the last product that used its registers, 64 cycles of
 * matrix work at a time (sched_barrier: left to itself the compiler gathers the reads at the end of
 * the step).  A wave raises its priority over its products.
 *
 * 2048 x 21504 x 5376: 213 to 222 us in calls one after the other, 2.1 to 2.2 POP/s; in kernel traces 210 at
 * best and 250 to 261 in the median (when it was 214: one barrier a step on 16 x 16 x 64 products 267; loads of
 * 16 rows x half lines 225).  The chip's power bounds it, not a unit: the same launch over zeros takes
 * 153 us, and torch's library product of the same codes 216 to 256. */
#ifndef R3D_I8_WIDE_H
#define R3D_I8_WIDE_H

#include "r3d_i8_tile.h"

namespace r3d {

template <class T>
__global__ __launch_bounds__(512) void i8_wide_kernel(typename T::TileArgs P) {
    constexpr int BN = 256, BM = 256, AOFF = BN * 128, STAGE = (BN + BM) * 128;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lj = lane & 31, lh = lane >> 5;
    const int wn = wave & 3, wm = wave >> 2;

    const int bid = blockIdx.x, units = P.tiles * P.kc;
    const int per = units >> 3, rem = units & 7, xcd = bid & 7;
    const int u = xcd * per + (xcd < rem ? xcd : rem) + (bid >> 3);
    const int kci = i8_uniform(u / P.tiles), t = u - kci * P.tiles;
    constexpr int GN = 8;
    const int grid_n = i8_uniform(P.tiles / P.grid_m);
    const int grp = i8_uniform(t / (GN * P.grid_m)), in = t - grp * GN * P.grid_m;
    const int gw = grid_n - grp * GN < GN ? grid_n - grp * GN : GN;
    const int tm = i8_uniform(in / gw);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)(grp * GN + in - tm * gw) * BN;
    const int k0 = kci * P.cst * 128;
    const int kend = k0 + P.cst * 128 < P.K ? k0 + P.cst * 128 : P.K;
    const int steps = (kend - k0 + 127) >> 7;

    const __amdgpu_buffer_rsrc_t rB = r3d_rsrc(P.B + n0 * P.b_pitch, (P.N - 1 - n0) * (int64_t)P.b_pitch + P.K);
    const __amdgpu_buffer_rsrc_t rA = r3d_rsrc(P.A + m0 * P.a_pitch, (P.M - 1 - m0) * (int64_t)P.a_pitch + P.K);
    /* image j: rows 8 j .. + 7 of 128 bytes, a line a row; lane (row lr, place) fetches the 16-byte
     * piece place ^ lr.  A wave loads weight images wave + 8 i; token images: i = 0, 1 the first
     * halves of the two token halves (rows 0-63 and 128-191), i = 2, 3 the second ones */
    const int lr = lane >> 3, col = 16 * ((lane & 7) ^ lr);
    uint32_t woff[4], aoff[4];
    int wimg[4], aimg[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        wimg[i] = wave + 8 * i;
        const int64_t n = n0 + 8 * wimg[i] + lr;
        woff[i] = (uint32_t)(((n < P.N ? n : P.N - 1) - n0) * P.b_pitch + col);
        aimg[i] = wave + 16 * (i & 1) + 8 * (i >> 1);
        const int64_t m = m0 + 8 * aimg[i] + lr;
        aoff[i] = (uint32_t)(((m < P.M ? m : P.M - 1) - m0) * P.a_pitch + col);
    }
    /* loads k of a stage in their order: 0-3 weights, 4-5 tokens' first halves, 6-7 second */
    auto issue = [&](int from, int to, int s, uint8_t* st) __attribute__((always_inline)) {
        const int k = k0 + 128 * s;
        const bool ok = col < kend - k;
#pragma unroll
        for (int i = from; i < to; ++i) {
            if (i < 4) r3d_buf_lds<16>(rB, st + 1024 * wimg[i], ok ? woff[i] : 0x80000000u, k);
            else r3d_buf_lds<16>(rA, st + AOFF + 1024 * aimg[i - 4], ok ? aoff[i - 4] : 0x80000000u, k);
        }
    };

    typename T::Acc16 acc[2][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0;
    r3d_i32x4 wf[2][4], xf[2][4];
    /* operand piece p (16 bytes of K) of 32 rows: lane (row lj, half lh) takes piece 2 p + lh of the
     * step's eight -- image half (2 p + lh) / 4, piece (2 p + lh) % 4 */
    int rd[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) rd[p] = 128 * lj + 16 * ((2 * p + lh) ^ (lj & 7));
    auto read_w = [&](const uint8_t* st, int a, int p) __attribute__((always_inline)) {
        wf[a][p] = *reinterpret_cast<const r3d_i32x4*>(st + 4096 * (2 * wn + a) + rd[p]);
    };
    auto read_x = [&](const uint8_t* st, int b, int p) __attribute__((always_inline)) {
        xf[b & 1][p] = *reinterpret_cast<const r3d_i32x4*>(st + AOFF + 4096 * (4 * wm + b) + rd[p]);
    };
    auto step = [&](int s, uint8_t* cur, uint8_t* nxt) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    acc[a][b] = T::mfma32(wf[a][p], xf[b & 1][p], acc[a][b]);
                    if (b == 3) read_w(nxt, a, p);
                }
                __builtin_amdgcn_s_setprio(0);
                if (b == 0) {
                    if (p == 1) {
                        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                        read_x(cur, 2, 0);
                        read_x(cur, 2, 1);
                    }
                    if (p > 1) {
                        read_x(cur, 2, p);
                        issue(p - 2, p - 1, s + 2, cur);
                    }
                } else if (b == 1) {
                    read_x(cur, 3, p);
                    issue(2 + p, 3 + p, s + 2, cur);
                } else if (b == 2) {
                    if (p == 1) {
                        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                        read_x(nxt, 0, 0);
                        read_x(nxt, 0, 1);
                    }
                    if (p > 1) {
                        read_x(nxt, 0, p);
                        issue(4 + p, 5 + p, s + 2, cur);
                    }
                } else {
                    read_x(nxt, 1, p);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    uint8_t* const r0 = smem;
    uint8_t* const r1 = smem + STAGE;
    issue(0, 8, 0, r0);
    issue(0, 6, 1, r1);
    asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");    /* stage 0's weights, first halves */
    issue(6, 8, 1, r1);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int p = 0; p < 4; ++p) read_w(r0, a, p);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        read_x(r0, 0, p);
        read_x(r0, 1, p);
    }
    int s = 0;
    for (; s + 2 <= steps; s += 2) {
        step(s, r0, r1);
        step(s + 1, r1, r0);
    }
    if (s < steps) step(s, r0, r1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    /* lane l's element i of a 32 x 32 result is weight row 8 (i / 4) + 4 (l / 32) + i % 4, token l % 32 */
    if (P.kc > 1) {
        typedef typename T::Sum Sum;
        Sum* const part = reinterpret_cast<Sum*>(P.part) + (int64_t)kci * P.M * P.N;
        typedef Sum sumx4_u4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int64_t m = m0 + 128 * wm + 32 * b + lj;
            if (m >= P.M) continue;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int64_t n = n0 + 64 * wn + 32 * a + 8 * g + 4 * lh;
                    if (n + 4 <= P.N) {
                        *reinterpret_cast<sumx4_u4*>(part + m * P.N + n) =
                            sumx4_u4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n + i < P.N) part[m * P.N + n + i] = acc[a][b][4 * g + i];
                    }
                }
        }
        return;
    }
    if constexpr (T::kEpi) {
        /* half the tokens at a time: the sums of all would take 256 KB */
        static_assert(128 * epi_row(BN) <= i8_tile_lds(BN, BM, 2), "the sums in the ring's place");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            __syncthreads();                                    /* the ring, or the half before, is read */
#pragma unroll
            for (int b2 = 0; b2 < 2; ++b2)
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const typename T::Acc16& v = acc[a][2 * h + b2];
                        *reinterpret_cast<typename T::Acc4*>(smem + (64 * wm + 32 * b2 + lj) * epi_row(BN) +
                                                             4 * (64 * wn + 32 * a + 8 * g + 4 * lh)) =
                            typename T::Acc4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                    }
            __syncthreads();
            epi_tile<T, BN, 512, 64>(P, smem, m0 + 64 * h, n0);
            epi_tile<T, BN, 512, 64>(P, smem + 64 * epi_row(BN), m0 + 128 + 64 * h, n0);
        }
        return;
    }
    constexpr int YP = 2 * BN + 32, CPR = BN / 8;
    __syncthreads();
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int nl = 64 * wn + 32 * a + 8 * g + 4 * lh;
            float sb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t n = n0 + nl + i;
                sb[i] = P.SB[(n < P.N ? n : P.N - 1) * P.sb_stride];
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int ml = 128 * wm + 32 * b + lj;
                const int64_t m = m0 + ml;
                const float sa = P.SA[(m < P.M ? m : P.M - 1) * P.sa_stride];
                *reinterpret_cast<uint2*>(smem + ml * YP + 2 * nl) = make_uint2(
                    r3d_pack_bf16x2(i8_out(acc[a][b][4 * g], sa, sb[0]), i8_out(acc[a][b][4 * g + 1], sa, sb[1])),
                    r3d_pack_bf16x2(i8_out(acc[a][b][4 * g + 2], sa, sb[2]), i8_out(acc[a][b][4 * g + 3], sa, sb[3])));
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < BM * CPR; e += 512) {
        const int r = e / CPR, cc = e - r * CPR;
        const int64_t m = m0 + r, n = n0 + 8 * cc;
        if (m >= P.M || n >= P.N) continue;
        const r3d_i32x4 v = *reinterpret_cast<const r3d_i32x4*>(smem + r * YP + 16 * cc);
        uint16_t* yp = P.Y + m * P.y_pitch + n;
        if (n + 8 <= P.N) {
            *reinterpret_cast<r3d_i32x4_u2*>(yp) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n + i < P.N) yp[i] = (uint16_t)((uint32_t)v[i >> 1] >> (16 * (i & 1)));
        }
    }
}

}  // namespace r3d

#endif /* R3D_I8_WIDE_H */
