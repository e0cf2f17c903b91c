/* r3d_i8_tile.h -- gemm_nt_q at i8a8 on LDS tiles, for more tokens than the GEMV takes.
 *
 * A workgroup of WVN x WVM waves owns BN = 16 WNF WVN weight rows x BM = 16 WMF WVM tokens; a wave
 * 16 WNF x 16 WMF of them, v_mfma_i32_16x16x64_i8 with the weights as source A, so lane l's result
 * is four consecutive weight rows of one token.  K is walked 128 a step.  A step's operands go
 * straight from memory to LDS (buffer loads, 16 bytes a lane) into a ring of NST stages; each 1 KB
 * load is 8 rows of 128 bytes, so that it asks for whole cache lines (with 16 rows of half a line the
 * loads were the bound), the 16-byte piece of a row at place piece ^ row
 * % 8: an operand read (ds_read_b128) touches every bank group once in any 8 lanes.  Rows past the
 * operands clamp to the last (their results are not stored); columns past K
 * (K % 128 = 16 .. 112) are asked for past the buffer's records and land as zeros.
 *
 * Rows that begin inside lines (a base or a pitch off 128 bytes; both are multiples of 16 here) would take
 * two lines a step each.  OFF loads whole lines all the same: a row's lines lie in the ring as they do in
 * memory, its pieces counted from its own beginning, and a step reads the last of them from the stage
 * after.  That asks for one stage more to have landed (M = 64 x 21504 x 5360 37.4 -> 27.7 us, 128 49.6 -> 33.5,
 * 333 82 -> 58; at K = 5376, where nothing asks for it, 1 to 9 % more).  The tiles of 192 and 256 tokens have no
 * LDS for that stage and take the two lines.
 *
 * One barrier a step: it says both that the next step's stage has landed (each wave has waited for
 * its own loads) and that the stage before this one is read, whose slot then takes the loads of
 * NST - 1 steps ahead.  A wave reads the operands of one half step while the products of the other
 * run.
 *
 * The sum is exact in i32, so K may be cut anywhere: with kc > 1 workgroup u takes K chunk
 * u / tiles of its tile and leaves an i32 plane, and i8_join_kernel adds the planes.
 *
 * Measured on MI355X (a 16384 x 16384 x 8192 product of the library's reaches 2.39 POP/s, a 1 GiB copy 5.14
 * TB/s): M = 13 x 5376 x 21504 23.3 to 24.3 us, 5.0 TB/s, bound by the weights; M = 333 x 8187 x 5360 22.6 to 23.8 us,
 * 1.3 POP/s: 256 tiles of 128 x 96, an eighth of them past the edges.  A step of a 128 x 128 tile takes 0.45 us a
 * compute unit, 9.3 TOP/s of the 9.3 that the library's product leaves each; one of 128 x 96 0.42, 7.5 TOP/s.
 */
#ifndef R3D_I8_TILE_H
#define R3D_I8_TILE_H

#include "r3d_device.h"
#include "r3d_i8_any.h"

namespace r3d {

struct I8TileArgs {
    const uint8_t* A;
    const uint8_t* B;
    const float* SA;
    const float* SB;
    uint16_t* Y;
    int* part;                       /* kc > 1: i32 [kc][M][N] */
    int M, N, K, a_pitch, b_pitch, grid_m, tiles, kc, cst;
    int64_t sa_stride, sb_stride, y_pitch;
};

template <int WNF, int WMF, int WVN, int WVM, int NST, bool OFF>
__global__ __launch_bounds__(64 * WVN * WVM) void i8_tile_kernel(I8TileArgs P) {
    constexpr int WV = WVN * WVM, BN = 16 * WNF * WVN, BM = 16 * WMF * WVM;
    constexpr int WLD = BN / 8 / WV, ALD = BM / 8 / WV, LOADS = WLD + ALD;   /* 1 KB loads a wave */
    static_assert(WLD * WV * 8 == BN && ALD * WV * 8 == BM, "whole loads a wave");
    static_assert(NST >= 3 + OFF, "the stages a step reads, and one to load");
    constexpr int AOFF = BN * 128, STAGE = (BN + BM) * 128;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, q = lane >> 4;
    const int wn = wave % WVN, wm = wave / WVN;

    /* workgroups go round-robin over the 8 XCDs: a contiguous run of units each, tiles in groups
     * of GN weight tiles with the token tile major, so an XCD's L2 sees few panels at a time */
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

    /* (OFF: a row's first line begins before the row; the records begin a line earlier, for offsets from
     * 0 on, and nothing is asked for there) */
    constexpr int LEAD = OFF ? 128 : 0;
    const __amdgpu_buffer_rsrc_t rB =
        r3d_rsrc(P.B + n0 * P.b_pitch - LEAD, (P.N - 1 - n0) * (int64_t)P.b_pitch + P.K + LEAD);
    const __amdgpu_buffer_rsrc_t rA =
        r3d_rsrc(P.A + m0 * P.a_pitch - LEAD, (P.M - 1 - m0) * (int64_t)P.a_pitch + P.K + LEAD);
    /* image j: rows 8 j .. + 7 of 128 bytes, a line a row; lane (row lr, place) fetches the 16-byte
     * piece place ^ lr of the row's own count, which lies `shift` pieces on in its line */
    const int lr = lane >> 3;
    auto shift = [](const uint8_t* base, int pitch, int r) {
        return OFF ? (int)(((uintptr_t)base >> 4) + (uint32_t)r * (uint32_t)(pitch >> 4)) & 7 : 0;
    };
    auto column = [&](int sh) { return 16 * (((((lane & 7) ^ lr) + sh) & 7) - sh); };
    const int wcol = column(shift(P.B, P.b_pitch, lr)), acol = column(shift(P.A, P.a_pitch, lr));
    uint32_t woff[WLD], aoff[ALD];
#pragma unroll
    for (int i = 0; i < WLD; ++i) {
        const int64_t n = n0 + 8 * (wave + WV * i) + lr;
        woff[i] = (uint32_t)(((n < P.N ? n : P.N - 1) - n0) * P.b_pitch + wcol + LEAD);
    }
#pragma unroll
    for (int i = 0; i < ALD; ++i) {
        const int64_t m = m0 + 8 * (wave + WV * i) + lr;
        aoff[i] = (uint32_t)(((m < P.M ? m : P.M - 1) - m0) * P.a_pitch + acol + LEAD);
    }
    auto issue = [&](int s, uint8_t* st) __attribute__((always_inline)) {
        const int k = k0 + 128 * s;
        /* outside the chunk's columns: zeros */
        const bool wok = (uint32_t)(128 * s + wcol) < (uint32_t)(kend - k0);
        const bool aok = (uint32_t)(128 * s + acol) < (uint32_t)(kend - k0);
#pragma unroll
        for (int i = 0; i < WLD; ++i)
            r3d_buf_lds<16>(rB, st + 1024 * (wave + WV * i), wok ? woff[i] : 0x80000000u, k);
#pragma unroll
        for (int i = 0; i < ALD; ++i)
            r3d_buf_lds<16>(rA, st + AOFF + 1024 * (wave + WV * i), aok ? aoff[i] : 0x80000000u, k);
    };

    r3d_i32x4 acc[WNF][WMF];
#pragma unroll
    for (int a = 0; a < WNF; ++a)
#pragma unroll
        for (int b = 0; b < WMF; ++b) acc[a][b] = r3d_i32x4{0, 0, 0, 0};
    const int rd0 = 128 * li + 16 * (q ^ (li & 7)), rd1 = 128 * li + 16 * ((4 + q) ^ (li & 7));
    /* fragments of one half step (64 of K): half 0 and half 1 each have a register set, read while
     * the other half's products run */
    r3d_i32x4 wf[2][WNF], xf[2][WMF];
    /* (OFF: the pieces past the end of the row's line are in the next stage) */
    const int wsh = shift(P.B, P.b_pitch, li) + q, ash = shift(P.A, P.a_pitch, li) + q;
    auto read = [&](int now, int then, int h) __attribute__((always_inline)) {
        const int rd = h ? rd1 : rd0;
        const uint8_t* const sw = smem + STAGE * (OFF && wsh + 4 * h >= 8 ? then : now) + rd;
        const uint8_t* const sx = smem + STAGE * (OFF && ash + 4 * h >= 8 ? then : now) + AOFF + rd;
#pragma unroll
        for (int a = 0; a < WNF; ++a)
            wf[h][a] = *reinterpret_cast<const r3d_i32x4*>(sw + 2048 * (wn * WNF + a));
#pragma unroll
        for (int b = 0; b < WMF; ++b)
            xf[h][b] = *reinterpret_cast<const r3d_i32x4*>(sx + 2048 * (wm * WMF + b));
    };
    auto products = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < WMF; ++b)
#pragma unroll
            for (int a = 0; a < WNF; ++a)
                acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[h][a], xf[h][b], acc[a][b], 0, 0, 0);
        /* a read between every so many products */
        constexpr int PER = WNF * WMF / (WNF + WMF) > 0 ? WNF * WMF / (WNF + WMF) : 1;
#pragma unroll
        for (int i = 0; i < WNF + WMF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(s, smem + STAGE * s);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(LOADS * (NST - 2 - OFF)) : "memory");
    read(0, 1, 0);
    int slot = 0;
    for (int s = 0; s < steps; ++s) {
        const int next = slot + 1 == NST ? 0 : slot + 1, last = slot == 0 ? NST - 1 : slot - 1;
        const int after = next + 1 == NST ? 0 : next + 1;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(LOADS * (NST - 3 - OFF)) : "memory");
        issue(s + NST - 1, smem + STAGE * last);                /* the slot read one step ago */
        read(slot, next, 1);
        products(0);
        read(next, after, 0);
        products(1);
        slot = next;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            /* the loads past the end, before LDS goes */

    if (P.kc > 1) {
        int* const part = P.part + (int64_t)kci * P.M * P.N;
#pragma unroll
        for (int b = 0; b < WMF; ++b) {
            const int64_t m = m0 + 16 * (wm * WMF + b) + li;
            if (m >= P.M) continue;
#pragma unroll
            for (int a = 0; a < WNF; ++a) {
                const int64_t n = n0 + 16 * (wn * WNF + a) + 4 * q;
                typedef int i32x4_u4 __attribute__((ext_vector_type(4), aligned(4)));
                if (n + 4 <= P.N) {
                    *reinterpret_cast<i32x4_u4*>(part + m * P.N + n) = acc[a][b];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < P.N) part[m * P.N + n + i] = acc[a][b][i];
                }
            }
        }
        return;
    }
    /* the bf16 tile through LDS, a token's row 32 bytes off a multiple of 128, then 16 bytes a lane */
    constexpr int YP = 2 * BN + 32, CPR = BN / 8;
    float sb[WNF][4];
#pragma unroll
    for (int a = 0; a < WNF; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + 16 * (wn * WNF + a) + 4 * q + i;
            sb[a][i] = P.SB[(n < P.N ? n : P.N - 1) * P.sb_stride];
        }
    __syncthreads();                                            /* every wave is done with the ring */
#pragma unroll
    for (int b = 0; b < WMF; ++b) {
        const int ml = 16 * (wm * WMF + b) + li;
        const int64_t m = m0 + ml;
        const float sa = P.SA[(m < P.M ? m : P.M - 1) * P.sa_stride];
#pragma unroll
        for (int a = 0; a < WNF; ++a) {
            const r3d_i32x4 v = acc[a][b];
            *reinterpret_cast<uint2*>(smem + ml * YP + 2 * (16 * (wn * WNF + a) + 4 * q)) =
                make_uint2(r3d_pack_bf16x2(i8_out(v[0], sa, sb[a][0]), i8_out(v[1], sa, sb[a][1])),
                           r3d_pack_bf16x2(i8_out(v[2], sa, sb[a][2]), i8_out(v[3], sa, sb[a][3])));
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < BM * CPR; e += 64 * WV) {
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

constexpr int i8_tile_lds(int bn, int bm, int nst) {
    const int ring = nst * (bn + bm) * 128, out = bm * (2 * bn + 32);
    return ring > out ? ring : out;
}

/* Y of kc i32 planes: four columns a lane, (ceil(N / 256) , M) workgroups of 64. */
__global__ __launch_bounds__(64) void i8_join_kernel(const int* __restrict__ part, const float* __restrict__ SA,
                                                     const float* __restrict__ SB, uint16_t* __restrict__ Y,
                                                     int kc, int M, int N, int64_t sa_stride,
                                                     int64_t sb_stride, int64_t y_pitch) {
    const int64_t n = 4 * ((int64_t)blockIdx.x * 64 + threadIdx.x), m = blockIdx.y;
    if (n >= N) return;
    const float sa = SA[m * sa_stride];
    const int64_t plane = (int64_t)M * N;
    const int* p = part + m * N + n;
    uint16_t* y = Y + m * y_pitch + n;
    if (n + 4 <= N) {
        typedef int i32x4_u4 __attribute__((ext_vector_type(4), aligned(4)));
        r3d_i32x4 v = *reinterpret_cast<const i32x4_u4*>(p);
#pragma unroll 4
        for (int c = 1; c < kc; ++c) v += *reinterpret_cast<const i32x4_u4*>(p + c * plane);
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = i8_out(v[i], sa, SB[(n + i) * sb_stride]);
        *reinterpret_cast<r3d_u32x2_u2*>(y) = r3d_u32x2_u2{r3d_pack_bf16x2(f[0], f[1]), r3d_pack_bf16x2(f[2], f[3])};
    } else {
        for (int i = 0; n + i < N; ++i) {
            int v = 0;
            for (int c = 0; c < kc; ++c) v += p[c * plane + i];
            y[i] = r3d_bf16_rne(i8_out(v, sa, SB[(n + i) * sb_stride]));
        }
    }
}

}  // namespace r3d

#endif /* R3D_I8_TILE_H */
