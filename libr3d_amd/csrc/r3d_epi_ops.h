/* r3d_epi_ops.h -- gemm_nt_epi on the int8 product's kernels (r3d_i8_gemv.h, r3d_i8_tile.h, r3d_i8_wide.h): bf16
 * operands move through them in the same 16-byte pieces, v_mfma_f32_16x16x32_bf16 and _32x32x16_bf16 in place of
 * the int8 instructions of twice the K (the same bytes a lane, the same cycles), and the epilogue of
 * r3d_epi_dev.h in place of the scales alone.  Below: the kernel for what 16-byte pieces cannot take, and the sum
 * of a K split's planes. */
#ifndef R3D_EPI_OPS_H
#define R3D_EPI_OPS_H

#include "r3d_epi_dev.h"
#include "r3d_i8_any.h"
#include "r3d_i8_gemv.h"
#include "r3d_i8_tile.h"
#include "r3d_i8_wide.h"

namespace r3d {

struct EpiGemvArgs : I8GemvArgs {
    EpiArgs e;
};
struct EpiTileArgs : I8TileArgs {
    EpiArgs e;
};

struct EpiI8 : I8Ops {
    typedef EpiGemvArgs GemvArgs;
    typedef EpiTileArgs TileArgs;
    static constexpr bool kEpi = true;
};

typedef float r3d_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 r3d_bf16x8 __attribute__((ext_vector_type(8)));

struct EpiBf16 {
    typedef float Sum;
    typedef r3d_f32x4 Acc4;
    typedef r3d_f32x16 Acc16;
    typedef EpiGemvArgs GemvArgs;
    typedef EpiTileArgs TileArgs;
    static constexpr bool kScaled = false;
    static constexpr bool kZeroBoth = true;     /* 0 * inf */
    static constexpr bool kEpi = true;
    static __device__ __forceinline__ Acc4 mfma16(r3d_i32x4 w, r3d_i32x4 x, Acc4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(r3d_bf16x8, w),
                                                       __builtin_bit_cast(r3d_bf16x8, x), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Acc16 mfma32(r3d_i32x4 w, r3d_i32x4 x, Acc16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(r3d_bf16x8, w),
                                                       __builtin_bit_cast(r3d_bf16x8, x), c, 0, 0, 0);
    }
};

/* Any K, base and pitch: i8_any_kernel's walk (r3d_i8_any.h), with the bytes past K set to zero on both sides
 * and a wave's 32 columns of each token through its own part of LDS, so that a lane finishes eight of them. */
template <class T, int TM>
__global__ __launch_bounds__(256) void epi_any_kernel(EpiTileArgs P) {
    constexpr int ROW = epi_row(32);
    __shared__ __attribute__((aligned(16))) uint8_t s_sum[4 * 16 * TM * ROW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 128 + 32 * wave;
    const int64_t m0 = (int64_t)blockIdx.y * 16 * TM;
    if (n0 >= P.N) return;                              /* whole wave: no barrier follows */
    AnyBuf bw[2], ba[TM];
    uint32_t ow[2], oa[TM];
    bool iw[2], ia[TM];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int64_t n = n0 + 16 * f;
        const int rows = P.N - n < 16 ? (int)(P.N > n ? P.N - n : 0) : 16;
        bw[f] = any_buf(P.B + (rows ? n : 0) * P.b_pitch, rows ? (int64_t)(rows - 1) * P.b_pitch + P.K : 0);
        ow[f] = (uint32_t)(r16 * P.b_pitch);
        iw[f] = r16 < rows;
    }
#pragma unroll
    for (int f = 0; f < TM; ++f) {
        const int64_t m = m0 + 16 * f;
        const int rows = P.M - m < 16 ? (int)(P.M > m ? P.M - m : 0) : 16;
        ba[f] = any_buf(P.A + (rows ? m : 0) * P.a_pitch, rows ? (int64_t)(rows - 1) * P.a_pitch + P.K : 0);
        oa[f] = (uint32_t)(r16 * P.a_pitch);
        ia[f] = r16 < rows;
    }
    typename T::Acc4 acc[2][TM];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[f][t] = typename T::Acc4{0, 0, 0, 0};
    for (int k0 = 0; k0 < P.K; k0 += 64) {
        const int k = k0 + 16 * q;
        r3d_i32x4 w[2], x[TM];
#pragma unroll
        for (int f = 0; f < 2; ++f)
            w[f] = i8_keep(any_ld16(bw[f], iw[f] && k < P.K ? ow[f] + k : kAnyOob, false), P.K - k);
#pragma unroll
        for (int t = 0; t < TM; ++t)
            x[t] = i8_keep(any_ld16(ba[t], ia[t] && k < P.K ? oa[t] + k : kAnyOob, false), P.K - k);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < TM; ++t) acc[f][t] = T::mfma16(w[f], x[t], acc[f][t]);
    }
    uint8_t* const s = s_sum + wave * 16 * TM * ROW;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < TM; ++t)
            *reinterpret_cast<typename T::Acc4*>(s + (16 * t + r16) * ROW + 4 * (16 * f + 4 * q)) = acc[f][t];
    /* the wave's own: its LDS accesses happen in order, and the compiler keeps theirs */
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int cc = lane & 3;
    const int64_t n = n0 + 8 * cc;
    if (n >= P.N) return;
    float sb[8];
    if (T::kScaled) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sb[i] = P.SB[(n + i < P.N ? n + i : P.N - 1) * P.sb_stride];
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int64_t m = m0 + 16 * t + (lane >> 2);
        if (m >= P.M) continue;
        const typename T::Acc4* p = reinterpret_cast<const typename T::Acc4*>(s + (16 * t + (lane >> 2)) * ROW + 32 * cc);
        const typename T::Acc4 lo = p[0], hi = p[1];
        const float sa = T::kScaled ? P.SA[m * P.sa_stride] : 1.0f;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = (float)(i < 4 ? lo[i & 3] : hi[i & 3]);
            v[i] = T::kScaled ? f * sa * sb[i] : f;
        }
        epi_values<8>(P.e, v, m, n, P.N);
        epi_store<8>(P.e, P.Y, P.y_pitch, v, m, n, P.N);
    }
}

/* Y of kc planes, added in their order: four columns a lane, (ceil(N / 256), M) workgroups of 64. */
template <class T>
__global__ __launch_bounds__(64) void epi_join_kernel(EpiTileArgs P) {
    const int64_t n = 4 * ((int64_t)blockIdx.x * 64 + threadIdx.x), m = blockIdx.y;
    if (n >= P.N) return;
    typedef typename T::Sum Sum;
    typedef Sum sumx4_u4 __attribute__((ext_vector_type(4), aligned(4)));
    const int64_t plane = (int64_t)P.M * P.N;
    const Sum* p = static_cast<const Sum*>(P.part) + m * P.N + n;
    typename T::Acc4 sum = {0, 0, 0, 0};
    if (n + 4 <= P.N) {
#pragma unroll 4
        for (int c = 0; c < P.kc; ++c) sum += *reinterpret_cast<const sumx4_u4*>(p + c * plane);
    } else {
        for (int c = 0; c < P.kc; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < P.N) sum[i] += p[c * plane + i];
    }
    const float sa = T::kScaled ? P.SA[m * P.sa_stride] : 1.0f;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = T::kScaled ? (float)sum[i] * sa * P.SB[(n + i < P.N ? n + i : P.N - 1) * P.sb_stride] : (float)sum[i];
    epi_values<4>(P.e, v, m, n, P.N);
    epi_store<4>(P.e, P.Y, P.y_pitch, v, m, n, P.N);
}

}  // namespace r3d

#endif /* R3D_EPI_OPS_H */
