/* r3d_i8_launch.h -- launches of the product kernels that gemm_nt_q at i8a8 and gemm_nt_epi share. */
#ifndef R3D_I8_LAUNCH_H
#define R3D_I8_LAUNCH_H

#include <hip/hip_runtime.h>

#include <stdio.h>

#include "r3d_i8.h"
#include "r3d_i8_gemv.h"
#include "r3d_i8_tile.h"
#include "r3d_i8_wide.h"

namespace r3d {

bool chip_ok();                  /* r3d_gemm.hip */
int cu_count();

inline int i8_failed(const char* what, hipError_t e) {
    fprintf(stderr, "libr3d_gfx950: %s launch FAILED (%s)\n", what, hipGetErrorName(e));
    return RAD_E_DEVICE;
}

template <class T>
inline int i8_launch_gemv(const I8Plan& P, const I8Geom& g, const EpiArgs* epi, hipStream_t stream) {
    int64_t lds = P.M * i8_gemv_row(P.K);
    if (g.kc > 1 && lds < (int64_t)g.waves * 256) lds = g.waves * 256;    /* the chunks' join */
    if (P.M < 1 || P.M > 8 || lds > kI8GemvLds || g.kc < 1 || g.waves % g.kc ||
        g.blocks > 0x7FFFFFFF || (int64_t)g.kc * g.per * 128 < P.K)
        return RAD_E_UNSUPPORTED;
    typename T::GemvArgs a{};
    static_cast<I8GemvArgs&>(a) = I8GemvArgs{P.A, P.B, P.SA, P.SB, P.Y, (int)P.M, (int)P.N, (int)P.K, (int)P.a_pitch,
                       (int)P.b_pitch, g.kc, g.per, P.sa_stride, P.sb_stride, P.y_pitch};
    if constexpr (T::kEpi) a.e = *epi;
    const dim3 grid((unsigned)g.blocks), block((unsigned)(64 * g.waves));
    if (g.waves == 4)
        hipLaunchKernelGGL((i8_gemv_kernel<T, 4>), grid, block, (size_t)lds, stream, a);
    else if (g.waves == 8)
        hipLaunchKernelGGL((i8_gemv_kernel<T, 8>), grid, block, (size_t)lds, stream, a);
    else
        return RAD_E_UNSUPPORTED;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("GEMV", e);
}

/* The tiles; with kc > 1 their planes go to `part`, and the caller adds them up. */
template <class T>
inline int i8_launch_tile(const I8Plan& P, const I8Geom& g, void* part, const EpiArgs* epi, hipStream_t stream) {
    if (g.blocks > 0x7FFFFFFF || (int64_t)g.kc * g.per * 128 < P.K || (g.kc > 1 && !part) ||
        (g.kc > 1 && P.M > 65535))
        return RAD_E_UNSUPPORTED;
    typename T::TileArgs a{};
    static_cast<I8TileArgs&>(a) = I8TileArgs{P.A, P.B, P.SA, P.SB, P.Y, part, (int)P.M, (int)P.N, (int)P.K, (int)P.a_pitch,
                       (int)P.b_pitch, (int)((P.M + g.bm - 1) / g.bm), (int)g.tiles, g.kc, g.per,
                       P.sa_stride, P.sb_stride, P.y_pitch};
    if constexpr (T::kEpi) a.e = *epi;
    const dim3 grid((unsigned)g.blocks);
#define R3D_I8T(WNF_, WMF_, WVN_, WVM_, NST_, OFF_, ONCE_)                                    \
    hipLaunchKernelGGL((i8_tile_kernel<T, WNF_, WMF_, WVN_, WVM_, NST_, OFF_, ONCE_>), grid,       \
                       dim3(64 * WVN_ * WVM_),                                                 \
                       (size_t)i8_tile_lds(16 * WNF_ * WVN_, 16 * WMF_ * WVM_, NST_), stream, a)
#define R3D_I8T2(WNF_, WMF_, WVN_, WVM_, NST_, ONST_)                                         \
    if (P.off) { R3D_I8T(WNF_, WMF_, WVN_, WVM_, ONST_, true, false); }                         \
    else { R3D_I8T(WNF_, WMF_, WVN_, WVM_, NST_, false, false); }                               \
    break
    /* gemm_nt_epi where one tile of tokens is all: nobody else asks for a tile's weights, and loads that the caches do not
     * keep stream faster (ONCE; four layers' weights by turns, 21504 x 5376 bf16: M = 13 45.3 -> 40.3 us, 64 53.1 -> 49.4,
     * 128 65.2 -> 61.7; i8a8 13 23.8 -> 21.3).  One layer's alone, again and again, stay in the 256 MB behind HBM without
     * it (M = 13 34.8 us for 38.6), which no model's do.  Where tiles of tokens share the weights it loses: M = 333 105 ->
     * 121 us.  Tiles of 192 and 256 tokens keep theirs: with one of them no time moved but that of 200 tokens, bf16 (77 us, 67). */
#define R3D_I8T3(WNF_, WMF_, WVN_, WVM_, NST_, ONST_)                                         \
    if (T::kEpi && a.grid_m == 1) {                                                             \
        if (P.off) { R3D_I8T(WNF_, WMF_, WVN_, WVM_, ONST_, true, T::kEpi); }                   \
        else { R3D_I8T(WNF_, WMF_, WVN_, WVM_, NST_, false, T::kEpi); }                         \
        break;                                                                                  \
    }                                                                                           \
    R3D_I8T2(WNF_, WMF_, WVN_, WVM_, NST_, ONST_)
    switch (g.tile) {
        case I8_T_256x256:
            hipLaunchKernelGGL(i8_wide_kernel<T>, grid, dim3(512), (size_t)i8_tile_lds(256, 256, 2), stream, a);
            break;
        case I8_T_128x256: R3D_I8T(4, 4, 2, 4, 3, false, false); break;
        case I8_T_128x192: R3D_I8T(2, 6, 4, 2, 3, false, false); break;
        case I8_T_128x128: R3D_I8T3(2, 4, 4, 2, 4, 5);
        case I8_T_128x96: R3D_I8T3(2, 6, 4, 1, 4, 5);
        case I8_T_128x64: R3D_I8T3(2, 4, 4, 1, 4, 5);
        case I8_T_64x64: R3D_I8T3(1, 4, 4, 1, 4, 5);
        case I8_T_64x32: R3D_I8T3(1, 2, 4, 1, 6, 6);
        case I8_T_32x32: R3D_I8T3(1, 2, 2, 1, 10, 10);
        default: R3D_I8T3(1, 1, 2, 1, 8, 8);
    }
#undef R3D_I8T3
#undef R3D_I8T2
#undef R3D_I8T
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("GEMM tiles", e);
}

}  // namespace r3d

#endif /* R3D_I8_LAUNCH_H */
