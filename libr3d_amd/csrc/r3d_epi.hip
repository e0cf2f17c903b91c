/* r3d_epi.hip -- entries of gemm_nt_epi's rows (bf16 and i8a8), behind the same launch signature as every row.
 * The plan (r3d_epi_plan.cpp), the gfx950 chip gate, then kernels on the caller's stream.  No allocation, no
 * synchronisation, no host<->device traffic.
 *
 * Measured on MI355X (a 1 GiB copy 5.05 TB/s; the library's largest products 1.61 PFLOP/s bf16, 2.40 POP/s int8), bias in
 * all but the second: 4 x 128 x 5376 bf16 5.8 us, a launch and one chain of loads; 1 x 5376 x 4096 int8 with residual 6.6; 13 x
 * 21504 x 5376 bf16, gelu_tanh 40.3, 5.75 TB/s, bound by the weights; 333 x 8187 x 5360 bf16 45, the tile's own rate; 2048 x
 * 21504 x 5376 int8, gelu_tanh 250 to 255, of which the epilogue's VALU some 30. */
#include <hip/hip_runtime.h>

#include <stdio.h>
#include <string.h>

#include "r3d_dump.h"
#include "r3d_epi.h"
#include "r3d_epi_ops.h"
#include "r3d_i8_launch.h"

namespace r3d {

template <class T>
static int epi_launch(const EpiPlan& P, const I8Geom& g, void* scratch, hipStream_t stream) {
    const EpiArgs e{P.bias, P.res, P.bias_stride, P.r_pitch, P.act, P.bias_bf16, P.res_bf16, P.y_bf16};
    const I8Plan& p = P.p;
    if (g.arm == I8_GEMV) return i8_launch_gemv<T>(p, g, &e, stream);
    int rc = RAD_OK;
    if (g.arm == I8_TILE) rc = i8_launch_tile<T>(p, g, scratch, &e, stream);
    if (rc != RAD_OK || (g.arm == I8_TILE && g.kc == 1)) return rc;
    EpiTileArgs k{};
    static_cast<I8TileArgs&>(k) = I8TileArgs{p.A, p.B, p.SA, p.SB, p.Y, scratch, (int)p.M, (int)p.N, (int)p.K,
                                             (int)p.a_pitch, (int)p.b_pitch, 0, 0, g.kc, 0, p.sa_stride,
                                             p.sb_stride, p.y_pitch};
    k.e = e;
    if (g.arm == I8_TILE) {
        hipLaunchKernelGGL(epi_join_kernel<T>, dim3((unsigned)((p.N + 255) / 256), (unsigned)p.M), dim3(64), 0, stream, k);
    } else {
        const int tm = p.M <= 16 ? 1 : 2;
        const int64_t gy = (p.M + 16 * tm - 1) / (16 * tm);
        if (gy > 65535) return RAD_E_UNSUPPORTED;
        const dim3 grid((unsigned)((p.N + 127) / 128), (unsigned)gy), block(256);
        if (tm == 1) hipLaunchKernelGGL((epi_any_kernel<T, 1>), grid, block, 0, stream, k);
        else hipLaunchKernelGGL((epi_any_kernel<T, 2>), grid, block, 0, stream, k);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? RAD_OK : i8_failed("gemm_nt_epi", err);
}

/* Scratch is optional: without it, or with less than the hook asks for or off 16 bytes, K stays in
 * as few chunks as its planes fit. */
static int epi_entry(const RadArgs* a, RadStream s, bool bf16) {
    if (env_no_epi()) return RAD_E_UNSUPPORTED;
    EpiPlan P{};
    const int rc = plan_epi(a, bf16, &P);
    if (rc) return rc;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    const bool sc = a->scratch && ((uintptr_t)a->scratch & 15) == 0;
    I8Geom g;
    i8_geom(P.p, cu_count(), sc ? a->scratch_bytes : 0, &g);
    return bf16 ? epi_launch<EpiBf16>(P, g, a->scratch, (hipStream_t)s)
                : epi_launch<EpiI8>(P, g, a->scratch, (hipStream_t)s);
}

}  // namespace r3d

extern "C" {

int r3d_rad_gemm_nt_epi_bf16(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("gemm_nt_epi_bf16", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::epi_entry(x, t, true);
    });
}
int r3d_rad_gemm_nt_epi_i8(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("gemm_nt_epi_i8a8", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::epi_entry(x, t, false);
    });
}
int64_t r3d_rad_gemm_nt_epi_bf16_scratch(const RadArgs* a) {
    return r3d::epi_scratch_bytes(a, true, r3d::cu_count());
}
int64_t r3d_rad_gemm_nt_epi_i8_scratch(const RadArgs* a) {
    return r3d::epi_scratch_bytes(a, false, r3d::cu_count());
}

}  /* extern "C" */
