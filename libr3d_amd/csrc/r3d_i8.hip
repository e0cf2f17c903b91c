/* r3d_i8.hip -- entries of the int8 rows: gemm_nt_q at i8a8 (decode band and any M) and the
 * producers of its activations, behind the same launch signature as every row
 *     int launch(const RadArgs* a, RadStream s)
 * The plan (r3d_i8_plan.cpp), the gfx950 chip gate, then kernels on the caller's stream.  No
 * allocation, no synchronisation, no host<->device traffic in any entry. */
#include <hip/hip_runtime.h>

#include <stdio.h>
#include <string.h>

#include "r3d_dump.h"
#include "r3d_i8.h"
#include "r3d_i8_any.h"
#include "r3d_i8_band.h"
#include "r3d_i8_launch.h"
#include "r3d_plan.h"

namespace r3d {

static int i8_launch_any(const I8Plan& P, hipStream_t stream) {
    const int tm = P.M <= 16 ? 1 : 2;
    const int64_t gx = (P.N + 127) / 128, gy = (P.M + 16 * tm - 1) / (16 * tm);
    if (gy > 65535) return RAD_E_UNSUPPORTED;
    const dim3 grid((unsigned)gx, (unsigned)gy), block(256);
#define R3D_I8_ANY(TM_)                                                                       \
    hipLaunchKernelGGL((i8_any_kernel<TM_>), grid, block, 0, stream, P.A, P.SA, P.B, P.SB, P.Y, \
                       (int)P.M, (int)P.N, (int)P.K, P.a_pitch, P.b_pitch, P.y_pitch,          \
                       P.sa_stride, P.sb_stride)
    if (tm == 1) R3D_I8_ANY(1); else R3D_I8_ANY(2);
#undef R3D_I8_ANY
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("i8a8 any-alignment GEMM", e);
}

/* Scratch is optional: without it, or with less than the hook asks for or off 16 bytes, K stays in
 * as few chunks as its planes fit. */
static int i8_entry(const RadArgs* a, RadStream s, bool decode) {
    if (env_no_i8() || (decode && env_no_i8_dec())) return RAD_E_UNSUPPORTED;
    I8Plan P{};
    const int rc = plan_i8(a, decode ? 16 : 0, &P);
    if (rc) return rc;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    const bool sc = a->scratch && ((uintptr_t)a->scratch & 15) == 0;
    I8Geom g;
    i8_geom(P, cu_count(), sc ? a->scratch_bytes : 0, &g);
    hipStream_t stream = (hipStream_t)s;
    if (g.arm == I8_GEMV) return i8_launch_gemv<I8Ops>(P, g, nullptr, stream);
    if (g.arm != I8_TILE) return i8_launch_any(P, stream);
    const int lrc = i8_launch_tile<I8Ops>(P, g, a->scratch, nullptr, stream);
    if (lrc != RAD_OK || g.kc == 1) return lrc;
    hipLaunchKernelGGL(i8_join_kernel, dim3((unsigned)((P.N + 255) / 256), (unsigned)P.M), dim3(64), 0,
                       stream, (const int*)a->scratch, P.SA, P.SB, P.Y, g.kc, (int)P.M, (int)P.N, P.sa_stride,
                       P.sb_stride, P.y_pitch);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("i8a8 GEMM", e);
}

static int i8_band_entry(const RadArgs* a, RadStream s, int op) {
    if (env_no_i8()) return RAD_E_UNSUPPORTED;
    I8BandPlan P{};
    const int rc = plan_i8_band(a, op, &P);
    if (rc) return rc;
    if (!chip_ok()) return RAD_E_UNSUPPORTED;
    const I8BandGeom g = i8_band_geom(P.rows, P.n);
    const I8BandArgs k{P.x, (const uint16_t*)P.res, (uint16_t*)P.res_out, P.w, P.q, P.scale, P.ob,
                       P.n, P.x_pitch, P.r_pitch, P.ro_pitch, P.q_pitch, P.s_stride, P.ob_pitch,
                       P.eps, P.wadd, P.silu, P.ob_bf16};
    const dim3 grid((unsigned)P.rows), block((unsigned)g.lanes);
    hipStream_t stream = (hipStream_t)s;
#define R3D_I8B(OP_, X_, W_)                                                                  \
    switch (g.chunks) {                                                                       \
        case 1: hipLaunchKernelGGL((i8_band_kernel<OP_, X_, W_, 1>), grid, block, 0, stream, k); break; \
        case 2: hipLaunchKernelGGL((i8_band_kernel<OP_, X_, W_, 2>), grid, block, 0, stream, k); break; \
        case 3: hipLaunchKernelGGL((i8_band_kernel<OP_, X_, W_, 3>), grid, block, 0, stream, k); break; \
        case 4: hipLaunchKernelGGL((i8_band_kernel<OP_, X_, W_, 4>), grid, block, 0, stream, k); break; \
        default: hipLaunchKernelGGL((i8_band_kernel<OP_, X_, W_, 0>), grid, block, 0, stream, k); break; \
    }
    if (op == I8_NORM) {
        if (P.w_bf16) { R3D_I8B(I8_NORM, true, true) } else { R3D_I8B(I8_NORM, true, false) }
    } else if (op == I8_GATED) {
        if (P.x_bf16) { R3D_I8B(I8_GATED, true, true) } else { R3D_I8B(I8_GATED, false, true) }
    } else {
        if (P.x_bf16) { R3D_I8B(I8_QUANT, true, true) } else { R3D_I8B(I8_QUANT, false, true) }
    }
#undef R3D_I8B
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RAD_OK : i8_failed("int8 producer", e);
}

}  // namespace r3d

extern "C" {

int r3d_rad_gemm_nt_q_i8(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("gemm_nt_q_i8a8", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::i8_entry(x, t, false);
    });
}
int64_t r3d_rad_gemm_nt_q_i8_scratch(const RadArgs* a) {
    return r3d::i8_scratch_bytes(a, r3d::cu_count());
}
int r3d_rad_gemm_nt_q_i8_decode(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("gemm_nt_q_i8a8_decode", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::i8_entry(x, t, true);
    });
}
int r3d_rad_quant_act_i8(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("quant_act_i8", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::i8_band_entry(x, t, r3d::I8_QUANT);
    });
}
int r3d_rad_gated_quant_i8(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("gated_quant_i8", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::i8_band_entry(x, t, r3d::I8_GATED);
    });
}
int r3d_rad_rmsnorm_quant_i8(const RadArgs* a, RadStream s) {
    return r3d::dump_wrap("rmsnorm_quant_i8", a, s, [](const RadArgs* x, RadStream t) {
        return r3d::i8_band_entry(x, t, r3d::I8_NORM);
    });
}

}  /* extern "C" */
