/* r3d_i8.h -- host-side plans of the int8 rows: gemm_nt_q at i8a8 and the three producers
 * of its activations (quant_act_i8, gated_quant_i8, rmsnorm_quant_i8).  Pure host C++, so
 * every refusal and every choice of kernel is testable without a GPU.
 *
 * The int8 linear layer: codes with one f32 scale a token (A) and one f32 scale an output
 * channel (B),
 *     Y[m, n] = bf16((f32(sum_k A[m, k] B[n, k]) * a_scale[m]) * b_scale[n]),
 * the sum exact in i32.
 */
#ifndef R3D_I8_H
#define R3D_I8_H

#include <stdint.h>
#include "rad_abi.h"

namespace r3d {

/* |sum| <= 2^14 K stays below 2^31 for any codes (-128 among them) */
constexpr int64_t kI8MaxK = 131071;

struct I8Plan {
    const uint8_t* A;        /* int8 [M, K] */
    const float*   SA;       /* f32, one a token, sa_stride elements apart */
    const uint8_t* B;        /* int8 [N, K] */
    const float*   SB;       /* f32, one a weight row, sb_stride elements apart */
    uint16_t*      Y;        /* bf16 [M, N] */
    int64_t M, N, K;
    int64_t a_pitch, b_pitch, y_pitch, sa_stride, sb_stride;
    int ua;                  /* K, a base or a pitch off 16 bytes: the any-alignment kernel */
    int off;                 /* a base or a pitch off 128: rows begin inside lines */
};

/* The operands and params of a gemm_nt_q call at i8a8; m_max: the row's bound on M (0: none). */
int plan_i8(const RadArgs* a, int64_t m_max, I8Plan* P);

/* Which kernel a call takes, and its launch. */
enum { I8_ANY = 0, I8_GEMV = 1, I8_TILE = 2 };
enum {
    I8_T_256x256, I8_T_128x256, I8_T_128x192, I8_T_128x128, I8_T_128x96, I8_T_128x64, I8_T_64x64,
    I8_T_64x32, I8_T_32x32, I8_T_32x16, I8_TILES
};

struct I8Geom {
    int arm;
    int tile;                /* I8_TILE: one of the above (weight rows x tokens) */
    int bn, bm;
    int64_t tiles;
    int kc;                  /* K chunks: waves of a workgroup (GEMV), or workgroups with an i32
                                plane each in scratch (tiles, kc > 1) */
    int per;                 /* 128-wide K steps a chunk */
    int waves;               /* GEMV: waves a workgroup */
    int64_t blocks;          /* workgroups */
};

/* GEMV: the tokens in LDS, rows this many bytes apart */
constexpr int64_t i8_gemv_row(int64_t K) { return ((K + 127) & ~(int64_t)127) + 16; }
/* and at most this much of it: with 56 KB and more, two workgroups a compute unit, the GEMV takes 1.05 to
 * 1.4 of the tiles' time */
constexpr int64_t kI8GemvLds = 48 * 1024;

/* The launch that suits a shape on ncu compute units, with at most `scratch` bytes for planes. */
void i8_geom(const I8Plan& P, int ncu, int64_t scratch, I8Geom* g);

/* The planes that a call's best launch wants: kc M N 4 bytes, 0 for none (the row's scratch hook).  Operands that
 * are given are planned as the launch plans them. */
int64_t i8_scratch_bytes(const RadArgs* a, int ncu);

/* Codes out of a band producer, one scale a row. */
struct I8BandPlan {
    const uint8_t* x;        /* the activation, or gate_up [rows, 2n] */
    const uint8_t* res;      /* rmsnorm: residual in, or null */
    uint8_t* res_out;        /* rmsnorm: bf16(residual + x), or null */
    const uint8_t* w;        /* rmsnorm: [n] */
    uint8_t* q;
    float* scale;
    uint8_t* ob;             /* the values the codes are of, or null */
    int x_bf16, w_bf16, ob_bf16, silu;
    int64_t rows, n, x_pitch, r_pitch, ro_pitch, q_pitch, s_stride, ob_pitch;
    double eps;
    float wadd;
};
enum { I8_QUANT = 0, I8_GATED = 1, I8_NORM = 2 };
int plan_i8_band(const RadArgs* a, int op, I8BandPlan* P);

/* Lanes of a row's workgroup and 8-element chunks a lane holds in registers; chunks 0: the row
 * is past what registers hold and is walked twice. */
struct I8BandGeom {
    int lanes, chunks;
};
I8BandGeom i8_band_geom(int64_t rows, int64_t n);

/* describe() for this table's rows; -1 when `row` is not one of them. */
int describe_i8(const char* row, const RadArgs* a, char* buf, int len);

bool env_no_i8();
bool env_no_i8_dec();

}  // namespace r3d

#endif /* R3D_I8_H */
