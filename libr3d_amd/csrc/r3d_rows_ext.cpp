/* r3d_rows_ext.cpp -- the library's second row table: ops and encodings past the set that the
 * reference plugin declares.  A radiance loader compares a plugin's schemas with the other
 * declarers' (src/r3d_rows.cpp:29-37), so rad_kernel_at lists only rows of that set; an engine
 * that knows these ops reads them here, in the same structures, and launches them the same way.
 *
 * Rows (resolver: as in r3d_rows.cpp):
 *   gemm_nt_q_i8a8           prio 1000  dtype IN i8a8                     int8 GEMM, any M
 *   gemm_nt_q_i8a8_decode    prio 1100  + M LE 16                          the same, decode band
 *   quant_act_i8             prio 1000  n GE 1, dtype IN f32 bf16           activation producer
 *   gated_quant_i8           prio 1000  n GE 1, dtype IN f32 bf16           gated producer
 *   rmsnorm_quant_i8         prio 1000  n GE 1, dtype IN bf16               norm producer
 *   sample_logits            prio 1000  n_vocab GE 1, dtype IN f32 bf16     sampler
 *
 * R3D_NO_I8 hides the int8 rows, R3D_NO_I8_DEC the int8 decode row (and turns off its GEMV in the other
 * one, which takes those calls on its tiles), R3D_NO_SAMPLE the sampler (presence-tested, read once; hidden at
 * registration as in r3d_rows.cpp).  gemm_nt_q's schema is rad_kernel_schema_at's. */
#include <stdint.h>
#include <string.h>

#include "rad_abi.h"
#include "r3d_i8.h"
#include "r3d_sample.h"

extern "C" {
int r3d_rad_gemm_nt_q_i8(const RadArgs* a, RadStream s);
int r3d_rad_gemm_nt_q_i8_decode(const RadArgs* a, RadStream s);
int64_t r3d_rad_gemm_nt_q_i8_scratch(const RadArgs* a);
int r3d_rad_quant_act_i8(const RadArgs* a, RadStream s);
int r3d_rad_gated_quant_i8(const RadArgs* a, RadStream s);
int r3d_rad_rmsnorm_quant_i8(const RadArgs* a, RadStream s);
int r3d_rad_sample_logits(const RadArgs* a, RadStream s);
int64_t r3d_rad_sample_logits_scratch(const RadArgs* a);
}

namespace {

const RadParamSpec kQuantParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n", RAD_P_INT, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
};
const RadOperandSpec kQuantOperands[] = {
    {"x", RAD_OPD_IN, 0},
    {"q", RAD_OPD_OUT, 0},
    {"scale", RAD_OPD_OUT, 0},
};
const RadParamSpec kGatedParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n", RAD_P_INT, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
    {"act", RAD_P_STR, RAD_OPTIONAL, 0},
};
const RadOperandSpec kGatedOperands[] = {
    {"gate_up", RAD_OPD_IN, 0},
    {"q", RAD_OPD_OUT, 0},
    {"scale", RAD_OPD_OUT, 0},
    {"out", RAD_OPD_OUT, 1},
};
const RadParamSpec kNormParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n", RAD_P_INT, RAD_REQUIRED, 0},
    {"eps", RAD_P_F64, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
    {"wadd", RAD_P_F64, RAD_OPTIONAL, 0},
};
const RadOperandSpec kNormOperands[] = {
    {"x", RAD_OPD_IN, 0},
    {"residual", RAD_OPD_IN, 1},
    {"w", RAD_OPD_WEIGHT, 0},
    {"q", RAD_OPD_OUT, 0},
    {"scale", RAD_OPD_OUT, 0},
    {"out", RAD_OPD_OUT, 1},
    {"residual_out", RAD_OPD_OUT, 1},
};

const RadParamSpec kSampleParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n_vocab", RAD_P_INT, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
};
const RadOperandSpec kSampleOperands[] = {
    {"logits", RAD_OPD_IN, 0},
    {"u", RAD_OPD_IN, 0},
    {"temperature", RAD_OPD_IN, 1},
    {"top_k", RAD_OPD_IN, 1},
    {"top_p", RAD_OPD_IN, 1},
    {"min_p", RAD_OPD_IN, 1},
    {"token", RAD_OPD_OUT, 0},
    {"prob", RAD_OPD_OUT, 1},
};

const RadOpSchema kSchemas[] = {
    {"quant_act_i8", kQuantParams, 3, kQuantOperands, 3,
     "symmetric int8 quantisation of an activation with one f32 scale a row, amax/127."},
    {"gated_quant_i8", kGatedParams, 4, kGatedOperands, 4,
     "silu(gate)*up or sigmoid(gate)*up in f32 (gate the first n columns of each row, up the "
     "next n), then quant_act_i8's quantiser; out carries the f32 values, or their bf16."},
    {"rmsnorm_quant_i8", kNormParams, 5, kNormOperands, 7,
     "RMS norm, optionally of bf16(residual + x) written to residual_out (which may be residual "
     "or x itself), then quant_act_i8's quantiser over the f32 normed values; out carries them."},
    {"sample_logits", kSampleParams, 3, kSampleOperands, 8,
     "one token a row of logits from a uniform number u in [0, 1): softmax at the row's temperature, "
     "top-k, top-p of those, min-p of those, then the first kept token in index order whose running "
     "mass passes u times the kept mass; prob is its share of that mass."},
};

const RadConstraint cI8[] = {
    {"dtype", RAD_C_IN, 0, "i8a8"},
};
const RadConstraint cI8Decode[] = {
    {"dtype", RAD_C_IN, 0, "i8a8"},
    {"M", RAD_C_LE, 16, nullptr},
};
const RadConstraint cBand[] = {
    {"n", RAD_C_GE, 1, nullptr},
    {"dtype", RAD_C_IN, 0, "f32 bf16"},
};
const RadConstraint cSample[] = {
    {"n_vocab", RAD_C_GE, 1, nullptr},
    {"dtype", RAD_C_IN, 0, "f32 bf16"},
};
const RadConstraint cNorm[] = {
    {"n", RAD_C_GE, 1, nullptr},
    {"dtype", RAD_C_IN, 0, "bf16"},
};

enum { kPrioTile = 1000, kPrioDecode = 1100 };

const RadKernelInfo kRows[] = {
    {"gemm_nt_q_i8a8", "gemm_nt_q", "gemm",
     "int8 GEMM on gfx950 matrix cores: LDS tiles of 32 x 16 to 256 x 256 (up to M = 8 a GEMV where that "
     "is the faster one), summed exactly in i32, one scale a token and one an output channel applied once; K split over "
     "workgroups into i32 planes in launch scratch where tiles leave compute units idle",
     "K up to 131071 (the sum stays in i32); operands at any alignment and pitch (K, bases and "
     "pitches off 16 bytes: dword loads); M derives from numel(y)/N; scratch optional",
     "int8 a with f32 a_scale [M] or [M, 1], int8 b with f32 b_scale [N] or [N, 1], bf16 y; a_sum "
     "and b_ref refused",
     RAD_DOMAIN_DEVICE, kPrioTile, cI8, 1, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_gemm_nt_q_i8, r3d_rad_gemm_nt_q_i8_scratch, nullptr, nullptr, nullptr, nullptr},
    {"gemm_nt_q_i8a8_decode", "gemm_nt_q", "gemm",
     "int8 decode-band product on gfx950 matrix cores: up to M = 8 a GEMV (a wave 8 weight rows, whole lines "
     "from memory to registers, the tokens in LDS) or LDS tiles, whichever its cost makes the faster one; "
     "above, LDS tiles",
     "M <= 16; else as gemm_nt_q_i8a8",
     "as gemm_nt_q_i8a8",
     RAD_DOMAIN_DEVICE, kPrioDecode, cI8Decode, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_gemm_nt_q_i8_decode, r3d_rad_gemm_nt_q_i8_scratch, nullptr, nullptr, nullptr, nullptr},
    {"quant_act_i8", "quant_act_i8", "band",
     "int8 quantisation with one scale a row: a workgroup a row, the row in registers",
     "any n, alignment and pitch; rows past 32768 elements are walked twice",
     "f32/bf16 x, int8 q, f32 scale [M] or [M, 1]",
     RAD_DOMAIN_DEVICE, kPrioTile, cBand, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_quant_act_i8, nullptr, nullptr, nullptr, nullptr, nullptr},
    {"gated_quant_i8", "gated_quant_i8", "band",
     "silu(gate)*up or sigmoid(gate)*up fused with quant_act_i8",
     "as quant_act_i8; act silu (default) or sigmoid",
     "f32/bf16 gate_up [M, 2n], int8 q, f32 scale, optional bf16/f32 out",
     RAD_DOMAIN_DEVICE, kPrioTile, cBand, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_gated_quant_i8, nullptr, nullptr, nullptr, nullptr, nullptr},
    {"rmsnorm_quant_i8", "rmsnorm_quant_i8", "quant",
     "RMS norm (after the residual's addition) fused with quant_act_i8, the sum of squares in f64",
     "as quant_act_i8; w rank 1; residual and residual_out together or not at all",
     "bf16 x, residual and residual_out, f32/bf16 w, int8 q, f32 scale, optional bf16/f32 out",
     RAD_DOMAIN_DEVICE, kPrioTile, cNorm, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_rmsnorm_quant_i8, nullptr, nullptr, nullptr, nullptr, nullptr},
    {"sample_logits", "sample_logits", "vocab",
     "temperature, top-k, top-p and min-p sampling from given uniform numbers: masses in 64-bit "
     "integers from an f64 exp, cuts through a histogram of the row and a sort of its border bins",
     "n_vocab up to 4194304, at most 65535 rows, any alignment and pitch; launch scratch of the size "
     "the hook asks for (16-byte aligned) required; settings per row, a stride of 0 for all rows; "
     "temperature <= 0: the lowest index of the maximum; a row with no token: -1",
     "f32/bf16 logits, f32 u, temperature, top_p, min_p, i32 top_k, i32 token, optional f32 prob",
     RAD_DOMAIN_DEVICE, kPrioTile, cSample, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_sample_logits, r3d_rad_sample_logits_scratch, nullptr, nullptr, nullptr, nullptr},
};

bool row_hidden(const RadKernelInfo& k) {
    if (!strcmp(k.name, "sample_logits")) return r3d::env_no_sample();
    if (!strcmp(k.name, "gemm_nt_q_i8a8_decode")) return r3d::env_no_i8() || r3d::env_no_i8_dec();
    return r3d::env_no_i8();
}

}  // namespace

extern "C" {

int r3d_gfx950_ext_schema_count(void) { return (int)(sizeof kSchemas / sizeof kSchemas[0]); }

const RadOpSchema* r3d_gfx950_ext_schema_at(int i) {
    if (i < 0 || i >= r3d_gfx950_ext_schema_count()) return nullptr;
    return &kSchemas[i];
}

int r3d_gfx950_ext_kernel_count(void) {
    int n = 0;
    for (const RadKernelInfo& k : kRows)
        if (!row_hidden(k)) ++n;
    return n;
}

const RadKernelInfo* r3d_gfx950_ext_kernel_at(int i) {
    if (i < 0) return nullptr;
    for (const RadKernelInfo& k : kRows)
        if (!row_hidden(k) && i-- == 0) return &k;
    return nullptr;
}

}  /* extern "C" */
