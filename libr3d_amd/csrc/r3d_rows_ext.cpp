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
 *   gemm_nt_epi_bf16         prio 1000  dtype IN bf16                     product with an epilogue
 *   gemm_nt_epi_i8a8         prio 1000  dtype IN i8a8                     the same over int8 codes
 *   moe_layer                prio 1000  dtype IN bf16 i8 mxfp4, M LE 64     mixture-of-experts layer
 *   rmsnorm_block            prio 1000  n GE 1, dtype IN f32 bf16           norms, gate and residual between blocks
 *
 * R3D_NO_I8 hides the int8 rows, R3D_NO_I8_DEC the int8 decode row (and turns off its GEMV in the other
 * one, which takes those calls on its tiles), R3D_NO_SAMPLE the sampler, R3D_NO_EPI gemm_nt_epi's rows,
 * R3D_NO_BLOCK_NORM rmsnorm_block, R3D_NO_MOE moe_layer (presence-tested, read once; hidden at registration as in
 * r3d_rows.cpp).  gemm_nt_q's schema is rad_kernel_schema_at's. */
#include <stdint.h>
#include <string.h>

#include "rad_abi.h"
#include "r3d_block.h"
#include "r3d_epi.h"
#include "r3d_i8.h"
#include "r3d_moe.h"
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
int r3d_rad_gemm_nt_epi_bf16(const RadArgs* a, RadStream s);
int64_t r3d_rad_gemm_nt_epi_bf16_scratch(const RadArgs* a);
int r3d_rad_gemm_nt_epi_i8(const RadArgs* a, RadStream s);
int64_t r3d_rad_gemm_nt_epi_i8_scratch(const RadArgs* a);
int r3d_rad_rmsnorm_block(const RadArgs* a, RadStream s);
int r3d_rad_moe_layer(const RadArgs* a, RadStream s);
int64_t r3d_rad_moe_layer_scratch(const RadArgs* a);
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

const RadParamSpec kEpiParams[] = {
    {"M", RAD_P_INT, RAD_DERIVED, 0},
    {"N", RAD_P_INT, RAD_REQUIRED, 0},
    {"K", RAD_P_INT, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
    {"act", RAD_P_STR, RAD_OPTIONAL, 0},
};
const RadOperandSpec kEpiOperands[] = {
    {"a", RAD_OPD_IN, 0},
    {"a_scale", RAD_OPD_IN, 1},
    {"b", RAD_OPD_WEIGHT, 0},
    {"b_scale", RAD_OPD_WEIGHT, 1},
    {"bias", RAD_OPD_WEIGHT, 1},
    {"residual", RAD_OPD_IN, 1},
    {"y", RAD_OPD_OUT, 0},
};

const RadParamSpec kBlockParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n", RAD_P_INT, RAD_REQUIRED, 0},
    {"eps", RAD_P_F64, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
    {"wadd", RAD_P_F64, RAD_OPTIONAL, 0},
    {"res_scale", RAD_P_F64, RAD_OPTIONAL, 0},
    {"group", RAD_P_INT, RAD_OPTIONAL, 0},
};
const RadOperandSpec kBlockOperands[] = {
    {"x", RAD_OPD_IN, 0},
    {"residual", RAD_OPD_IN, 1},
    {"w_post", RAD_OPD_WEIGHT, 1},
    {"gate", RAD_OPD_IN, 1},
    {"w_pre", RAD_OPD_WEIGHT, 1},
    {"residual_out", RAD_OPD_OUT, 1},
    {"out", RAD_OPD_OUT, 1},
    {"q", RAD_OPD_OUT, 1},
    {"scale", RAD_OPD_OUT, 1},
};

const RadParamSpec kMoeParams[] = {
    {"M", RAD_P_INT, RAD_REQUIRED, 0},
    {"n", RAD_P_INT, RAD_REQUIRED, 0},
    {"f", RAD_P_INT, RAD_REQUIRED, 0},
    {"E", RAD_P_INT, RAD_REQUIRED, 0},
    {"top_k", RAD_P_INT, RAD_REQUIRED, 0},
    {"dtype", RAD_P_STR, RAD_REQUIRED, 0},
    {"act", RAD_P_STR, RAD_OPTIONAL, 0},
    {"score", RAD_P_STR, RAD_OPTIONAL, 0},
    {"renorm", RAD_P_INT, RAD_OPTIONAL, 0},
    {"weight_scale", RAD_P_F64, RAD_OPTIONAL, 0},
};
const RadOperandSpec kMoeOperands[] = {
    {"x", RAD_OPD_IN, 0},
    {"logits", RAD_OPD_IN, 0},
    {"gate_up", RAD_OPD_WEIGHT, 0},
    {"gate_up_scale", RAD_OPD_WEIGHT, 1},
    {"down", RAD_OPD_WEIGHT, 0},
    {"down_scale", RAD_OPD_WEIGHT, 1},
    {"y", RAD_OPD_OUT, 0},
    {"ids", RAD_OPD_OUT, 1},
    {"weights", RAD_OPD_OUT, 1},
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
    {"gemm_nt_epi", kEpiParams, 5, kEpiOperands, 7,
     "y = act(S * a . b^T + bias) + residual, rounded once: S = 1 at bf16, a_scale * b_scale at i8a8; act none "
     "(default), relu, silu, sigmoid, gelu or gelu_tanh; y may be the residual's memory."},
    {"rmsnorm_block", kBlockParams, 7, kBlockOperands, 9,
     "h = res_scale * residual + gate * norm(x; w_post), to residual_out in bf16, then norm(h; w_pre) of the f32 h: to out, "
     "and to q as int8 codes with one scale a row or e4m3 codes with one a group of 128; norm is the RMS norm times "
     "w + wadd, x itself without w_post; gate a value a channel [n], a token [M, 1] or an element [M, n]."},
    {"moe_layer", kMoeParams, 10, kMoeOperands, 9,
     "each token's top_k experts by falling router logit (ties to the lower index; NaN and -inf are not there), weights by "
     "softmax over the logits (default) or sigmoid, of the chosen ones' sum unless renorm is 0, times weight_scale; y = the "
     "sum of weight * down(act(gate x) * up x) in f32; ids (-1: none) and weights as chosen."},
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

const RadConstraint cMoe[] = {
    {"dtype", RAD_C_IN, 0, "bf16 i8 mxfp4"},
    {"M", RAD_C_LE, 64, nullptr},
};
const RadConstraint cEpiBf16[] = {
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
    {"gemm_nt_epi_bf16", "gemm_nt_epi", "gemm",
     "bf16 product with bias, activation and residual applied to its f32 sums: up to M = 8 a GEMV or LDS tiles, above "
     "LDS tiles of 32 x 16 to 256 x 256, K split over workgroups into f32 planes in launch scratch where tiles leave "
     "compute units idle",
     "K up to 1048576; operands at any alignment and pitch (row bytes, bases and pitches off 16 bytes: dword loads); "
     "M derives from numel(y)/N; scratch optional",
     "bf16 a and b, f32/bf16 bias [N], residual [M, N] and y",
     RAD_DOMAIN_DEVICE, kPrioTile, cEpiBf16, 1, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_gemm_nt_epi_bf16, r3d_rad_gemm_nt_epi_bf16_scratch, nullptr, nullptr, nullptr, nullptr},
    {"gemm_nt_epi_i8a8", "gemm_nt_epi", "gemm",
     "int8 product (gemm_nt_q_i8a8's) with bias, activation and residual applied to its scaled f32 values",
     "K up to 131071; else as gemm_nt_epi_bf16",
     "int8 a with f32 a_scale [M] or [M, 1], int8 b with f32 b_scale [N] or [N, 1], f32/bf16 bias, residual and y",
     RAD_DOMAIN_DEVICE, kPrioTile, cI8, 1, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_gemm_nt_epi_i8, r3d_rad_gemm_nt_epi_i8_scratch, nullptr, nullptr, nullptr, nullptr},
    {"rmsnorm_block", "rmsnorm_block", "quant",
     "the norm after a block, its gate, the residual's scale and addition, and the norm before the next block with its "
     "quantiser, in one pass: a workgroup a row, the row in registers, sums of squares in f64",
     "n up to 32768; any alignment and pitch; residual_out and out may be x's, the residual's or the gate's memory; q with "
     "scale; w_pre with out or q",
     "bf16/f32 x, bf16 residual and residual_out, w_post, gate and w_pre of one type (bf16/f32), bf16/f32 out, int8 q with "
     "f32 scale [M] or [M, 1], e4m3 q with f32 scale [M, ceil(n / 128)]",
     RAD_DOMAIN_DEVICE, kPrioTile, cBand, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_rmsnorm_block, nullptr, nullptr, nullptr, nullptr, nullptr},
    {"moe_layer", "moe_layer", "gemm",
     "a mixture-of-experts layer for up to 64 tokens: choice and gate/up products with their activation, then "
     "down products and the weighted sum; the chosen experts' planes are streamed, once for every 8 or 16 of an expert's "
     "tokens (fewer where n is over 8192 or so), codes become bf16 in registers",
     "E up to 512, top_k up to 16, n and f multiples of 8 (bf16), 16 (i8) or 32 (mxfp4), n up to 66560 (i8: 62464), f up to "
     "65536; x and the code planes on 16 bytes; launch scratch of the size the hook asks for (16-byte aligned) required",
     "bf16 x, f32/bf16 logits [M, E], gate_up [E, 2f, n] (gate rows, then up) and down [E, n, f] in bf16, in int8 with f32 "
     "scales [E, rows], or in e2m1 with E8M0 scales [E, rows, K / 32]; f32/bf16 y, i32 ids and f32 weights [M, top_k]",
     RAD_DOMAIN_DEVICE, kPrioTile, cMoe, 2, nullptr, 0, nullptr, nullptr, nullptr,
     r3d_rad_moe_layer, r3d_rad_moe_layer_scratch, nullptr, nullptr, nullptr, nullptr},
};

bool row_hidden(const RadKernelInfo& k) {
    if (!strcmp(k.name, "sample_logits")) return r3d::env_no_sample();
    if (!strcmp(k.op, "gemm_nt_epi")) return r3d::env_no_epi();
    if (!strcmp(k.name, "rmsnorm_block")) return r3d::env_no_block();
    if (!strcmp(k.name, "moe_layer")) return r3d::env_no_moe();
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
