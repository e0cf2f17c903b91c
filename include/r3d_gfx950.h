/* r3d_gfx950.h -- the C ABI exported by libr3d_gfx950.so.
 *
 * Every entry point replaces the reference libr3d export of the same name; the engine
 * (radiance, ABI 26) dlopens the library, reads the row table through the rad_* calls
 * and reaches the gemm_nt_q entries through RadKernelInfo::launch.  Plain C types and
 * device pointers only.
 */
#ifndef R3D_GFX950_H
#define R3D_GFX950_H

#include <stdint.h>
#include "rad_abi.h"
#include "rad_planes.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Plugin identity.  Replaces src/r3d_rows.cpp:16 (returns RAD_ABI_VERSION, 26) and
 * src/r3d_rows.cpp:18-27 (name, version, description, targets "gfx950"). */
uint32_t rad_plugin_abi_version(void);
const RadPluginInfo* rad_plugin_info(void);

/* Op schemas this plugin declares: gemm_nt_q (src/r3d_rows.cpp:186-210) and quant_act_fp8
 * (src/r3d_rows.cpp:615-625,985-990), parameters and operands exactly as there.
 * Replaces src/r3d_rows.cpp:2238-2247. */
int rad_kernel_schema_count(void);
const RadOpSchema* rad_kernel_schema_at(int i);

/* The row table after the registration-time kill switches (R3D_NO_MXFP4,
 * R3D_NO_FP4_DEC, R3D_NO_FP8A8, R3D_NO_FP8_DEC).  Replaces src/r3d_rows.cpp:2266-2278
 * with the gate of src/r3d_rows.cpp:2216-2236. */
int rad_kernel_count(void);
const RadKernelInfo* rad_kernel_at(int i);

/* gemm_nt_q at mxfp4a8, prefill row (any M).  Replaces src/r3d_gemm_mxfp4.hip:1587-1691.
 * Operands (a, a_scale, b, b_scale, y, a_sum?, b_ref?); params N, K, dtype "mxfp4a8";
 * M = numel(y)/N.  Returns RAD_OK, or RAD_E_UNSUPPORTED / RAD_E_SHAPE / RAD_E_STRIDE for a
 * refused format and RAD_E_DEVICE for a failed launch.  Asynchronous on `s`. */
int r3d_rad_gemm_nt_q(const RadArgs* a, RadStream s);

/* gemm_nt_q at mxfp4a8, decode band M <= 16.  Replaces src/r3d_gemm_mxfp4.hip:1712-2170
 * (r3d_rad_gemm_nt_q_mxfp4_decode and its q8x sibling share this one row here).  Beyond the
 * reference: at M = 1 it also takes a bf16 activation row with a_scale absent and quantises
 * it as quant_act_fp8 does (src/r3d_band.hip:117-153) before the products. */
int r3d_rad_gemm_nt_q_mxfp4_decode(const RadArgs* a, RadStream s);

/* gemm_nt_q at fp8a8, prefill row.  Replaces src/r3d_gemm_fp8a8.hip:1054-1099. */
int r3d_rad_gemm_nt_q_fp8(const RadArgs* a, RadStream s);

/* Scratch hooks (RadKernelInfo::scratch) of the two tile rows, r3d_rad_gemm_nt_q (mxfp4a8)
 * and r3d_rad_gemm_nt_q_fp8.  No counterpart in the reference, whose tile rows take no
 * scratch: up to M = 128 on an N too narrow to fill the chip with 128-row tiles, and from
 * M = 144 on where a whole-K walk of the larger tiles would leave compute units idle (planes of
 * at most 256 MiB), these rows split K across workgroups into f32 partial planes in
 * RadArgs::scratch and sum them in order on the same stream.  The hook returns the bytes of those planes (kc * M * N * 4 at
 * the N and K parameters and M = numel(y) / N -- without y the M parameter, else 128), 0 when no split applies.
 * The scratch is optional: a launch without it, or with less, or at an address that is not
 * 16-byte aligned, runs the unsplit arms (never a refusal). */
int64_t r3d_rad_gemm_nt_q_scratch(const RadArgs* a);
int64_t r3d_rad_gemm_nt_q_fp8_scratch(const RadArgs* a);

/* gemm_nt_q at fp8a8, decode band M <= 16.  Replaces src/r3d_gemm_fp8a8.hip:1101-1130.
 * Takes a bf16 activation row at M = 1 as the mxfp4a8 decode entry does. */
int r3d_rad_gemm_nt_q_fp8_decode(const RadArgs* a, RadStream s);

/* Scratch hooks (RadKernelInfo::scratch) of the two decode rows, r3d_rad_gemm_nt_q_mxfp4_decode
 * and r3d_rad_gemm_nt_q_fp8_decode.  No counterpart in the reference, whose decode rows take
 * no scratch: where the quad GEMV does not take the launch (M = 5..16, or an M <= 4 shape
 * whose activation rows it cannot stage) on a plane of at least 2^26 weights, and no
 * "splitk" tunable pins the GEMV's split, these rows split K across workgroups into f32
 * partial planes in RadArgs::scratch and sum them in order on the same stream.  The hook
 * returns the bytes of those planes (kc * M * N * 4 at the N and K parameters and M =
 * numel(y) / N -- without y the M parameter, else 16), 0 when no split applies.  The
 * scratch is optional: a launch without it, or with less, or at an address that is not
 * 16-byte aligned, runs the decode GEMVs (never a refusal). */
int64_t r3d_rad_gemm_nt_q_mxfp4_decode_scratch(const RadArgs* a);
int64_t r3d_rad_gemm_nt_q_fp8_decode_scratch(const RadArgs* a);

/* gemm_nt_q at dtype "mxfp4a16", prefill row (any M).  No counterpart in the reference:
 * the bf16-activation variant of the mxfp4 prefill (a bf16 [M, K], a_scale absent,
 * weights as mxfp4a8), for engines that feed unquantised activations.  The launch
 * quantises a to mxfp8 (e4m3 + E8M0 per 32 of K) into RadArgs::scratch, then runs the
 * block-scaled MFMA GEMM; both kernels run on `s`.  The launch-signature convention is
 * src/r3d_gemm_mxfp4.hip:1587-1588; the scratch refusal follows
 * src/r3d_gemm_fp8a8.hip:1214-1218 (RAD_E_UNSUPPORTED when scratch is missing or short). */
int r3d_rad_gemm_nt_q_mxfp4a16(const RadArgs* a, RadStream s);

/* The mxfp4a16 row's scratch hook (RadKernelInfo::scratch): bytes of launch scratch for
 * the M and K parameters, 0 when either is missing: the quantised activations, and after them
 * the f32 partial planes of a K split where one pays (from M = 144 on, with the N parameter).
 * A launch needs the former; with less than both it runs unsplit.  Same role as the reference's
 * src/r3d_gemm_fp8a8.hip:1249-1253. */
int64_t r3d_rad_gemm_nt_q_mxfp4a16_scratch(const RadArgs* a);

/* quant_act_fp8, the activation producer of the fp8a8 / mxfp4a8 rows: per-(row, group)
 * symmetric e4m3 codes of a bf16 or f32 activation, plain row-major, and the f32 dequant
 * scale amax/448 per group.  Operands (x, q, scale); params M, n, group, dtype.  Replaces
 * src/r3d_band.hip:460-487 (gates and refusal codes as there: RAD_E_INVAL for a missing
 * operand, RAD_E_DTYPE, RAD_E_SHAPE, RAD_E_STRIDE; RAD_E_DEVICE for a failed launch).
 * Asynchronous on `s`. */
int r3d_rad_quant_act_fp8(const RadArgs* a, RadStream s);

/* gated_quant_fp8: silu(gate) * up (or sigmoid(gate) * up), narrowed to bf16, then the
 * quant_act_fp8 quantiser.  Replaces src/r3d_band.hip:489-547 (r3d_rad_gated_quant_fp8). */
int r3d_rad_gated_quant_fp8(const RadArgs* a, RadStream s);

/* rmsnorm_quant_fp8: RMS norm (after an optional residual add written back) and the fp8
 * group quantiser over the bf16 normed row.  Replaces src/r3d_more.hip:479-539
 * (r3d_rad_rmsnorm_quant_fp8). */
int r3d_rad_rmsnorm_quant_fp8(const RadArgs* a, RadStream s);

/* gemm_nt_q_gated at fp8a8: the fp8a8 GEMM into the launch scratch, then gated_quant_fp8
 * over it.  Replaces src/r3d_gemm_fp8a8.hip:1163-1241 (r3d_rad_gemm_nt_q_gated_fp8). */
int r3d_rad_gemm_nt_q_gated_fp8(const RadArgs* a, RadStream s);

/* The gated row's scratch hook: 64 * N * 2 bytes (0 without N).  Replaces
 * src/r3d_gemm_fp8a8.hip:1246-1253 (r3d_rad_gemm_nt_q_gated_fp8_scratch). */
int64_t r3d_rad_gemm_nt_q_gated_fp8_scratch(const RadArgs* a);

/* logits_gemm over a joined e4m3 + block-scale head: bf16 x [M, n_embd], lm_head a
 * joined-planes blob (rad_planes.h: "codes" e4m3 [n_vocab, n_embd] dense, "scale" bf16 /
 * f16 / f32 per (1 or 128 rows, 128 columns)), f32 logits [M, n_vocab], M =
 * numel(logits) / n_vocab.  Replaces src/r3d_gemm_logits.hip:144-226
 * (r3d_rad_logits_gemm_e4m3).  n_embd a multiple of 4 at any alignment of x, codes and
 * scale (off a multiple of 16 or off 16-byte alignment: a slower dword walk).  The first
 * launch over a blob in device memory reads its header and entries with a copy on the
 * launch stream and waits for it (cached per device and address; refused with
 * RAD_E_UNSUPPORTED under graph capture -- launch once first); see
 * r3d_gfx950_logits_head_forget. */
int r3d_rad_logits_gemm_e4m3(const RadArgs* a, RadStream s);

/* The logits_gemm_e4m3 row's weight-layout hooks (host only).  Replace
 * src/r3d_gemm_logits.hip:233-272 (r3d_layout_head / r3d_relayout_head /
 * r3d_unrelayout_head, registered at src/r3d_rows.cpp:1598-1599).  They admit the head
 * (operand 1) as an untransformed "affine" encoding whose selected planes are "codes"
 * (tiled 1 x 1, e4m3, [n_vocab, n_embd]) then "scale" (tiled bf16 / f16 / f32, block
 * (1 or 128) x 128, [ceil(n_vocab / block), ceil(n_embd / 128)]) with n_embd a multiple of
 * 4 the launch can stage, and answer with the canonical rad.planes join (rad_planes.h):
 * layout gives its tag and bytes, relayout writes it into host memory dst, unrelayout
 * reads the planes back.  Any other operand: RAD_E_UNSUPPORTED (stored as is); any other
 * head, a plain one without that encoding included: declined (RAD_E_DTYPE, or RAD_E_SHAPE
 * for grids that disagree). */
int r3d_layout_head(const RadParam* p, int n_p, int operand, const RadEncoding* enc,
                    const int* sel, const RadTensor* planes, int n, RadLayout* out);
int r3d_relayout_head(const RadParam* p, int n_p, int operand, const RadEncoding* enc,
                      const int* sel, const RadTensor* planes, int n, void* dst,
                      int64_t dst_bytes);
int r3d_unrelayout_head(const RadParam* p, int n_p, int operand, const RadEncoding* enc,
                        const int* sel, const void* src, int64_t src_bytes,
                        const RadTensor* planes, int n);

/* The same join for a caller holding the two planes directly, no counterpart in the
 * reference (it is what r3d_relayout_head writes for the head's encoding), in host memory:
 *   _bytes: the blob's size for n_vocab x n_embd codes and a scale plane of scale_dtype
 *           (RAD_BF16 / RAD_F16 / RAD_F32) with scale_block_rows (1 or 128) rows per
 *           element, or a negative RAD_E_* code;
 *   _header: the same, and the blob's header and entries into *out (the planes go at the
 *           entries' offsets: a caller can stream them straight into device memory);
 *   _join:  writes header, entries, codes (rows codes_pitch bytes apart) and scale (rows
 *           scale_pitch_bytes apart, (n_embd + 127) / 128 elements each) into dst;
 *   _split: the inverse, into dense planes (either pointer may be null), after checking
 *           each plane's dtype, grid, pitch and extent against the blob; the planes take
 *           the blob's own grids (codes rows x cols bytes, scale rows x cols elements, as
 *           its entries state: read them first, _header or rad_planes_find, to size the
 *           destinations). */
int64_t r3d_gfx950_logits_head_bytes(int64_t n_vocab, int64_t n_embd, uint32_t scale_dtype,
                                     int64_t scale_block_rows);
int64_t r3d_gfx950_logits_head_header(int64_t n_vocab, int64_t n_embd, uint32_t scale_dtype,
                                      int64_t scale_block_rows, RadPlanesHead* out);
int r3d_gfx950_logits_head_join(const uint8_t* codes, int64_t codes_pitch, const void* scale,
                                int64_t scale_pitch_bytes, int64_t n_vocab, int64_t n_embd,
                                uint32_t scale_dtype, int64_t scale_block_rows, void* dst,
                                int64_t dst_bytes);
int r3d_gfx950_logits_head_split(const void* blob, int64_t blob_bytes, uint8_t* codes,
                                 void* scale);

/* No counterpart in the reference: drops the cached header of the blob at `blob` (every
 * device).  Call it before a different head is joined at an address a launch has used;
 * a launch whose cached header no longer matches the device's writes NaN logits. */
void r3d_gfx950_logits_head_forget(const void* blob);

/* gemm_nt_q at dtype "mxfp4a16" that allocates nothing: no counterpart in the reference,
 * for callers that cannot allocate (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  Same operands, parameters, kernels and results as
 * r3d_rad_gemm_nt_q_mxfp4a16 with R3D_NOALLOC_SCRATCH_BYTES of scratch, but RadArgs::scratch
 * is not used: the quantised activations, and a K split's planes where they fit behind them
 * (else the launch runs unsplit, its sums rounded in another order), go to a static device
 * buffer of that size per GPU, held until the process ends.  A call needing more (round256(M*K) + M*K/32 bytes) is refused with
 * RAD_E_SHAPE and a line on stderr.  All calls on one GPU share its buffer: calls that
 * overlap on one GPU (other streams, other threads) race. */
#define R3D_NOALLOC_SCRATCH_BYTES (16ll << 20)
int r3d_rad_gemm_nt_q_mxfp4a16_noalloc(const RadArgs* a, RadStream s);

/* Host-only diagnostic with no counterpart in the reference: runs `row`'s preamble and
 * plan on `a` and writes the chosen arm and launch geometry (or the refusal) into buf.
 * Launches nothing and copies nothing from the device: a logits head's header is read in
 * place when the blob is host-accessible, else taken from the copy an earlier launch
 * cached (RAD_E_UNSUPPORTED when there is none).  Plans for 256 compute units, a whole card; a launch for those
 * that its device has.  Returns the plan's status code. */
int r3d_gfx950_describe(const char* row, const RadArgs* a, char* buf, int len);

/* Diagnostic with no counterpart in the reference: one stage of a gemm_nt_q_mxfp4a16 call
 * on `s`, for timing and checking the stages apart.  stage 0 = the whole call (as the
 * row's launch), 1 = the mxfp8 quantiser alone (fills RadArgs::scratch), 2 = the
 * block-scaled GEMM alone on the planes already in RadArgs::scratch.  Same gates and
 * refusal codes as the row; RAD_E_INVAL for another stage; RAD_E_UNSUPPORTED where the
 * call would take the skinny band's decode passes (no quantiser stage there). */
int r3d_gfx950_mxfp4a16_stage(const RadArgs* a, RadStream s, int stage);

/* Measurement diagnostic with no counterpart in the reference: a read-only stream over
 * `bytes` of device memory at src on `s` -- each wave one contiguous run of kb KB read by
 * 1 KB loads (64 lanes x 16 bytes, non-temporal) kept 8 deep in flight, waves_per_wg
 * (1..8) waves a workgroup -- the ceiling an HBM-bound kernel of that access pattern and
 * size is held against.  bytes = 0 launches kb waves that do nothing (the launch floor).
 * sink: a device dword written only if the XOR of the data hits a fixed value.  RAD_OK,
 * RAD_E_INVAL for a bad argument, RAD_E_DEVICE if the launch fails. */
int r3d_gfx950_stream_probe(const void* src, int64_t bytes, int waves_per_wg, int64_t kb,
                            uint32_t* sink, RadStream s);

/* Measurement diagnostic with no counterpart in the reference: one wave on `s` runs `iters`
 * rounds of four 16 x 16 x 128 e4m3 MFMAs (four in-place accumulator chains) with `nv`
 * independent f32 fused multiply-adds before each (nv 0, 4, 8 or 16; with lag3 != 0, 4 or 8
 * multiply-adds that read the result of the MFMA issued three earlier), and writes the
 * shader-clock ticks the loop took to the device int64 at `cycles`.  work: a device buffer
 * of at least 1 KB (inputs read from its first 512 bytes, results written after them).
 * Divided by 4 * iters it gives the cost of one MFMA plus its share of VALU work: how much
 * VALU a wave hides under its own MFMAs.  RAD_OK, RAD_E_INVAL for a bad argument,
 * RAD_E_DEVICE if the launch fails. */
int r3d_gfx950_mfma_valu_probe(int nv, int lag3, int iters, void* work, int64_t* cycles,
                               RadStream s);

/* The second row table, with no counterpart in the reference: rows of ops and encodings past the
 * set that radiance's other plugins declare (int8: gemm_nt_q at i8a8 and its producers; a
 * sampler; a product with an epilogue; the norms between blocks; an expert layer), in the same structures, resolved
 * and launched the same way.  A loader compares the schemas of
 * rad_kernel_schema_at with other plugins', so these are listed apart; an engine that knows the ops
 * reads them here.  R3D_NO_I8, R3D_NO_I8_DEC, R3D_NO_SAMPLE, R3D_NO_EPI, R3D_NO_BLOCK_NORM and R3D_NO_MOE hide rows at
 * registration (R3D_NO_I8_DEC: the decode row, and no int8 call takes its GEMV; gemm_nt_epi's do not take it
 * either).  gemm_nt_q's schema is rad_kernel_schema_at's. */
int r3d_gfx950_ext_schema_count(void);
const RadOpSchema* r3d_gfx950_ext_schema_at(int i);
int r3d_gfx950_ext_kernel_count(void);
const RadKernelInfo* r3d_gfx950_ext_kernel_at(int i);

/* gemm_nt_q at i8a8: Y[m, n] = bf16((f32(sum_k A[m, k] B[n, k]) * a_scale[m]) * b_scale[n]), the
 * sum exact in i32.  Operands (a int8 [M, K], a_scale f32 [M] or [M, 1], b int8 [N, K], b_scale
 * f32 [N] or [N, 1], y bf16 [M, N]); params N, K, dtype "i8a8", group K if given; M =
 * numel(y) / N.  K <= 131071.  The _decode entry takes M <= 16.  RAD_OK, RAD_E_UNSUPPORTED /
 * RAD_E_SHAPE / RAD_E_STRIDE for refused operands, RAD_E_DEVICE for a failed launch.
 * Asynchronous on `s`. */
int r3d_rad_gemm_nt_q_i8(const RadArgs* a, RadStream s);
int r3d_rad_gemm_nt_q_i8_decode(const RadArgs* a, RadStream s);
/* Both rows' scratch hook: kc * M * N * 4 bytes of i32 planes where K is best split over
 * workgroups, else 0; at most 256 MiB.  Of a whole call its operands' alignment and pitches count, as they do
 * at the launch; with some of them absent: N, K and M = numel(y) / N (without y the M parameter, else 128),
 * as of dense operands on lines.  Optional, as for the other tile rows: with less, or off 16 bytes, K takes as few chunks
 * as fit.  Calls that share one buffer are ordered on one stream. */
int64_t r3d_rad_gemm_nt_q_i8_scratch(const RadArgs* a);

/* Producers of i8a8 activations: int8 codes q [M, n] and one f32 scale a row, [M] or [M, 1], of
 *   quant_act_i8       (x bf16/f32 [M, n], q, scale)
 *   gated_quant_i8     (gate_up bf16/f32 [M, 2n], q, scale, out?): act(gate) * up in f32, act
 *                      "silu" (default) or "sigmoid"
 *   rmsnorm_quant_i8   (x bf16, residual? bf16, w bf16/f32 [n], q, scale, out?, residual_out?):
 *                      r = bf16(residual + x) to residual_out (given together; residual_out may be
 *                      the memory of residual or of x), then (r / rms) * (w + wadd) in f32
 * scale = max(amax / 127, 2^-126), 1 for a row of zeros; q to nearest even.  A row of which these values (x,
 * act(gate) * up, the normed ones) hold a NaN, or else an infinity, has that as its scale and codes 0; an infinity
 * in rmsnorm_quant_i8's x, or -inf as silu's gate, makes a NaN of them.  Params n, dtype (x's), eps, wadd, act; M =
 * numel(x) / n.  out (bf16/f32 [M, n]) carries the values that the codes are of.  RAD_OK,
 * RAD_E_INVAL for a missing operand, RAD_E_DTYPE / RAD_E_SHAPE / RAD_E_STRIDE / RAD_E_UNSUPPORTED
 * (act) for refused ones, RAD_E_DEVICE.  Asynchronous on `s`. */
int r3d_rad_quant_act_i8(const RadArgs* a, RadStream s);
int r3d_rad_gated_quant_i8(const RadArgs* a, RadStream s);
int r3d_rad_rmsnorm_quant_i8(const RadArgs* a, RadStream s);

/* sample_logits: one token a row.  Operands (logits f32/bf16 [M, n_vocab], u f32, temperature? f32,
 * top_k? i32, top_p? f32, min_p? f32, token i32 out, prob? f32 out), the latter seven [M] or [M, 1],
 * inputs with a stride of 0 for one value for all rows; params n_vocab, dtype (the logits'); M =
 * numel(logits) / n_vocab.  In order: softmax at the temperature (<= 0: the lowest index of the
 * maximum), top_k (<= 0: off; ties to the lowest index), top_p of those (>= 1: off; at least one
 * token), min_p of those (times the largest probability; <= 0: off), then the first kept token in
 * index order whose running mass passes u times the kept mass.  NaN and -inf logits are not there;
 * a row of them gives token -1, prob 0.  n_vocab <= 4194304, M <= 65535.  Launch scratch of the size
 * the hook gives, 16-byte aligned, is required (else RAD_E_UNSUPPORTED); calls that share it are
 * ordered on one stream.  A cut among more than 8192 equal logits is slow (2 to 4 ms for some 20 us a row of
 * 262144): mask with -inf, not with a finite number, where top_k may ask for more tokens than are allowed.  RAD_E_INVAL / RAD_E_DTYPE / RAD_E_SHAPE / RAD_E_STRIDE for refused operands,
 * RAD_E_DEVICE for a failed launch.  Asynchronous on `s`; results do not depend on the run. */
int r3d_rad_sample_logits(const RadArgs* a, RadStream s);
int64_t r3d_rad_sample_logits_scratch(const RadArgs* a);

/* gemm_nt_epi: Y[m, n] = act(S * sum_k A[m, k] B[n, k] + bias[n]) + residual[m, n], rounded once.  The _bf16 entry takes bf16
 * a [M, K] and b [N, K] (S = 1, no scales), the _i8 entry int8 ones with a_scale f32 [M] or [M, 1] and b_scale f32 [N]
 * or [N, 1] (S their product, the sum exact in i32).  Operands (a, a_scale?, b, b_scale?, bias? f32/bf16 [N],
 * residual? f32/bf16 [M, N], y f32/bf16 [M, N]); params N, K, dtype "bf16" or "i8a8", act "none" (default), "relu", "silu",
 * "sigmoid", "gelu" (erf) or "gelu_tanh"; M = numel(y) / N.  K <= 1048576 at bf16, 131071 at i8a8.  y may be the residual's own
 * elements (same type and pitch) and meets no other operand; a residual or bias stride of 0 repeats one row or value.
 * Any alignment and pitch of the elements' own size; K, bases or pitches off 16 bytes are slow.  Sums are f32 at bf16, in an
 * order that the shape alone sets.  RAD_OK, RAD_E_INVAL / RAD_E_DTYPE / RAD_E_SHAPE / RAD_E_STRIDE /
 * RAD_E_UNSUPPORTED for refused operands, RAD_E_DEVICE for a failed launch.  Asynchronous on `s`.
 * The hooks: bytes of launch scratch (planes where K is split), optional as the int8 rows' is. */
int r3d_rad_gemm_nt_epi_bf16(const RadArgs* a, RadStream s);
int r3d_rad_gemm_nt_epi_i8(const RadArgs* a, RadStream s);
int64_t r3d_rad_gemm_nt_epi_bf16_scratch(const RadArgs* a);
int64_t r3d_rad_gemm_nt_epi_i8_scratch(const RadArgs* a);

/* rmsnorm_block: what lies between two blocks of a model, a row of n values at a time:
 *     t = x rs(x) (w_post + wadd), or x without w_post      rs(a) = 1 / sqrt(sum a^2 / n + eps)
 *     h = res_scale residual + gate t                       to residual_out, rounded to bf16
 *     v = h rs(h) (w_pre + wadd), of the f32 h              to out, and to q and scale as codes
 * Operands (x bf16/f32 [M, n], residual? bf16 [M, n], w_post? [n], gate? [n], [M, 1] or [M, n], w_pre? [n], residual_out? bf16
 * [M, n], out? bf16/f32 [M, n], q? [M, n], scale?); w_post, gate and w_pre of one type, bf16 or f32; w_pre with out or q, and
 * q with scale: int8 with one f32 a row (quant_act_i8's quantiser, [M] or [M, 1]), or e4m3 (RAD_U8 too) with one a group of 128
 * columns, [M, ceil(n / 128)], max(amax / 448, 2^-126), 1 for zeros.  Params n (<= 32768), eps, dtype (x's), wadd, res_scale
 * (1), group.  An output may be the own elements of x, the residual or the gate (same type and pitch) and meets nothing else.
 * Refusals and statuses as above; no scratch.  Asynchronous on `s`. */
int r3d_rad_rmsnorm_block(const RadArgs* a, RadStream s);

/* moe_layer: a mixture-of-experts layer for up to 64 tokens.  Of each token's router logits the top_k largest are chosen, by
 * falling logit, ties to the lower index; NaN and -inf are not there, and a token of which nothing is has ids -1, weights 0
 * and a y of zeros.  Weights: softmax over the logits or a sigmoid of each (score), divided by the chosen ones' sum (renorm,
 * default 1), times weight_scale.  Then y = sum over the choices of W_down (weight * act(W_gate x) * (W_up x)).
 * Operands (x bf16 [M, n], logits f32/bf16 [M, E], gate_up [E, 2f, n]: f gate rows, then f up rows; gate_up_scale?, down [E, n,
 * f], down_scale?, y f32/bf16 [M, n], ids? i32 [M, top_k], weights? f32 [M, top_k]); params n (<= 66560; i8: 62464), f (<= 65536),
 * E (<= 512), top_k (<= 16),
 * dtype, act (as above; silu), score "softmax" or "sigmoid", renorm, weight_scale.  dtype:
 *     "bf16"   no scales; n, f multiples of 8
 *     "i8"     int8 codes, f32 scales [E, rows] or [E, rows, 1]; multiples of 16
 *     "mxfp4"  e2m1 codes, E8M0 scales [E, rows, columns / 32] (0: 2^-127, 255: NaN); multiples of 32
 * x and the code planes on 16 bytes, their pitches too, an expert's plane under 2^31 bytes from its first to its last; any
 * distance between experts.  h is kept in f32; results do not depend on the run.  y may be x's or the logits' memory, ids and
 * weights may not, and no result may meet another, the planes or their scales.  Launch scratch of the size the hook gives,
 * 16-byte aligned, is required (else RAD_E_UNSUPPORTED); calls that share it are ordered on one stream.  Refusals and
 * statuses as above.  Asynchronous on `s`. */
int r3d_rad_moe_layer(const RadArgs* a, RadStream s);
int64_t r3d_rad_moe_layer_scratch(const RadArgs* a);

/* Build identity with no counterpart in the reference: the SHA-256 (hex) of the compile
 * flags and of the sources this library was compiled from -- the flags as one line, then
 * every file under libr3d_amd/csrc and include, in name order, each as "<relative
 * path>\n<bytes>" -- so a test harness can tell whether the binary it loaded was built
 * from the tree beside it. */
const char* r3d_gfx950_build_id(void);

#ifdef __cplusplus
}
#endif

#endif /* R3D_GFX950_H */
