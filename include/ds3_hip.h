/*
 * ds3_hip.h -- MI355X (gfx950) backend for the qw3 MoE-FFN path.
 *
 * A C ABI that replaces the MoE subset of the reference's Metal backend
 * (reference src/ds3_metal.h).  Every ds3_metal_* entry point the engine calls
 * on this path has a ds3_hip_* counterpart with the same argument order,
 * argument meaning, return convention (0 ok, -1 error with a diagnostic on
 * stderr) and accumulate/zeroing rules; the citation on each declaration names
 * the reference declaration it replaces.  ds3_metal_compat.h maps the
 * ds3_metal_* names onto these for source-level drop-in.
 *
 * Differences a caller can observe:
 *   - Routing (softmax, top-k, renormalisation) runs on the device; nothing is
 *     read back to the host.  gate_logits still receives the router logits.
 *   - The expert_up / expert_down / hidden scratch arguments are validated as
 *     in the reference but not used: the library keeps its own device
 *     workspace.
 *   - ds3_hip_buffer_from_mmap copies the host bytes into device memory once
 *     (the MI355X is a discrete device); the buffer stays read-only.
 *   - moe_router_topk_batch_tokens writes [n_layers][n_tokens][n_used] as its
 *     documentation states (the Metal kernel's stride is only right for
 *     n_layers == 1).
 *
 * Threading: one global device context and stream, as in the reference; not
 * thread-safe.  Outside begin_batch/end_batch every call is synchronous;
 * inside, calls are enqueued on the library stream and end_batch waits.
 */
#ifndef DS3_HIP_H
#define DS3_HIP_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* GGUF tensor type ids: the values of the reference's ds3_type_t
 * (reference src/ds3.h:201-216).  Passed as plain int32. */
typedef int32_t ds3_hip_type_t;
#define DS3_HIP_TYPE_F32  0
#define DS3_HIP_TYPE_F16  1
#define DS3_HIP_TYPE_Q8_0 8
#define DS3_HIP_TYPE_Q4_K 12
#define DS3_HIP_TYPE_Q6_K 14
/* Microscaled types of the *_mx calls, outside the range of GGUF's ids. */
#define DS3_HIP_TYPE_MXFP4  256
#define DS3_HIP_TYPE_MXINT8 257

/* Opaque device buffer (reference src/ds3_metal.h:14). */
typedef struct ds3_hip_buffer ds3_hip_buffer_t;

/* ---------------------------------------------------------------------- */
/* Lifecycle and buffers                                                  */
/* ---------------------------------------------------------------------- */

/* reference src/ds3_metal.h:19-20 */
int  ds3_hip_init(void);
void ds3_hip_shutdown(void);

/* reference src/ds3_metal.h:25-26.  NULL on failure or bytes == 0. */
ds3_hip_buffer_t *ds3_hip_buffer_alloc(size_t bytes);
void              ds3_hip_buffer_free(ds3_hip_buffer_t *buf);

/* reference src/ds3_metal.h:31.  base must be page-aligned; its bytes are
 * copied to the device; the buffer refuses writes. */
ds3_hip_buffer_t *ds3_hip_buffer_from_mmap(const void *base, size_t bytes);

/* reference src/ds3_metal.h:35-36.  Shares the parent's memory. */
ds3_hip_buffer_t *ds3_hip_buffer_view(const ds3_hip_buffer_t *base, size_t offset, size_t bytes);

/* reference src/ds3_metal.h:39-42 */
int ds3_hip_buffer_write(ds3_hip_buffer_t *buf, size_t offset, const void *src, size_t bytes);
int ds3_hip_buffer_read(ds3_hip_buffer_t *buf, size_t offset, void *dst, size_t bytes);

/* ---------------------------------------------------------------------- */
/* Products with (quantised) weights                                      */
/* ---------------------------------------------------------------------- */

/* reference src/ds3_metal.h:90-94: y[out] = W[out][in] . x, F32 W */
int ds3_hip_vec_matmul_f32(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                           uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);

/* reference src/ds3_metal.h:102-107: Q4_K / Q6_K / Q8_0 W */
int ds3_hip_vec_matmul_quantized(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                 uint32_t in_dim, uint32_t out_dim, uint64_t row_stride, ds3_hip_type_t type);

/* reference src/ds3_metal.h:115-137 (SIMD-group variants; same results) */
int ds3_hip_vec_matmul_f32_simd(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);
int ds3_hip_vec_matmul_q8_0_simd(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                 uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);
int ds3_hip_vec_matmul_q4k_simd(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);
int ds3_hip_vec_matmul_q6k_simd(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);

/* reference src/ds3_metal.h:142-146: Q4_K product with an fp16 input vector
 * x[in_dim] (widened exactly to fp32), y[out_dim] fp32. */
int ds3_hip_vec_matmul_q4k_half(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *y,
                                uint32_t in_dim, uint32_t out_dim, uint64_t row_stride);

/* reference src/ds3_metal.h:154-161: C[M][N] = A[M][K] . W[N][K]^T, fp32,
 * W at byte weight_offset inside the buffer.  Below the dense-MFMA row
 * count (ds3_hip_set_dense_mfma_min_rows, default 64), and for shapes the fp16
 * path does not take, every product is of fp32 operands, the weights decoded
 * exactly, and summed in fp32: by VALU FMAs or, from two or three rows and for
 * long one-row products, on the fp32 matrix cores.  The order of the sums
 * differs between the two and from the reference kernel's (relative L2 error
 * 1.2e-7 either way).  From that many rows, for Q4_K / Q6_K / Q8_0 with K a
 * multiple of 512 and N a multiple of 256 (the engine's prefill projections),
 * the product runs on the matrix cores with fp16 operands (A and the decoded
 * weights rounded to fp16, fp32 accumulation), the precision of the MoE
 * grouped products: relative L2 error ~5e-4 against fp32. */
int ds3_hip_matmul_quantized_batch(const ds3_hip_buffer_t *A, const ds3_hip_buffer_t *W, ds3_hip_buffer_t *C,
                                   uint32_t M, uint32_t N, uint32_t K, uint64_t weight_row_stride,
                                   uint64_t weight_offset, ds3_hip_type_t type);

/* ---------------------------------------------------------------------- */
/* Elementwise                                                            */
/* ---------------------------------------------------------------------- */

/* reference src/ds3_metal.h:168-178 */
int ds3_hip_buffer_copy_f32(const ds3_hip_buffer_t *src, ds3_hip_buffer_t *dst, size_t bytes);
int ds3_hip_buffer_zero_f32(ds3_hip_buffer_t *buf, size_t bytes);
int ds3_hip_vec_add_inplace(ds3_hip_buffer_t *acc, const ds3_hip_buffer_t *addend, uint32_t n);
int ds3_hip_vec_add(const ds3_hip_buffer_t *a, const ds3_hip_buffer_t *b, ds3_hip_buffer_t *c, uint32_t n);

/* reference src/ds3_metal.h:184-192:
 *   gather : dst[i][j]  = src[ids[offset+i]][j]
 *   scatter: dst[ids[offset+i]][j] += scores[offset+i] * src[i][j] */
int ds3_hip_gather_rows_f32(const ds3_hip_buffer_t *src, const ds3_hip_buffer_t *ids, ds3_hip_buffer_t *dst,
                            uint32_t n_cols, uint32_t count, uint32_t offset);
int ds3_hip_scatter_add_weighted_f32(const ds3_hip_buffer_t *src, const ds3_hip_buffer_t *scores,
                                     const ds3_hip_buffer_t *ids, ds3_hip_buffer_t *dst,
                                     uint32_t n_cols, uint32_t count, uint32_t offset);

/* reference src/ds3_metal.h:195-198: out[i] = silu(gate[i]) * up[i] */
int ds3_hip_silu_mul_f32(const ds3_hip_buffer_t *gate, const ds3_hip_buffer_t *up, ds3_hip_buffer_t *out,
                         uint32_t n);

/* reference src/ds3_metal.h:48-57 (the FFN block's prologue, src/ds3_engine.c:522):
 * out[r] = x[r] / sqrt(mean(x[r]^2) + eps) * weight for n_rows rows of n.
 * The reference's formula; the sum of squares is a fixed-order tree, so the
 * result can differ from the CPU reference's left-to-right sum in the last
 * bits (as the reference's own Metal kernel's does). */
int ds3_hip_rms_norm(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *weight, ds3_hip_buffer_t *out,
                     uint32_t n, uint32_t n_rows, float eps);

/* ---------------------------------------------------------------------- */
/* MoE FFN                                                                */
/* ---------------------------------------------------------------------- */

/* reference src/ds3_metal.h:340-374 (one token).  output accumulates
 * (caller zeroes it).  expert_offsets: optional [n_expert][3] uint64 byte
 * offsets {gate, up, down}; when NULL expert e starts at e*rows*row_stride.
 * Routing uses the certified router (see ds3_hip_set_router_mode): the
 * selected experts are the reference's; gate_logits are within a proven
 * bound of the reference's sequential fp32 sums. */
int ds3_hip_moe_ffn(
    const ds3_hip_buffer_t *input, const ds3_hip_buffer_t *w_gate_inp,
    const ds3_hip_buffer_t *w_gate_exps, const ds3_hip_buffer_t *w_up_exps, const ds3_hip_buffer_t *w_down_exps,
    ds3_hip_type_t gate_type, ds3_hip_type_t up_type, ds3_hip_type_t down_type,
    uint64_t gate_row_stride, uint64_t up_row_stride, uint64_t down_row_stride,
    const ds3_hip_buffer_t *w_shared_gate, const ds3_hip_buffer_t *w_shared_up, const ds3_hip_buffer_t *w_shared_down,
    ds3_hip_type_t shared_gate_type, ds3_hip_type_t shared_up_type, ds3_hip_type_t shared_down_type,
    uint64_t shared_gate_row_stride, uint64_t shared_up_row_stride, uint64_t shared_down_row_stride,
    ds3_hip_buffer_t *output, ds3_hip_buffer_t *gate_logits, const ds3_hip_buffer_t *expert_offsets,
    ds3_hip_buffer_t *hidden, ds3_hip_buffer_t *expert_up, ds3_hip_buffer_t *expert_down,
    uint32_t n_embd, uint32_t n_expert, uint32_t n_used, uint32_t n_ff_exp, uint32_t n_ff_shared,
    uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);

/* reference src/ds3_metal.h:380-387: gate_logits = router . input */
int ds3_hip_moe_ffn_router(const ds3_hip_buffer_t *input, const ds3_hip_buffer_t *w_gate_inp,
                           ds3_hip_buffer_t *gate_logits, uint32_t n_embd, uint32_t n_expert,
                           uint64_t router_row_stride, ds3_hip_type_t router_type);

/* reference src/ds3_metal.h:389-418: shared + host-selected experts */
int ds3_hip_moe_ffn_experts(
    const ds3_hip_buffer_t *input,
    const ds3_hip_buffer_t *w_gate_exps, const ds3_hip_buffer_t *w_up_exps, const ds3_hip_buffer_t *w_down_exps,
    ds3_hip_type_t gate_type, ds3_hip_type_t up_type, ds3_hip_type_t down_type,
    uint64_t gate_row_stride, uint64_t up_row_stride, uint64_t down_row_stride,
    const ds3_hip_buffer_t *w_shared_gate, const ds3_hip_buffer_t *w_shared_up, const ds3_hip_buffer_t *w_shared_down,
    ds3_hip_type_t shared_gate_type, ds3_hip_type_t shared_up_type, ds3_hip_type_t shared_down_type,
    uint64_t shared_gate_row_stride, uint64_t shared_up_row_stride, uint64_t shared_down_row_stride,
    ds3_hip_buffer_t *output, ds3_hip_buffer_t *hidden, ds3_hip_buffer_t *expert_up, ds3_hip_buffer_t *expert_down,
    uint32_t n_embd, uint32_t n_used, uint32_t n_ff_exp, uint32_t n_ff_shared,
    const int32_t *indices_host, const float *scores_host);

/* reference src/ds3_metal.h:424-431: logits [L][E] -> indices/scores [L][k] */
int ds3_hip_moe_router_topk_batch(const ds3_hip_buffer_t *logits, ds3_hip_buffer_t *indices,
                                  ds3_hip_buffer_t *scores, uint32_t n_layers, uint32_t n_expert,
                                  uint32_t n_used, bool norm_topk_prob);

/* reference src/ds3_metal.h:437-445: logits [L][T][E] -> [L][T][k] */
int ds3_hip_moe_router_topk_batch_tokens(const ds3_hip_buffer_t *logits, ds3_hip_buffer_t *indices,
                                         ds3_hip_buffer_t *scores, uint32_t n_layers, uint32_t n_tokens,
                                         uint32_t n_expert, uint32_t n_used, bool norm_topk_prob);

/* ---------------------------------------------------------------------- */
/* Batching and profiling                                                 */
/* ---------------------------------------------------------------------- */

/* reference src/ds3_metal.h:457-462 */
int  ds3_hip_begin_batch(void);
void ds3_hip_end_batch(void);
void ds3_hip_synchronize(void);

/* reference src/ds3_metal.h:467-468 (enabled by DS3_HIP_PROFILE=1) */
void ds3_hip_profile_reset(void);
void ds3_hip_profile_print(const char *label);

/* ---------------------------------------------------------------------- */
/* Device-routed extensions (no ds3_metal.h counterpart)                  */
/* ---------------------------------------------------------------------- */

/* The whole MoE FFN for T tokens with no host round trip: router logits,
 * softmax/top-k/renorm, then either per-token expert GEMVs (T at most the
 * crossover, see ds3_hip_set_prefill_min_tokens) or bucketing + grouped
 * fp16-MFMA products + in-order combine.  Replaces the engine's decode and
 * gathered-prefill sequences (reference src/ds3_engine.c:520-597, 895-1022).
 *   input [T][n_embd] f32; output [T][n_embd] f32 accumulates (caller
 *   zeroes); residual (optional) [T][n_embd] is added to output; output
 *   may be input itself (input += MoE(input), in place, no residual);
 *   indices / scores (optional) receive the routing [T][n_used];
 *   gate_logits (optional) receives the logits [T][n_expert].
 * The grouped products take fp16 operands (x, decoded weights, h) and keep
 * the down outputs in fp16 before the fp32 combine: outputs within rel-L2
 * 1e-3 of the fp32 reference; the per-token GEMVs are fp32 throughout.
 * Up to 16 tokens (see ds3_hip_set_router_mode) the router is the certified
 * one: indices equal the reference's; gate_logits hold the fp32 rounding of
 * the exact sum of the reference's fp32 products (the reference's own
 * sequential sums for experts whose order needed them), within a proven
 * bound of the reference's logits. */
int ds3_hip_moe_ffn_batch(
    const ds3_hip_buffer_t *input, const ds3_hip_buffer_t *w_gate_inp,
    const ds3_hip_buffer_t *w_gate_exps, const ds3_hip_buffer_t *w_up_exps, const ds3_hip_buffer_t *w_down_exps,
    ds3_hip_type_t gate_type, ds3_hip_type_t up_type, ds3_hip_type_t down_type,
    uint64_t gate_row_stride, uint64_t up_row_stride, uint64_t down_row_stride,
    const ds3_hip_buffer_t *expert_offsets,
    ds3_hip_buffer_t *output, const ds3_hip_buffer_t *residual,
    ds3_hip_buffer_t *gate_logits, ds3_hip_buffer_t *indices, ds3_hip_buffer_t *scores,
    uint32_t n_tokens, uint32_t n_embd, uint32_t n_expert, uint32_t n_used, uint32_t n_ff_exp,
    uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);

/* The engine's whole FFN block for T tokens in one call (reference
 * src/ds3_engine.c:519-527 and 675-720: rms_norm, zeroing, moe_ffn and the
 * residual vec_add): hidden[t] += MoE(rms_norm(hidden[t]) * ffn_norm), in
 * place.  The normalised rows go to x_norm when given (it must not overlap
 * hidden), else to the library's workspace; everything else as
 * ds3_hip_moe_ffn_batch with input = the normalised rows, output = hidden
 * (accumulating) and no separate residual.  No counterpart in ds3_metal.h. */
int ds3_hip_moe_block(
    ds3_hip_buffer_t *hidden, const ds3_hip_buffer_t *ffn_norm, float eps, const ds3_hip_buffer_t *w_gate_inp,
    const ds3_hip_buffer_t *w_gate_exps, const ds3_hip_buffer_t *w_up_exps, const ds3_hip_buffer_t *w_down_exps,
    ds3_hip_type_t gate_type, ds3_hip_type_t up_type, ds3_hip_type_t down_type,
    uint64_t gate_row_stride, uint64_t up_row_stride, uint64_t down_row_stride,
    const ds3_hip_buffer_t *expert_offsets, ds3_hip_buffer_t *x_norm,
    ds3_hip_buffer_t *gate_logits, ds3_hip_buffer_t *indices, ds3_hip_buffer_t *scores,
    uint32_t n_tokens, uint32_t n_embd, uint32_t n_expert, uint32_t n_used, uint32_t n_ff_exp,
    uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);

/* ds3_hip_moe_ffn_batch that allocates nothing.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * Same arguments, semantics and results as ds3_hip_moe_ffn_batch; every
 * intermediate (routing rows, bucketing lists, h, y) lives in one library-owned
 * scratch array of ds3_hip_noalloc_scratch_bytes() bytes per GPU (64 MiB: a
 * Qwen3-30B-A3B layer call of up to 1,284 tokens), held until the process ends.
 * A call whose intermediates do not fit returns -1 with a diagnostic; split it
 * into fewer tokens.  ds3_hip_init must have been called.  Every call on a GPU
 * shares that GPU's array: calls that overlap on one GPU (from several host
 * threads, or a graph replay with an eager call of this entry point on another
 * stream) race.  The array keeps the last call's contents; no kernel reads a
 * byte of it before the same call has written it. */
int ds3_hip_moe_ffn_batch_noalloc(
    const ds3_hip_buffer_t *input, const ds3_hip_buffer_t *w_gate_inp,
    const ds3_hip_buffer_t *w_gate_exps, const ds3_hip_buffer_t *w_up_exps, const ds3_hip_buffer_t *w_down_exps,
    ds3_hip_type_t gate_type, ds3_hip_type_t up_type, ds3_hip_type_t down_type,
    uint64_t gate_row_stride, uint64_t up_row_stride, uint64_t down_row_stride,
    const ds3_hip_buffer_t *expert_offsets,
    ds3_hip_buffer_t *output, const ds3_hip_buffer_t *residual,
    ds3_hip_buffer_t *gate_logits, ds3_hip_buffer_t *indices, ds3_hip_buffer_t *scores,
    uint32_t n_tokens, uint32_t n_embd, uint32_t n_expert, uint32_t n_used, uint32_t n_ff_exp,
    uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);
size_t ds3_hip_noalloc_scratch_bytes(void);

/* Router only, for T tokens: logits (bit-identical to the reference's
 * sequential fp32 sums), then indices/scores [T][n_used]. */
int ds3_hip_moe_route(const ds3_hip_buffer_t *input, const ds3_hip_buffer_t *w_gate_inp,
                      ds3_hip_buffer_t *gate_logits, ds3_hip_buffer_t *indices, ds3_hip_buffer_t *scores,
                      uint32_t n_tokens, uint32_t n_embd, uint32_t n_expert, uint32_t n_used,
                      uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);

/* Bucketing of routed slots (reference src/ds3_engine.c:932-955, compacted):
 * counts [n_expert], offsets [n_expert+1], ids/wts/slot_pos [T*n_used]. */
int ds3_hip_moe_bucket(const ds3_hip_buffer_t *indices, const ds3_hip_buffer_t *scores,
                       uint32_t n_tokens, uint32_t n_used, uint32_t n_expert,
                       ds3_hip_buffer_t *counts, ds3_hip_buffer_t *offsets, ds3_hip_buffer_t *ids,
                       ds3_hip_buffer_t *wts, ds3_hip_buffer_t *slot_pos);

/* Dequantise n values of `type` from src (byte offset src_offset) to f32 dst
 * (the parity probe for the block decoders). */
int ds3_hip_dequantize(const ds3_hip_buffer_t *src, uint64_t src_offset, ds3_hip_type_t type, uint64_t n,
                       ds3_hip_buffer_t *dst);

/* ---------------------------------------------------------------------- */
/* Microscaled operators (no ds3_metal.h counterpart)                     */
/* ---------------------------------------------------------------------- */

/* 4-bit weights that the matrix cores take as they are, and rows in 8 bits
 * for them.  A microscaled matrix [n_rows][n_cols], n_cols a multiple of 32
 * up to 2^27, is two buffers (the element and scale formats of the OCP MX
 * specification):
 *   scales [n_rows][n_cols / 32]: a byte c per 32 consecutive values, for
 *     2^(c - 127); 255 makes the whole block NaN;
 *   codes, starting on a multiple of 16 bytes, rows without gaps:
 *     DS3_HIP_TYPE_MXFP4  [n_rows][n_cols / 2]: E2M1 nibbles, bit 3 the sign,
 *       bits 0..2 the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6; value 2j in the
 *       low half of byte j;
 *     DS3_HIP_TYPE_MXINT8 [n_rows][n_cols]: signed bytes q, for q / 64.
 * All calls: -1 for a null or too small buffer, sizes that a type does not
 * take, an output that overlaps an input or another output, or a read-only
 * output; 0 and nothing done for zero rows.  All but
 * ds3_hip_moe_block_mx need no workspace and can be captured without a call
 * before. */

/* Rounds rows of src (F32, F16, Q8_0, Q4_K or Q6_K rows, src_row_stride bytes
 * apart; n_cols a multiple of 256 for Q4_K / Q6_K; src and its stride
 * multiples of 4 / 2 / 2 / 16 / 2 bytes) to a microscaled type, to nearest
 * with ties to even.  A block's scale is 2^floor(log2 amax) for MXINT8, whose q
 * saturates at +-127, and for MXFP4 the smallest power of two with amax at
 * most 7 times it.  A block with an infinity or a NaN gets scale 255, one of
 * zeros scale 0. */
int ds3_hip_mx_quantize(const ds3_hip_buffer_t *src, ds3_hip_type_t src_type, uint64_t src_row_stride,
                        ds3_hip_buffer_t *codes, ds3_hip_buffer_t *scales, ds3_hip_type_t mx_type,
                        uint32_t n_rows, uint32_t n_cols);

/* The values of a microscaled matrix, to F32 or F16 rows without gaps: exact in
 * F32 but for magnitudes of 2^128 and more (scale 254 only), which become
 * infinite, and rounded once to F16. */
int ds3_hip_mx_dequantize(const ds3_hip_buffer_t *codes, const ds3_hip_buffer_t *scales, ds3_hip_type_t mx_type,
                          uint32_t n_rows, uint32_t n_cols, ds3_hip_buffer_t *dst, ds3_hip_type_t dst_type);

/* The prologue of an FFN block in one pass over n_rows rows of n: s = x +
 * delta (delta NULL: s = x), y = s / sqrt(mean(s^2) + eps) * weight, and y
 * rounded to MXINT8 rows as ds3_hip_mx_quantize rounds it.  sum (optional)
 * receives s and may be x or delta; x_norm (optional) receives y, for the
 * router.  sum is rounded once; y is computed in 64 bits from the unrounded
 * s and rounded once.
 * n is a multiple of 32; every row's result is the same on every call. */
int ds3_hip_add_rms_norm_mx(const ds3_hip_buffer_t *x, const ds3_hip_buffer_t *delta, const ds3_hip_buffer_t *weight,
                            float eps, ds3_hip_buffer_t *sum, ds3_hip_buffer_t *x_norm, ds3_hip_buffer_t *codes,
                            ds3_hip_buffer_t *scales, uint32_t n, uint32_t n_rows);

/* C[M][N] = X[M][K] . W[N][K]^T in fp32 of MXINT8 rows and MXFP4 weights.
 * Every product is exact and summed in fp32; the order of a sum depends on
 * the sizes alone.  Blocks of x whose scale is below 2^-122 are the exception:
 * their values are first rounded to multiples of 2^-128. */
int ds3_hip_matmul_mx(const ds3_hip_buffer_t *x_codes, const ds3_hip_buffer_t *x_scales,
                      const ds3_hip_buffer_t *w_codes, const ds3_hip_buffer_t *w_scales, ds3_hip_buffer_t *C,
                      uint32_t M, uint32_t N, uint32_t K);

/* The same for rows grouped by expert, as ds3_hip_moe_bucket orders them:
 *   C[r][n] = x[ids ? ids[r] : r] . w[g * N + n],  offsets[g] <= r < offsets[g + 1]
 * offsets int32 [n_group + 1], never decreasing, n_group at most 1024; ids
 * int32 [n_rows]; x has n_x rows, w n_group * N.  Groups may be empty and of
 * any size.  Rows of C outside every group, and rows whose id is no row of x,
 * are left as they were.  Offsets are taken into 0 .. n_rows; where they
 * decrease the values of C are unspecified, nothing outside it is touched. */
int ds3_hip_matmul_mx_grouped(const ds3_hip_buffer_t *x_codes, const ds3_hip_buffer_t *x_scales,
                              const ds3_hip_buffer_t *w_codes, const ds3_hip_buffer_t *w_scales,
                              const ds3_hip_buffer_t *offsets, const ds3_hip_buffer_t *ids, ds3_hip_buffer_t *C,
                              uint32_t n_x, uint32_t n_rows, uint32_t n_group, uint32_t N, uint32_t K);

/* The experts' first half: h[r] = silu(x . gate) * (x . up) with rows and
 * groups as in ds3_hip_matmul_mx_grouped (N = n_ff, K = n_embd), rounded to
 * MXINT8 rows, the x of the down product.  n_ff is a multiple of 32. */
int ds3_hip_moe_gate_up_mx(const ds3_hip_buffer_t *x_codes, const ds3_hip_buffer_t *x_scales,
                           const ds3_hip_buffer_t *gate_codes, const ds3_hip_buffer_t *gate_scales,
                           const ds3_hip_buffer_t *up_codes, const ds3_hip_buffer_t *up_scales,
                           const ds3_hip_buffer_t *offsets, const ds3_hip_buffer_t *ids,
                           ds3_hip_buffer_t *h_codes, ds3_hip_buffer_t *h_scales, uint32_t n_x, uint32_t n_rows,
                           uint32_t n_group, uint32_t n_ff, uint32_t n_embd);

/* The experts' outputs back in token order: out[t] (+)= the sum over j, in
 * order, of scores[t][j] * y[slot_pos[t][j]], y f32 [n_rows][n_cols] (as
 * ds3_hip_matmul_mx_grouped writes it for ds3_hip_moe_bucket's lists), slot_pos
 * int32 and scores f32 [n_tokens][n_used], out f32 [n_tokens][n_cols].  Slots
 * that are no row of y (moe_bucket marks dropped ones -1) add nothing. */
int ds3_hip_moe_combine(const ds3_hip_buffer_t *y, const ds3_hip_buffer_t *slot_pos, const ds3_hip_buffer_t *scores,
                        ds3_hip_buffer_t *out, uint32_t n_tokens, uint32_t n_used, uint32_t n_rows, uint32_t n_cols,
                        bool accumulate);

/* ds3_hip_moe_block with microscaled experts, in place: hidden[t] += delta[t]
 * (delta may be NULL), then hidden[t] += MoE(rms_norm(s[t]) * ffn_norm), s the sum
 * before its rounding, as in ds3_hip_add_rms_norm_mx.
 * The experts are MXFP4 matrices: gate and up [n_expert * n_ff_exp][n_embd], down
 * [n_expert * n_embd][n_ff_exp]; the router reads the normalised rows in f32,
 * the experts the same rows in MXINT8, and h is rounded to MXINT8.  gate_logits /
 * indices / scores (optional) as in ds3_hip_moe_ffn_batch, with its limits on
 * n_expert and n_used, but that the certified router's scores come from its
 * logits in 64 bits.  n_tokens is below 2^26.  It uses the library's workspace:
 * before a capture the call is made once. */
int ds3_hip_moe_block_mx(ds3_hip_buffer_t *hidden, const ds3_hip_buffer_t *delta, const ds3_hip_buffer_t *ffn_norm,
                         float eps, const ds3_hip_buffer_t *w_gate_inp,
                         const ds3_hip_buffer_t *gate_codes, const ds3_hip_buffer_t *gate_scales,
                         const ds3_hip_buffer_t *up_codes, const ds3_hip_buffer_t *up_scales,
                         const ds3_hip_buffer_t *down_codes, const ds3_hip_buffer_t *down_scales,
                         ds3_hip_buffer_t *gate_logits, ds3_hip_buffer_t *indices, ds3_hip_buffer_t *scores,
                         uint32_t n_tokens, uint32_t n_embd, uint32_t n_expert, uint32_t n_used, uint32_t n_ff_exp,
                         uint64_t router_row_stride, ds3_hip_type_t router_type, bool norm_topk_prob);

/* Attention and sampling operators (no ds3_metal.h counterpart): what lies
 * between a layer's q / k / v products and its output product, and between the
 * output head and the next token.
 *
 * A paged cache of one layer is two F16 buffers, k and v, each
 * [n_blocks][n_head_kv][block_size][head_dim]; block_size is a power of two.  A
 * slot is block * block_size + row of the block.  Request i's block_table row
 * ([max_blocks] int32) names the blocks of its positions in order.  The tokens of
 * a call lie request after request: rows q_offsets[i] .. q_offsets[i + 1] - 1 of
 * n_seq + 1 int32 belong to request i; rows from q_offsets[n_seq] on belong to none.
 * What device buffers hold cannot be refused by the host: slots and block ids
 * outside the cache are passed over (not written, not read), and each entry point
 * says what other values do.
 * Buffers: int32 ones, logits and settings start on multiples of 4 bytes, tables of
 * angles on multiples of 8, heads, caches and norms on multiples of 16; rows of heads lie
 * a multiple of 16 bytes apart. */

/* Angles of rotary positions, computed on the host in 64 bits and written to
 * `table` (rotary_dim / 2 + 1 doubles): pair i turns by position * f(theta_i),
 * theta_i = base^(-2 i / rotary_dim).  With r_i = original_ctx * theta_i / (2 pi),
 * the turns of pair i over the trained context:
 *   PLAIN       f = theta
 *   LINEAR      f = theta / factor
 *   WAVELENGTH  f = theta * (s + (1 - s) / factor), s = (r - low) / (high - low)
 *               held to 0 .. 1
 *   YARN        f = theta * (1 - s + s / factor), s = (i - a) / (b - a) held to
 *               0 .. 1, a and b the pair indices (rounded down and up, held to 0 ..
 *               rotary_dim - 1) at which r is `high` and `low`; rotated values are
 *               scaled by 0.1 ln(factor) + 1 where factor > 1.
 * rotary_dim is even, up to 512.  Not allowed during graph capture. */
#define DS3_HIP_ROPE_PLAIN      0
#define DS3_HIP_ROPE_LINEAR     1
#define DS3_HIP_ROPE_WAVELENGTH 2
#define DS3_HIP_ROPE_YARN       3
int ds3_hip_rope_table(ds3_hip_buffer_t *table, uint32_t rotary_dim, double base, int32_t scaling, double factor,
                       double low, double high, uint32_t original_ctx);

/* out = x rotated by its tokens' positions (int32, any value).  A row of x holds
 * n_head heads of head_dim values (F32 or F16), rows x_row_stride bytes apart; out
 * likewise.  With norm (F32 [head_dim]) each head is first x * rsqrt(mean(x^2) +
 * eps) * norm, in F32.  The first rotary_dim values of a head turn: value i with
 * value i + rotary_dim / 2, or interleaved, 2 i with 2 i + 1; the rest are copied
 * (normalised).  Angles are reduced in 64 bits.  out may be x itself (one type,
 * one stride).  head_dim is a multiple of 8 up to 512, rotary_dim even.  Calls of more
 * than 2^24 - 1 workgroups are refused: 256 lanes each, a head's lanes its values / 8
 * (rotary_dim a multiple of 8; / 4 or / 2 else) up to a power of two, at most 64, for
 * up to five of its token's heads. */
int ds3_hip_rope(const ds3_hip_buffer_t *x, ds3_hip_type_t x_type, uint64_t x_row_stride,
                 const ds3_hip_buffer_t *positions, const ds3_hip_buffer_t *table, const ds3_hip_buffer_t *norm,
                 float eps, ds3_hip_buffer_t *out, ds3_hip_type_t out_type, uint64_t out_row_stride, uint32_t n_tokens,
                 uint32_t n_head, uint32_t head_dim, uint32_t rotary_dim, bool interleaved);

/* New tokens of a layer in one launch: q_out = q and the cache's k rows = k, both
 * normalised (q_norm, k_norm, optional) and rotated as in ds3_hip_rope, and the
 * cache's v rows = v, k and v at slots[t] (int32; a slot outside the cache: the
 * row is not written).  q, k, v are rows of `type`, their strides in bytes (of one
 * packed buffer: views); q_out is dense, or q itself where that is dense and of its
 * type.  table may be NULL: no rotation, positions (then unused) may be NULL too.  q
 * and q_out may be NULL: k and v only.  The slots of a call differ; of rows with one
 * slot it is not defined which is kept.  Values beyond F16's range become infinite in
 * the cache. */
int ds3_hip_rope_append(const ds3_hip_buffer_t *q, const ds3_hip_buffer_t *k, const ds3_hip_buffer_t *v,
                        ds3_hip_type_t type, uint64_t q_row_stride, uint64_t k_row_stride, uint64_t v_row_stride,
                        const ds3_hip_buffer_t *positions, const ds3_hip_buffer_t *slots,
                        const ds3_hip_buffer_t *table, const ds3_hip_buffer_t *q_norm, const ds3_hip_buffer_t *k_norm,
                        float eps, ds3_hip_buffer_t *q_out, ds3_hip_type_t q_out_type, ds3_hip_buffer_t *k_cache,
                        ds3_hip_buffer_t *v_cache, uint32_t n_tokens, uint32_t n_head, uint32_t n_head_kv,
                        uint32_t head_dim, uint32_t rotary_dim, bool interleaved, uint32_t n_blocks,
                        uint32_t block_size);

/* The step's plan from lengths on the device: request i has kv_lens[i] tokens in
 * the cache and new_lens[i] to come (below 0: none).  Its table row gets the blocks
 * that it lacks, taken from the end of free_blocks[0 .. n_free - 1] in the order of
 * requests (the r-th block taken is free_blocks[n_free - 1 - r]).  Written:
 *   kv_lens_out[i] = kv_lens[i] + new_lens[i], n_free_out (kv_lens and n_free
 *   themselves, or buffers of their own), q_offsets[n_seq + 1], and for each of
 *   max_tokens rows its position and slot (rows of no request: 0 and -1).
 *   status[4] = { new tokens, blocks taken, blocks lacking, requests longer than
 *   max_blocks blocks }.
 * A plan that lacks blocks, has such a request or more than max_tokens tokens is
 * not carried out: lengths, table and n_free stay, every offset is 0, every slot
 * -1.  Each of them is then safe to run the layer's calls on, which do nothing (status
 * tells the blocks that it would have taken).  free_blocks holds n_blocks entries;
 * n_free is held to 0 .. n_blocks.
 * It uses the library's workspace: before a capture the call is made once. */
int ds3_hip_kv_plan(const ds3_hip_buffer_t *new_lens, const ds3_hip_buffer_t *kv_lens, ds3_hip_buffer_t *kv_lens_out,
                    ds3_hip_buffer_t *block_table, const ds3_hip_buffer_t *free_blocks, const ds3_hip_buffer_t *n_free,
                    ds3_hip_buffer_t *n_free_out, ds3_hip_buffer_t *q_offsets, ds3_hip_buffer_t *positions,
                    ds3_hip_buffer_t *slots, ds3_hip_buffer_t *status, uint32_t n_seq, uint32_t max_blocks,
                    uint32_t n_blocks, uint32_t block_size, uint32_t max_tokens);

/* Requests with done[i] != 0 give their blocks back: the table entries of their
 * kv_lens[i] tokens go to the end of free_blocks, in the order of requests and
 * positions, n_free grows by their number and kv_lens[i] becomes 0.  Blocks that do
 * not fit (more than n_blocks in all: one was given back twice): nothing changes. */
int ds3_hip_kv_release(const ds3_hip_buffer_t *done, ds3_hip_buffer_t *kv_lens, const ds3_hip_buffer_t *block_table,
                       ds3_hip_buffer_t *free_blocks, ds3_hip_buffer_t *n_free, uint32_t n_seq, uint32_t max_blocks,
                       uint32_t n_blocks, uint32_t block_size);

/* Attention of new tokens over the paged cache, which holds their own k and v
 * already: token j of request i's m new ones is at position p = kv_lens[i] - m + j
 * and sees positions 0 .. p, or with window != 0 the last `window` of those.
 * out = softmax(scale * q . k) . v by head; q head h reads kv head h / (n_head /
 * n_head_kv).  A token that sees nothing gets zeros: one at a position below 0, or
 * whose blocks all lie outside the cache.  A value of the cache that is infinite or
 * NaN makes what it enters infinite or NaN (F32: NaN for an infinite v too) in the rows
 * that see it, and in no others; an infinite k whose score is -inf may leave its key
 * without weight instead.  Rows of out that belong to no request are left as
 * they were, as are those of a request whose rows do not lie within n_tokens.  q and
 * out are of `type`, rows of n_head heads.
 *   F32: products to 22 bits of q and of the softmax's weights (two F16 parts each),
 *        against the cache's exact F16 values
 *   F16: q as it is, the softmax's weights rounded to F16
 * Sums and the softmax are F32.  head_dim is a multiple of 8 up to 256, max_blocks *
 * block_size at most 2^31 - 2^16, scale's magnitude at most 2^127.  A call has at most
 * 2^23 - 1 tiles over all kv heads, counted as one a request and one for every 16 rows
 * (tokens times n_head / n_head_kv; 256 where a request has more than 64, 128 for heads
 * above 128): 2^20 requests of one token at seven kv heads, say.  Requests' rows do not
 * overlap (of those that do it is not defined which are written).
 * It uses the library's workspace: before a capture the call is made once. */
int ds3_hip_attention_paged(const ds3_hip_buffer_t *q, ds3_hip_type_t type, uint64_t q_row_stride,
                            const ds3_hip_buffer_t *k_cache, const ds3_hip_buffer_t *v_cache,
                            const ds3_hip_buffer_t *block_table, const ds3_hip_buffer_t *q_offsets,
                            const ds3_hip_buffer_t *kv_lens, ds3_hip_buffer_t *out, uint64_t out_row_stride,
                            uint32_t n_tokens, uint32_t n_seq, uint32_t n_head, uint32_t n_head_kv, uint32_t head_dim,
                            uint32_t n_blocks, uint32_t block_size, uint32_t max_blocks, float scale, uint32_t window);

/* One token a row from logits (F32 [n_rows][n_vocab], rows row_stride bytes apart)
 * and given random numbers: uniform[r] in 0 <= u < 1 (others are held to it).  The
 * row's tokens are ordered by logit, equal ones by index; NaN counts as -inf.
 * Weights are exp((x - largest) / temperature).  Kept are
 *   the first top_k tokens (0 or less: all), of those
 *   the shortest run whose weights reach top_p of theirs (1 or more, NaN: all), of those
 *   the ones of at least min_p times the first's weight (0 or less, NaN: all),
 * always the first one.  Drawn is the first kept token in that order at which the summed
 * weights pass u times all kept ones'.  probs[r] (optional) is its share of them.
 * temperature 0 or less or NaN, or a logit of +inf: the first token, share 1.  A row of nothing but
 * -inf and NaN: token -1, share 0.  The settings are one F32 (top_k: int32) a row;
 * NULL: temperature 1, all tokens.
 * Weights are summed in 64 bits, where only sums of many small ones matter each to
 * 2^-28 of itself, in an order that the sizes fix: the same call gives the same token.
 * (One with another number of rows does but where a sum meets u, top_p or min_p to
 * within 2^-28.)  n_vocab is at most 2^18.  It uses the library's workspace: before a
 * capture the call is made once. */
int ds3_hip_sample(const ds3_hip_buffer_t *logits, uint64_t row_stride, const ds3_hip_buffer_t *uniform,
                   const ds3_hip_buffer_t *temperature, const ds3_hip_buffer_t *top_k, const ds3_hip_buffer_t *top_p,
                   const ds3_hip_buffer_t *min_p, ds3_hip_buffer_t *tokens, ds3_hip_buffer_t *probs, uint32_t n_rows,
                   uint32_t n_vocab);

/* Router selection.  0 (default): the certified router (fp64 wavefront sums
 * with a proven error bound, exact sequential sums only where the bound
 * cannot certify the top-k order) in ds3_hip_moe_ffn and, up to 16 tokens,
 * in ds3_hip_moe_ffn_batch; the reference's sequential-order sums (logits
 * bit-identical to the reference's) everywhere else.  1: sequential-order
 * sums everywhere.  2: the certified router wherever its shape limits allow
 * (n_embd a multiple of 256 up to 4096), ds3_hip_moe_route included.
 * Returns the previous mode. */
int ds3_hip_set_router_mode(int mode);

/* Tokens the certified router has certified / repaired (exact sequential
 * sums for some candidates) since init or the last reset; synchronises. */
int ds3_hip_router_stats(uint64_t *certified, uint64_t *repaired, int reset);

/* Test hook (no ds3_metal.h counterpart): the bucketing lists the grouped
 * path of ds3_hip_moe_ffn_batch / _noalloc / ds3_hip_moe_block built on the
 * device for the last chunk of its last call -- the lists the reference's
 * host loop builds (src/ds3_engine.c:932-965) plus the grouped kernels' work
 * items and run lists.  Call it before any other library call that may reuse
 * the workspace; synchronises.  meta[DS3_HIP_LISTS_META] = { chunk's first
 * token, chunk's tokens tc, n_used k, n_expert E, work items n_tiles,
 * gate_up runs, down runs, 1 if the lists came from the routing's bitmaps
 * (else from the routed indices), gate_up runs per work item, down runs per
 * work item, max work items, tokens per work item }.  Each array not NULL
 * receives: counts[E], offsets[E + 1], ids / wts / slot_pos[tc * k],
 * tiles[n_tiles], runs_gu / runs_dn[their counts].  Work item = expert << 16
 * | token tile; run = work item index << 12 | n run.  -1 when no grouped call
 * ran since the workspace last moved. */
#define DS3_HIP_LISTS_META 12
int ds3_hip_debug_grouped_lists(int32_t *meta, int32_t *counts, int32_t *offsets, int32_t *ids, float *wts,
                                int32_t *slot_pos, int32_t *tiles, int32_t *runs_gu, int32_t *runs_dn);

/* No ds3_metal.h counterpart (a test hook, like ds3_hip_debug_grouped_lists):
 * the run descriptors the grouped kernels start each run from, entry for
 * entry with that call's runs_gu / runs_dn (their counts are meta[5] and
 * meta[6] there): two int32 per run, { first list position of the run's work
 * item, expert << 16 | the work item's rows << 8 | n run }.  Synchronises;
 * -1 when no grouped call ran since the workspace last moved. */
int ds3_hip_debug_grouped_descs(int32_t *desc_gu, int32_t *desc_dn);

/* No ds3_metal.h counterpart (a test hook): the kernel and grid that
 * ds3_hip_matmul_quantized_batch, or for M = 1 ds3_hip_vec_matmul_*, takes for
 * these arguments.  plan = { kernel (0 general, 1 one-token chunked, 2 fp32
 * MFMA, 3 fp16 MFMA), workgroups in x and y (0 for kernel 1, which sizes its
 * grid from the device), threads per workgroup, rows of A per workgroup
 * (kernel 2: blocks of 16; kernel 3 instead: sets of 128 rows of W), for
 * kernel 3 whether consecutive workgroups share rows of A and not of W }.
 * Launches nothing and needs no device; -1 for arguments that no product
 * takes. */
int ds3_hip_debug_product_plan(ds3_hip_type_t type, uint32_t M, uint32_t N, uint32_t K, uint64_t weight_row_stride,
                               uint64_t weight_offset, int64_t *plan);

/* No ds3_metal.h counterpart (a test hook): the kernel that the microscaled
 * products take for n_rows rows in n_group groups (0: ds3_hip_matmul_mx; gate_up:
 * ds3_hip_moe_gate_up_mx with N = n_ff, else ds3_hip_matmul_mx_grouped).  plan =
 * { kernel (0 few rows, 1 many), waves and rows of x a workgroup, output columns
 * a tile (gate_up: of h), tiles of output columns, how many of them a workgroup
 * takes, for kernel 1 whether its waves transpose weights beside others' work }.
 * A wave of kernel 1 takes every `waves`-th tile of its workgroup's.
 * Launches nothing and needs no device; -1 for sizes that no product takes. */
int ds3_hip_debug_mx_plan(uint32_t n_rows, uint32_t n_group, uint32_t N, uint32_t K, bool gate_up, int64_t *plan);

/* No ds3_metal.h counterpart (a test hook): how ds3_hip_attention_paged splits a
 * call, from offsets and lengths in host memory.  split = of tiles of many rows
 * (requests of more than 64), then of few: { keys a unit, tiles, units (a tile and
 * a run of its keys), units launched, tiles whose units are joined, units that the
 * workspace holds }, each of one kv head; zeros where none are launched.
 * Launches nothing and needs no device; -1 for calls that are refused. */
int ds3_hip_debug_attention_split(const int32_t *q_offsets, const int32_t *kv_lens, uint32_t n_tokens, uint32_t n_seq,
                                  uint32_t n_head, uint32_t n_head_kv, uint32_t head_dim, uint32_t block_size,
                                  uint32_t max_blocks, uint32_t window, int64_t *split);

/* No ds3_metal.h counterpart: the row count of A from which
 * ds3_hip_matmul_quantized_batch takes its fp16 MFMA path (see there).  0
 * restores the default (64).  Returns the previous value. */
int ds3_hip_set_dense_mfma_min_rows(int min_rows);

/* ds3_hip_moe_ffn_batch uses the grouped (prefill) path when
 * n_tokens >= min_tokens, the per-token GEMV path otherwise.  0 restores the
 * default.  Returns the previous value. */
int ds3_hip_set_prefill_min_tokens(int min_tokens);

/* Per-kernel timing with HIP events on the library stream.  While enabled,
 * each kernel launch is bracketed by an event pair; ds3_hip_kernel_stats
 * synchronises and reports, for kernel i (0-based; returns -1 past the end),
 * its name, launch count and summed duration in milliseconds. */
void ds3_hip_kernel_timing(int enable);
/* Restrict kernel timing to launches of the kernel called `name` (NULL or ""
 * restores timing of every kernel), so that one kernel can be timed without
 * event pairs between the others. */
void ds3_hip_kernel_timing_only(const char *name);
void ds3_hip_kernel_timing_reset(void);
int  ds3_hip_kernel_stats(int i, char *name, size_t name_len, int64_t *count, double *total_ms);

/* Occupies the library stream for `us` microseconds (0 .. 1e6) with one
 * wave that touches no memory.  Enqueued ahead of kernels timed with
 * ds3_hip_kernel_timing when the host enqueues more slowly than the GPU runs
 * them (few tokens): the held stream lets the host queue the work first, so
 * that each event pair spans its kernel and not the host's enqueue.
 * Refused during graph capture. */
int ds3_hip_hold_stream(double us);

/* Event pair on the library stream around a caller-defined region. */
int    ds3_hip_timer_start(void);
double ds3_hip_timer_stop_ms(void);

/* Device name (e.g. "gfx950"), compute-unit count and HBM bytes. */
int ds3_hip_device_info(char *arch, size_t arch_len, int *n_cu, uint64_t *hbm_bytes);

/* HIP graphs (no ds3_metal.h counterpart; for callers that replay the same
 * calls many times, such as a decode step through every layer).  The calls
 * made between graph_begin and graph_end are captured on the library's
 * stream instead of run: they wait for nothing, nothing may be read back,
 * and the library's workspace must already be large enough (make the same
 * calls once before capturing; a call that would grow it fails).  The
 * captured calls hold no memset nodes.  graph_end returns an executable
 * graph; each graph_launch replays it on the library's stream with the
 * buffers the calls named (synchronous outside begin_batch / end_batch).
 * Not allowed while in batch mode or with kernel timing on.  During a capture
 * every entry point that would allocate, free, copy from or to the host or
 * wait (buffer_alloc / from_mmap / write / read, moe_ffn_experts,
 * synchronize, end_batch, router_stats, the timers, graph_launch) returns -1
 * (or does nothing) with a diagnostic; buffer_free is deferred to graph_end.
 * A live graph (graph_end .. graph_destroy) keeps the workspace block its
 * kernels address: a later eager call that needs a larger workspace gets a
 * new block and the old one is freed when the last live graph is destroyed.
 * Buffers the captured calls named must outlive the graph.  ds3_hip_shutdown
 * destroys every live graph. */
/* Test hook for the capture refusals above: marks a capture as open (on = 1)
 * or closed (0) without a device.  Refused (-1) once ds3_hip_init has run. */
int  ds3_hip_debug_simulate_capture(int on);
int  ds3_hip_graph_begin(void);
int  ds3_hip_graph_end(void **graph);
int  ds3_hip_graph_launch(void *graph);
void ds3_hip_graph_destroy(void *graph);

#ifdef __cplusplus
}
#endif

#endif /* DS3_HIP_H */
