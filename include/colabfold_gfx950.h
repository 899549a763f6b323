/* colabfold_gfx950.h: the C ABI of the gfx950 (MI355X) ColabFold legacy-kernel library.
 *
 * One entry point per XLA FFI target of the reference. Each takes the stream, the buffers in
 * the FFI binding's order (arguments, then results) and the FFI attributes, and returns a
 * status: CLK_OK, CLK_INVALID_ARGUMENT or CLK_INTERNAL (the XLA FFI / absl error codes). The
 * message of the last failure on the calling thread is clk_last_error(). Validation runs
 * before any HIP call, so a rejected call touches no device; work is enqueued on `stream`
 * only, with no host synchronisation. No entry point allocates device memory: the backward
 * takes its scratch as a workspace argument, as the reference takes it from XLA's
 * ScratchAllocator.
 *
 * Buffers are described by clk_buffer: a device pointer, an element type (the XLA FFI
 * DataType numbering), a rank and the dimensions, exactly what an XLA_FFI_Buffer carries.
 * Optional inputs and results follow the reference: a one-element buffer plus a flag
 * (want_lse, has_keep, has_residual, n == 0, heads == 0).
 */
#ifndef COLABFOLD_GFX950_H_
#define COLABFOLD_GFX950_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* clk_stream; /* a hipStream_t; NULL is the null stream */

enum clk_dtype { CLK_S8 = 2, CLK_S32 = 4, CLK_U8 = 6, CLK_F16 = 10, CLK_F32 = 11, CLK_BF16 = 16 };

enum clk_status { CLK_OK = 0, CLK_INVALID_ARGUMENT = 3, CLK_INTERNAL = 13 };

typedef struct clk_buffer {
    void* data;
    int32_t dtype;       /* enum clk_dtype */
    int32_t rank;
    const int64_t* dims; /* rank entries, row-major, last dimension contiguous */
} clk_buffer;

/* The message of the last failed call on this thread ("" after a success). */
const char* clk_last_error(void);

/* Version of this library, e.g. "0.6.0+gfx950". */
const char* clk_version(void);

/* Measurement hook, no counterpart in the reference. With count > 0, each later entry point
 * records events[0] on its stream before its first kernel launch and events[i] after its i-th,
 * for i < count (hipEvent_t handles, owned by the caller). count 0 turns it off. The setting is
 * process-wide and meant for a single-threaded benchmark. */
int clk_set_stage_events(void* const* events, int32_t count);

/* ---- attention ------------------------------------------------------------------------ */

/* VoltaMma (reference cuda/volta_mma_attn.cu:522-542, handler 625-640).
 * q [N,H,Sq,D], k, v [N,H,Sk,D], bias [H,Sq,Sk] F16; kmask [N,Sk] U8
 * -> out [N,H,Sq,D] F16, lse [N,H,Sq] F32 (log2 domain; untouched, any size, without want_lse).
 * (D, block_q, block_k) must be one of the reference's dispatch entries (volta_mma_attn.cu:508-517). */
int clk_attention_fwd(clk_stream stream, int32_t device, const clk_buffer* q, const clk_buffer* k,
                      const clk_buffer* v, const clk_buffer* bias, const clk_buffer* kmask,
                      const clk_buffer* out, const clk_buffer* lse, float scale, int64_t block_q,
                      int64_t block_k, int32_t want_lse);

/* VoltaMmaPacked (volta_mma_attn.cu:544-583, handler 594-607): q, k, v (and the gate when
 * G == 4) read in place from p [X,Y,G,H,D]; out [X,Y,H,D]; rows attend along Y, columns
 * (column != 0) along X. bias [H,S,S], kmask [N,S], gate_bias [H,D] (any size when G == 3). */
int clk_attention_packed(clk_stream stream, int32_t device, const clk_buffer* p,
                         const clk_buffer* bias, const clk_buffer* kmask,
                         const clk_buffer* gate_bias, const clk_buffer* out, float scale,
                         int64_t block_q, int64_t block_k, int32_t column);

/* VoltaMmaPackedTrim (volta_mma_attn.cu:585-592, handler 609-623): as clk_attention_packed
 * with lims S32 [N+1] (each batch row's last live key + 1, then the largest). */
int clk_attention_packed_trim(clk_stream stream, int32_t device, const clk_buffer* p,
                              const clk_buffer* bias, const clk_buffer* kmask,
                              const clk_buffer* gate_bias, const clk_buffer* lims,
                              const clk_buffer* out, float scale, int64_t block_q,
                              int64_t block_k, int32_t column);

/* VoltaMmaBwd (reference cuda/volta_mma_attn_bwd.cu:385-451, handler 455-473).
 * q, k, v, bias F16; kmask U8; out, dout F16; lse F32 [N,H,Sq] -> dq, dk, dv F16,
 * dbias F32 [H,Sq,Sk] (the sum of dS over the N rows; all zeros without want_dbias).
 * workspace: device scratch of at least clk_attention_bwd_workspace_size() bytes, 256-byte
 * aligned; the reference takes the same kind of scratch from XLA's ScratchAllocator.
 * Results are bit-identical from run to run (no atomics). */
int clk_attention_bwd(clk_stream stream, int32_t device, const clk_buffer* q, const clk_buffer* k,
                      const clk_buffer* v, const clk_buffer* bias, const clk_buffer* kmask,
                      const clk_buffer* out, const clk_buffer* dout, const clk_buffer* lse,
                      const clk_buffer* dq, const clk_buffer* dk, const clk_buffer* dv,
                      const clk_buffer* dbias, float scale, int32_t want_dbias, void* workspace,
                      size_t workspace_bytes);

/* Bytes of workspace clk_attention_bwd needs for these shapes on this device (0 on a shape the
 * backward would reject; the call itself then reports why). */
size_t clk_attention_bwd_workspace_size(int32_t device, const clk_buffer* q, const clk_buffer* k);

/* No counterpart in the reference: clk_attention_bwd for callers that cannot allocate (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). Same buffers, flags,
 * validation and results (bit-identical), but no workspace argument: the scratch is a static
 * device array of the library, one per GPU, of clk_attention_bwd_noalloc_scratch_size() bytes
 * (96 MiB, enough for [512, 8, 384, 32]), held until the process ends. The array is part of the
 * library's code object, so loading the library reserves those 96 MiB on every GPU it runs a
 * kernel on, whether or not this entry point is ever called. Shapes whose scratch
 * would exceed it are rejected with CLK_INVALID_ARGUMENT before any launch (but at D = 32 and Sq <=
 * 384, that of the kernel with its dBias partial in LDS, whichever runs). The call allocates
 * nothing. Every call on a GPU shares that GPU's scratch, so calls that overlap on one GPU (two
 * streams, or two threads) race and must be serialised by the caller. */
int clk_attention_bwd_noalloc(clk_stream stream, int32_t device, const clk_buffer* q,
                              const clk_buffer* k, const clk_buffer* v, const clk_buffer* bias,
                              const clk_buffer* kmask, const clk_buffer* out,
                              const clk_buffer* dout, const clk_buffer* lse, const clk_buffer* dq,
                              const clk_buffer* dk, const clk_buffer* dv, const clk_buffer* dbias,
                              float scale, int32_t want_dbias);

/* Bytes of the static scratch behind clk_attention_bwd_noalloc. */
size_t clk_attention_bwd_noalloc_scratch_size(void);

/* Diagnostic, no counterpart in the reference: the backward's launch plan for these shapes on
 * this device, plan[0..count) = {row groups per dK/dV workgroup, batch rows per workgroup
 * (chunk), chunks, row passes per workgroup, query windows, 1 where the dK/dV kernel keeps its
 * dBias partial in registers (D <= 32 only), 0 where in LDS}. */
int clk_attention_bwd_plan(int32_t device, int64_t N, int64_t H, int64_t Sq, int64_t Sk,
                           int64_t D, int64_t* plan, int32_t count);

/* ---- LayerNorm-fused pair-stack projections (reference cuda/volta_fused_ffi.h) --------- */

/* Activation types, an addition to the reference (whose handlers bind F16 only): the activation
 * buffers of each entry point below (x, o, residual and every activation result: left, right,
 * out, p, bias) may be BF16 instead of F16, all together; weights, biases and keep stay F16 and
 * LayerNorm parameters F32. A BF16 input is read exactly into fp32, the LayerNorm output (and
 * o, and the transition's hidden activation) enter the matrix cores as fp16, and the results
 * are rounded to BF16 once. A mix of F16 and BF16 activations is CLK_INVALID_ARGUMENT. The XLA
 * FFI handlers keep the reference's F16-only binding. */

/* VoltaLnGdp (volta_fused_ffi.h:42-80, handler 337-351): left, right [P/2, M] = the two halves
 * of max(mask,0) * (y@wp + bp) * sigmoid(y@wg + bg), channel major, y = LN(x).
 * x [M,K] F16; scale, offset [K] F32; wpT [P,K], bp [P], wgT [P,K], bg [P], mask [M] F16.
 * K and P/2 in {64, 128}. The mask is also the row-tile keep. */
int clk_ln_gdp(clk_stream stream, const clk_buffer* x, const clk_buffer* scale,
               const clk_buffer* offset, const clk_buffer* wpT, const clk_buffer* bp,
               const clk_buffer* wgT, const clk_buffer* bg, const clk_buffer* mask,
               const clk_buffer* left, const clk_buffer* right, float eps);

/* VoltaTrimulEpilogue (volta_fused_ffi.h:82-133, handler 353-371):
 * out [M,O] = (LN(x_cm.T)@wo + bo) * sigmoid(LN_in(x)@wg + bg) [+ x with add_input].
 * x_cm [C,M] F32; x [M,CA] F16; in_scale, in_offset [CA], ln_scale, ln_offset [C] F32;
 * woT [O,C], bo [O], wgT [O,CA], bg [O], keep [M] (or any size without has_keep) F16.
 * C, CA, O in {64, 128}; O == CA with add_input (then out may alias x). */
int clk_trimul_epilogue(clk_stream stream, const clk_buffer* x_cm, const clk_buffer* x,
                        const clk_buffer* in_scale, const clk_buffer* in_offset,
                        const clk_buffer* ln_scale, const clk_buffer* ln_offset,
                        const clk_buffer* woT, const clk_buffer* bo, const clk_buffer* wgT,
                        const clk_buffer* bg, const clk_buffer* keep, const clk_buffer* out,
                        float eps, int32_t add_input, int32_t has_keep);

/* VoltaLnProj (volta_fused_ffi.h:135-176, handler 373-388): p [M,n] = LN(x)@w and
 * bias [heads,M] = (LN(x)@wb).T. x [M,K] F16 (K in {64,128}); scale, offset [K] F32;
 * wT [n,K], wbT [heads,K], keep [M] F16. n a multiple of 64 (0: p untouched), heads <= 8
 * (0: bias untouched). */
int clk_ln_projection(clk_stream stream, const clk_buffer* x, const clk_buffer* scale,
                      const clk_buffer* offset, const clk_buffer* wT, const clk_buffer* wbT,
                      const clk_buffer* keep, const clk_buffer* p, const clk_buffer* bias,
                      float eps, int64_t n, int64_t heads, int32_t has_keep);

/* VoltaOutProj (volta_fused_ffi.h:178-214, handler 390-401): out [M,N] = o@w + b
 * [+ residual]. o [M,K], wT [N,K], b [N], residual [M,N], keep [M] F16; K, N in {64,128}.
 * With has_residual out may alias residual. */
int clk_output_projection(clk_stream stream, const clk_buffer* o, const clk_buffer* wT,
                          const clk_buffer* b, const clk_buffer* residual, const clk_buffer* keep,
                          const clk_buffer* out, int32_t has_residual, int32_t has_keep);

/* VoltaTransition (volta_fused_ffi.h:216-259, handler 403-418): out [M,C] =
 * relu(LN(x)@w1 + b1)@w2 + b2 [+ x]. x [M,C] F16 (C in {64,128,256}); scale, offset [C] F32;
 * w1T [H,C], b1 [H], w2T [H/64][C][64] (w2T[j][c][i] = w2[64j+i][c]), b2 [C], keep [M] F16;
 * H in {2C, 4C}. With add_input out may alias x. */
int clk_transition(clk_stream stream, const clk_buffer* x, const clk_buffer* scale,
                   const clk_buffer* offset, const clk_buffer* w1T, const clk_buffer* b1,
                   const clk_buffer* w2T, const clk_buffer* b2, const clk_buffer* keep,
                   const clk_buffer* out, float eps, int32_t add_input, int32_t has_keep);

/* ---- unfused pair-stack ops (reference cuda/volta_ops.cu) ------------------------------ */

/* VoltaLayerNorm (volta_ops.cu:27-84, handler 86-94): out [M,C] = LN(x) over the last axis with
 * one-pass fp32 statistics (var = max(E[x^2] - mean^2, 0)). x [M,C] F16; scale, offset [C] F32;
 * out [M,C] F16. */
int clk_layer_norm(clk_stream stream, const clk_buffer* x, const clk_buffer* scale,
                   const clk_buffer* offset, const clk_buffer* out, float eps);

/* VoltaGdp (volta_ops.cu:97-256, handler 258-269): out [M,N] = mask * (x@wp + bp) *
 * act(x@wg + bg), act = sigmoid (activation 0) or swish (1). x [M,K]; wp, wg [K,N] row-major;
 * bp, bg [N]; mask [M]; all F16. N a multiple of 8. */
int clk_gated_dual_proj(clk_stream stream, int32_t device, const clk_buffer* x,
                        const clk_buffer* wp, const clk_buffer* bp, const clk_buffer* wg,
                        const clk_buffer* bg, const clk_buffer* mask, const clk_buffer* out,
                        int64_t activation);

/* ---- outer product mean (reference cuda/volta_ops.cu) ---------------------------------- */

/* VoltaOpmUpdate (volta_ops.cu:643-704, handler cuda/volta_fused_ffi.h:261-297, 420-431):
 * out[b,d,:] = fp16((lhs[b] @ t[:,d,:] + bias) / (eps + norm[b,d]) [+ residual[b,d,:]]), fp32
 * accumulation. lhs [B,K], t [K,D,F], residual [B,D,F] F16 (read only with has_residual; may
 * alias out); bias [F], norm [B,D] F32; out [B,D,F] F16. K a multiple of 32, F in
 * {16,32,64,128}, D at most 65535. */
int clk_opm_update(clk_stream stream, const clk_buffer* lhs, const clk_buffer* t,
                   const clk_buffer* bias, const clk_buffer* norm, const clk_buffer* residual,
                   const clk_buffer* out, float eps, int32_t has_residual);

/* VoltaOpmOuter (volta_ops.cu:706-792, handler volta_fused_ffi.h:299-335, 433-440):
 * out[b,d,f] = fp16(sum_c sum_e fp16(sum_a left[a,b,c] right[a,d,e]) wT[f, c E + e]) over the
 * 16 rows a. left [16,B,C], right [16,D,E=32], wT [F,C*E], out [B,D,F], all F16. C a multiple of
 * 16, D a multiple of 4 (D/4 at most 65535), F in {16,32,64,128}. */
int clk_opm_outer(clk_stream stream, const clk_buffer* left, const clk_buffer* right,
                  const clk_buffer* wT, const clk_buffer* out);

/* ---- RMS norm and 8-bit rows (no counterpart in the reference) ------------------------- */

/* Activations (x, residual, sum, s, dout, dsum, ds, and out where it is 16-bit) are F16 or BF16, all of
 * a call's one type. An absent optional buffer is any buffer of its type, unread and unwritten.
 *
 * 8-bit rows are a pair: q [R,Kp] S8 and scale [R] F32, with Kp = K rounded up to a multiple of 64 and
 * the columns past K zero; column k of row r stands for q[r,k] * scale[r]. A row is quantised by its
 * largest magnitude a: q = 127 t / a to the nearest integer (ties to even) and scale = a / 127, so q lies
 * in -127..127. A row whose a is under 2^-119 (its scale would leave fp32's normal range) is all
 * zeros with scale 0; a row that holds an infinity or NaN is all zeros with scale NaN. (A norm's bf16 row
 * of values under 2^-40 with eps under 2^-100, which is taken times 2^90, is zeros under 2^-209 only.) */

/* out [M,C] = s / sqrt(mean(s^2) + eps) * scale over the last axis, with s = x, or with has_residual
 * s = x + residual rounded to the activation type, which is also written to sum [M,C] (the residual
 * stream). scale [C] F32; rstd [M] F32 receives 1 / sqrt(mean(s^2) + eps) with want_rstd, for the
 * backward. C at least 1. sum may alias x or residual, and out either of them,
 * but not sum. */
int clk_rms_norm(clk_stream stream, const clk_buffer* x, const clk_buffer* residual,
                 const clk_buffer* scale, const clk_buffer* sum, const clk_buffer* out,
                 const clk_buffer* rstd, float eps, int32_t has_residual, int32_t want_rstd);

/* The same norm with its result as 8-bit rows: q [M,Kp] S8, q_scale [M] F32. The rounding to 8 bits is
 * the only one: s * scale is quantised from fp32, and q_scale carries 1 / sqrt(mean(s^2) + eps). */
int clk_rms_norm_q8(clk_stream stream, const clk_buffer* x, const clk_buffer* residual,
                    const clk_buffer* scale, const clk_buffer* sum, const clk_buffer* q,
                    const clk_buffer* q_scale, float eps, int32_t has_residual);

/* Gradients of clk_rms_norm: s [M,C] (x, or the forward's sum), scale [C], rstd [M], dout [M,C] and, with
 * has_dsum, the gradient of sum, dsum [M,C] -> ds [M,C] = rstd (g - xh mean(g xh)) + dsum with xh =
 * s rstd and g = dout scale (the gradient of x and of residual alike), dscale [C] F32 = the sum over the
 * M rows of dout xh (zeros for M = 0). C at most 2^27. ds may alias dout or dsum. workspace: device scratch of at least
 * clk_rms_norm_bwd_workspace_size() bytes, 256-byte aligned, not shared by two calls in flight.
 * Bit-identical from run to run (no atomics). */
int clk_rms_norm_bwd(clk_stream stream, const clk_buffer* s, const clk_buffer* scale,
                     const clk_buffer* rstd, const clk_buffer* dout, const clk_buffer* dsum,
                     const clk_buffer* ds, const clk_buffer* dscale, int32_t has_dsum,
                     void* workspace, size_t workspace_bytes);

/* Bytes of workspace clk_rms_norm_bwd needs for s [M,C] (0 on a shape that it would reject). */
size_t clk_rms_norm_bwd_workspace_size(const clk_buffer* s);

/* 8-bit rows q [M,Kp], q_scale [M] of h [M,K]: activation 0: h = x [M,K]; 1: h = relu(x); 2: h =
 * swish(x[:, :K]) x[:, K:] with x [M,2K], swish(g) = g / (1 + exp(-g)). x F16, BF16 or F32; h is held in
 * fp32. The same entry point quantises activations by token and weights wT [N,K] by output channel. */
int clk_quantize_rows(clk_stream stream, const clk_buffer* x, const clk_buffer* q,
                      const clk_buffer* q_scale, int64_t activation);

/* out [M,K] (F16, BF16 or F32) = what the 8-bit rows q [M,Kp], q_scale [M] stand for. */
int clk_dequantize_rows(clk_stream stream, const clk_buffer* q, const clk_buffer* q_scale,
                        const clk_buffer* out);

/* out [M,N] = (q w^T) * q_scale[m] * w_scale[n] [+ b[n]] [+ residual[m,n]], the products of 8-bit
 * integers summed exactly in 32 bits. q [M,Kp] S8, q_scale [M] F32: 8-bit rows; wq S8
 * [ceil(N/64), Kp/64, 4, 4, 16, 16]: the rows of 8-bit weights [N,Kp] in blocks of 64 channels by 64
 * inputs, entry [., ., b, c, 4 g + i, j] being channel 16 g + 4 b + i, input 16 c + j of its block, zeros
 * for channels past N; w_scale [N], b [N] F32; residual, out [M,N] F16 or BF16, one type. Kp at most
 * 131008. out may alias residual. */
int clk_q8_projection(clk_stream stream, const clk_buffer* q, const clk_buffer* q_scale,
                      const clk_buffer* wq, const clk_buffer* w_scale, const clk_buffer* b,
                      const clk_buffer* residual, const clk_buffer* out, int32_t has_b,
                      int32_t has_residual);

/* ---- heads, the key-value cache and its attention (no counterpart in the reference) ------ */

/* Activations (qkv, q, k, v, out and the gradients) are F16 or BF16, all of a call's one type, their buffers 16-byte
 * aligned.
 *
 * A cache is a pair of buffers k_cache, v_cache [pages,heads,page,D], D a multiple of 32 up to 256 and page, the tokens of a
 * page, a multiple of 16: of the activations' type, or S8 with k_scale, v_scale [pages,heads,page] F32 (for 16 bits any F32
 * buffers, unread and unwritten). Token s % page of page s / page is slot s, and a cache holds fewer than 2^31. An 8-bit
 * cache holds each token's head as an 8-bit row. Within a page's head, blocks of 16 tokens lie one after another:
 *   keys    [D / W][16][W], W = 8 (16-bit) or 16 (8-bit) channels
 *   values  [D / (16 C)][4][16][C][4]: token 4 g + j, channel 16 (C b + e) + i at [b][g][i][e][j], C = 2, or 4 for 8 bits
 *           where D is a multiple of 64 */

/* The queries, keys and values of a projection, qkv [T,Hq+2*Hkv,D] (query heads, then keys', then values'), apart and ready
 * for attention: q [T,Hq,D], k and v [T,Hkv,D]. Each query and key head n = x / sqrt(mean(x^2) + eps) * w, w = q_norm or
 * k_norm [D] F32, and its first R channels rotated by the angles of the token's position: pairs (a, b) = channels (i, i +
 * R/2), or with interleaved (2 i, 2 i + 1), become (a cos - b sin, a sin + b cos), rounded once. Values are copied. rope [P,R] F32: the
 * cosines of a position's R/2 angles, then their sines; positions [T] S32. A token whose position the table does not have
 * gets NaN for its queries and keys. D and R multiples of 8, D up to 256, R up to D. */
int clk_qk_norm_rope(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm,
                     const clk_buffer* k_norm, const clk_buffer* rope, const clk_buffer* positions,
                     const clk_buffer* q, const clk_buffer* k, const clk_buffer* v, float eps,
                     int32_t interleaved);

/* Its gradients: dq [T,Hq,D], dk, dv [T,Hkv,D] -> dqkv [T,Hq+2*Hkv,D] and dq_norm, dk_norm [D] F32, the sums over tokens and
 * heads (zeros for T = 0). workspace: device scratch of at least clk_qk_norm_rope_bwd_workspace_size() bytes, 256-byte
 * aligned, not shared by two calls in flight. Bit-identical from run to run (no atomics). */
int clk_qk_norm_rope_bwd(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm,
                         const clk_buffer* k_norm, const clk_buffer* rope,
                         const clk_buffer* positions, const clk_buffer* dq, const clk_buffer* dk,
                         const clk_buffer* dv, const clk_buffer* dqkv, const clk_buffer* dq_norm,
                         const clk_buffer* dk_norm, float eps, int32_t interleaved,
                         void* workspace, size_t workspace_bytes);

/* Bytes of workspace clk_qk_norm_rope_bwd needs (0 on shapes that it would reject). */
size_t clk_qk_norm_rope_bwd_workspace_size(const clk_buffer* qkv, const clk_buffer* dk);

/* clk_qk_norm_rope with keys and values written into the cache, token t at slot slots[t] (S32 [T]), and q [T,Hq,D] beside.
 * Keys of an 8-bit cache are quantised from fp32. A token whose slot the cache does not have (a negative one, as in
 * the rows of a padded batch) writes nothing there. Two tokens of a call must not have the same slot: what it
 * holds afterwards may be of either, value by value. */
int clk_qk_norm_rope_cache(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm,
                           const clk_buffer* k_norm, const clk_buffer* rope,
                           const clk_buffer* positions, const clk_buffer* slots,
                           const clk_buffer* q, const clk_buffer* k_cache,
                           const clk_buffer* v_cache, const clk_buffer* k_scale,
                           const clk_buffer* v_scale, float eps, int32_t interleaved);

/* k, v [T,heads,D] into the cache as they are, token t at slot slots[t], with the rules of clk_qk_norm_rope_cache. */
int clk_kv_cache_write(clk_stream stream, const clk_buffer* k, const clk_buffer* v,
                       const clk_buffer* slots, const clk_buffer* k_cache,
                       const clk_buffer* v_cache, const clk_buffer* k_scale,
                       const clk_buffer* v_scale);

/* k, v [T,heads,D] = what the slots hold, zeros for a slot that the cache does not have; 8-bit rows in k's type. A slot may
 * be read any number of times. */
int clk_kv_cache_read(clk_stream stream, const clk_buffer* k_cache, const clk_buffer* v_cache,
                      const clk_buffer* k_scale, const clk_buffer* v_scale, const clk_buffer* slots,
                      const clk_buffer* k, const clk_buffer* v);

/* One new token's attention for each of B sequences: out [B,Hq,D] = softmax(scale q K^T) V over the first lengths[b] tokens of
 * the pages page_table[b,:], query head h on the cache's head h / (Hq / heads). q [B,Hq,D]; page_table [B,N], lengths [B] S32;
 * lse [B,Hq] F32 (with want_lse) = log2 of the sum of exp(scale q k), in the log2 domain. Statistics and sums are fp32. A
 * sequence of no tokens (or a negative length) gives zeros, and -inf as lse. Entries of page_table past a sequence's last
 * token are not read; a page among the others that the cache does not have, or a length past N pages, makes the
 * sequence's results NaN. What pages hold past the last token does not matter. workspace: device scratch of at
 * least clk_paged_attention_workspace_size() bytes, 256-byte aligned, not shared by two calls in flight.
 * Bit-identical from run to run. */
int clk_paged_attention(clk_stream stream, const clk_buffer* q, const clk_buffer* k_cache,
                        const clk_buffer* v_cache, const clk_buffer* k_scale,
                        const clk_buffer* v_scale, const clk_buffer* page_table,
                        const clk_buffer* lengths, const clk_buffer* out, const clk_buffer* lse,
                        float scale, int32_t want_lse, void* workspace, size_t workspace_bytes);

/* Bytes of workspace clk_paged_attention needs (0 where it needs none, and on shapes that it would reject). */
size_t clk_paged_attention_workspace_size(const clk_buffer* q, const clk_buffer* k_cache,
                                          const clk_buffer* page_table);

#ifdef __cplusplus
}
#endif

#endif /* COLABFOLD_GFX950_H_ */
