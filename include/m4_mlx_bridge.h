/*
 * m4_mlx_bridge.h -- C-ABI of the MI355X quantization-router prefill path.
 *
 * Drop-in for the reference's core/bridge/m4_mlx_bridge.h:23-106: the same
 * eight entry points with the same argument meaning, return values and
 * validation order, exported from libm4_bridge.so.  Pointers are DEVICE
 * pointers (hipMalloc / torch-ROCm data_ptr()); host pointers are accepted
 * too and staged through device memory (slower, PCIe-bound).  Kernels run
 * on the bridge stream (m4_bridge_set_stream) asynchronously;
 * m4_bridge_synchronize() waits for everything issued so far.
 *
 * Error codes (checked in this order, before any device work,
 * core/bridge/m4_mlx_bridge.mm:201-230):
 *   -1 bridge not initialized
 *   -2 null pointer, odd (non-2-byte-aligned) X or Y, or a buffer too small
 *   -3 invalid format (the projection entry points accept ids 0..5)
 *   -4 invalid dimension: M, K or N zero; K % 32; K % 256 for formats 2, 4, 5
 *   -5 device staging allocation failed
 *   -6 kernel launch / device failure
 *
 * The entry points below the first block have no single counterpart in the
 * reference's C-ABI; each names the reference routine it replaces.
 */
#ifndef M4_MLX_BRIDGE_H
#define M4_MLX_BRIDGE_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define M4_API __attribute__((visibility("default")))
#else
#define M4_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ---- reference C-ABI (core/bridge/m4_mlx_bridge.h) ---------------------- */

/* m4_mlx_bridge.h:23 -- selects the HIP device, creates the bridge stream.
 * The path argument is accepted for compatibility and ignored (kernels are
 * compiled into the library). */
M4_API bool m4_bridge_init(const char* metallib_path);

/* m4_mlx_bridge.h:33 -- minimum W bytes for format 0..5, else 0. */
M4_API size_t m4_bridge_get_expected_weight_bytes(int format, uint32_t K, uint32_t N);

/* m4_mlx_bridge.h:57 -- Y[M,N] (fp16) = X[M,K] (fp16) . W^T, W packed [N, K]. */
M4_API int m4_bridge_dispatch_gemm(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes, void* Y_ptr,
                            size_t Y_bytes, int format, uint32_t M, uint32_t K, uint32_t N);

/* m4_mlx_bridge.h:79 -- GEMM with M = 1 (m4_mlx_bridge.mm:293-302). */
M4_API int m4_bridge_dispatch_gemv(void* x_ptr, size_t x_bytes, void* W_ptr, size_t W_bytes, void* y_ptr,
                            size_t y_bytes, int format, uint32_t K, uint32_t N);

/* m4_mlx_bridge.h:90 -- waits for all work issued on the bridge stream. */
M4_API void m4_bridge_synchronize(void);

/* m4_mlx_bridge.h:96 -- process footprint in MB: host resident set plus the
 * device memory the bridge itself holds. */
M4_API double m4_bridge_get_uma_footprint_mb(void);

/* m4_mlx_bridge.h:101 */
M4_API bool m4_bridge_is_initialized(void);

/* m4_mlx_bridge.h:106 -- waits, releases staging memory and the stream. */
M4_API void m4_bridge_shutdown(void);

/* ---- extensions: same router, other reference routines ------------------ */

/* Validation only: the code m4_bridge_dispatch_gemm would return for these
 * arguments on an initialized bridge (0 if it would launch), computed without
 * touching a device (m4_mlx_bridge.mm:204-230). */
M4_API int m4_bridge_validate_gemm(const void* X_ptr, size_t X_bytes, const void* W_ptr, size_t W_bytes,
                            const void* Y_ptr, size_t Y_bytes, int format, uint32_t M, uint32_t K,
                            uint32_t N);

/* Projection for every format with a kernel: formats 0..5 as
 * m4_bridge_dispatch_gemm, plus PRISM_Q2_0 (7; K % 128 == 0) and Q8_0 weights
 * (6).  Replaces the registry's kernels reached by name,
 * quant_router_gemm_<fmt>_64x64 (quant_router_kernels.metal:588-750,
 * prism_q2_0 at :726; names from src/router/quant_registry.mm:60-172 --
 * quant_router_gemm_q8_0_64x64 is named there but has no Metal kernel).
 * Same validation order and codes as dispatch_gemm with the wider format set. */
M4_API int m4_bridge_dispatch_router_gemm(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes, void* Y_ptr,
                                   size_t Y_bytes, int format, uint32_t M, uint32_t K, uint32_t N);

/* Direct-head projection: Y is [H, M, D] with N = H * D; replaces
 * quant_router_head_gemm_<fmt>_64x64 (quant_router_kernels.metal:754-927,
 * index map :570-574).  Same validation as dispatch_router_gemm with N = H * D
 * (formats 0..7). */
M4_API int m4_bridge_dispatch_head_gemm(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes, void* Y_ptr,
                                 size_t Y_bytes, int format, uint32_t M, uint32_t H, uint32_t D,
                                 uint32_t K);

/* A router kernel by its Metal pipeline name, with that kernel's buffer and
 * constant slots: A = X (buffer 0), B = W (1), C = Y (2), and dims = the
 * constants from slot 3 on -- {M, N, K} for quant_router_gemm_<fmt>_64x64
 * (quant_router_kernels.metal:588-750) and {M, H, D, K} for
 * quant_router_head_gemm_<fmt>_64x64 (:754-927); kernel names as listed by the
 * registry (src/router/quant_registry.mm:60-172).  The vector-ALU ternary
 * kernels quant_router_gemm_ternary_1_58_vec (:934-1064) and
 * quant_router_head_gemm_ternary_1_58_vec (:1067-1201) compute the same
 * projection and run the matrix-core path here.  Returns -3 for an unknown
 * name, -4 when ndims does not match the kernel's constant slots, otherwise
 * what dispatch_router_gemm / dispatch_head_gemm return. */
M4_API int m4_bridge_dispatch_router_kernel(const char* kernel_name, void* X_ptr, size_t X_bytes, void* W_ptr,
                                            size_t W_bytes, void* Y_ptr, size_t Y_bytes, const uint32_t* dims,
                                            uint32_t ndims);

/* Projection with a fused residual: Y = fp16(X . W^T + R), R fp16 [M, N];
 * replaces a GEMM followed by vector_add_residual (unified_kernels.metal:
 * 78-88; unified_prefill_engine.mm:183-186).  Y may alias R. */
M4_API int m4_bridge_dispatch_gemm_residual(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes,
                                     void* R_ptr, size_t R_bytes, void* Y_ptr, size_t Y_bytes,
                                     int format, uint32_t M, uint32_t K, uint32_t N);

/* Fused dual-projection SwiGLU: Out[M, N_mlp] = silu(X . Wg^T) * (X . Wu^T);
 * replaces swiglu_mma_dual_simd (brick3_swiglu_kernels.metal:428-698), which
 * takes Q4_0 only; any format with kernels (0..7) is accepted here. */
M4_API int m4_bridge_dispatch_swiglu(void* X_ptr, size_t X_bytes, void* Wg_ptr, size_t Wg_bytes, void* Wu_ptr,
                              size_t Wu_bytes, void* Out_ptr, size_t Out_bytes, int format, uint32_t M,
                              uint32_t N_mlp, uint32_t K);

/* Q8_0 quantization of num_blocks groups of 32 fp16 values into 34-byte
 * blocks; replaces quantize_kv_to_q8_0 (unified_kernels.metal:118-145). */
M4_API int m4_bridge_quantize_kv_q8_0(void* src_ptr, size_t src_bytes, void* dst_ptr, size_t dst_bytes,
                               uint64_t num_blocks);

/* Causal flash attention over a Q8_0 KV cache; replaces
 * flash_attn_mma_64x64_q8_0_d64/_d128 (brick4_attn_kernels.metal:868-911).
 * Q fp16 [H, M, D]; K_q8, V_q8 Q8_0 blocks over [H, M, D]; D in {64, 128}.
 * O fp16 [H, M, D] (o_token_major = 0) or [M, H * D] (o_token_major = 1). */
M4_API int m4_bridge_dispatch_flash_attn_q8_0(void* Q_ptr, size_t Q_bytes, void* Kq_ptr, size_t Kq_bytes,
                                       void* Vq_ptr, size_t Vq_bytes, void* O_ptr, size_t O_bytes,
                                       uint32_t H, uint32_t M, uint32_t D, float scale,
                                       int o_token_major);

/* One prefill layer (no norm, no RoPE), composed as the reference's
 * TransformerLayerCoordinator::forward (models/transformer_layer.mm:75-218)
 * with the Q8_0 KV cache of unified_prefill_engine.mm:554-572:
 *   Q,K,V head GEMMs -> Q8_0(K,V) -> flash attention -> O-proj + residual ->
 *   fused SwiGLU -> down-proj + residual.
 * X, X_out fp16 [M, d_model]; Wq/Wk/Wv [H*D, d_model], Wo [d_model, H*D],
 * Wg/Wu [N_mlp, d_model], Wd [d_model, N_mlp], all in `format`.  Scratch is
 * held by the bridge.  X_out must not alias X. */
M4_API int m4_bridge_prefill_layer(void* X_ptr, void* Wq, void* Wk, void* Wv, void* Wo, void* Wg, void* Wu,
                            void* Wd, void* X_out, int format, uint32_t M, uint32_t d_model, uint32_t H,
                            uint32_t D, uint32_t N_mlp, float attn_scale);

/* Grouped-query variant: K/V carry Hkv heads ([Hkv, M, D] Q8_0 blocks) and
 * query head h reads KV head h / (H / Hkv) (H % Hkv == 0), as the MLX block
 * passes them to scaled_dot_product_attention (src/engine/model.py:234-236).
 * Hkv == H is m4_bridge_dispatch_flash_attn_q8_0. */
M4_API int m4_bridge_dispatch_flash_attn_q8_0_gqa(void* Q_ptr, size_t Q_bytes, void* Kq_ptr, size_t Kq_bytes,
                                           void* Vq_ptr, size_t Vq_bytes, void* O_ptr, size_t O_bytes,
                                           uint32_t H, uint32_t Hkv, uint32_t M, uint32_t D, float scale,
                                           int o_token_major);

/* RMSNorm of the MLX block (src/engine/model.py:17-48) over rows of X [M, D]
 * (D % 8 == 0): Y = fp16(fp16(x / sqrt(mean(x^2) + eps)) * w) for norm_type 1
 * ("rmsnorm"), with fp16(1 + w) in place of w for norm_type 2
 * ("gemma_add_one").  W fp16 [D].  Codes: -1, -2 (null / short buffers),
 * -3 (norm_type), -4 (dims), -5, -6 as dispatch_gemm. */
M4_API int m4_bridge_rmsnorm(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes, void* Y_ptr,
                      size_t Y_bytes, uint32_t M, uint32_t D, float eps, int norm_type);

/* Rotary position embedding in place on T [H, M, D] (D % 16 == 0): nn.RoPE
 * (dims = D, traditional, base = theta) applied at positions offset + m
 * (src/engine/model.py:112-116, :215-226).  Pairs (i, i + D/2), or (2i, 2i + 1)
 * when traditional, rotate by (offset + m) theta^(-2i/D). */
M4_API int m4_bridge_rope(void* T_ptr, size_t T_bytes, uint32_t H, uint32_t M, uint32_t D, float theta,
                   uint32_t offset, int traditional);

/* The MLX transformer block (src/engine/model.py:181-265) on the router's
 * kernels: RMSNorm(X, w_attn) -> Q [Hq], K, V [Hkv] head GEMMs -> RoPE(Q, K)
 * -> Q8_0(K, V) -> grouped-query flash attention -> O-proj + residual ->
 * RMSNorm(w_ffn) -> fused SwiGLU -> down-proj + residual.  w_attn / w_ffn
 * fp16 [d_model] or NULL (no norm); rope = 0 skips RoPE.  Wq [Hq*D, d_model],
 * Wk/Wv [Hkv*D, d_model], Wo [d_model, Hq*D], Wg/Wu [N_mlp, d_model],
 * Wd [d_model, N_mlp].  Device pointers, 16-byte aligned; X_out must not
 * alias X.  Hkv == Hq, no norms, no RoPE is m4_bridge_prefill_layer. */
M4_API int m4_bridge_prefill_layer_ex(void* X_ptr, void* w_attn, void* Wq, void* Wk, void* Wv, void* Wo,
                               void* w_ffn, void* Wg, void* Wu, void* Wd, void* X_out, int format,
                               uint32_t M, uint32_t d_model, uint32_t Hq, uint32_t Hkv, uint32_t D,
                               uint32_t N_mlp, float attn_scale, int norm_type, float norm_eps, int rope,
                               float rope_theta, uint32_t rope_offset, int rope_traditional);

/* m4_bridge_prefill_layer_ex that also hands back the layer's Q8_0 KV cache
 * (the d_K_q8 / d_V_q8 buffers of unified_prefill_engine.mm:548-572): Kq_out
 * and Vq_out, device memory of Hkv * M * D / 32 * 34 bytes each, receive the
 * Q8_0 blocks of K and V ([Hkv, M, D], 32 consecutive d per 34-byte block,
 * K after RoPE).  Both NULL: m4_bridge_prefill_layer_ex; only one: -2. */
M4_API int m4_bridge_prefill_layer_ex_kv(void* X_ptr, void* w_attn, void* Wq, void* Wk, void* Wv, void* Wo,
                                  void* w_ffn, void* Wg, void* Wu, void* Wd, void* X_out, void* Kq_out,
                                  void* Vq_out, int format, uint32_t M, uint32_t d_model, uint32_t Hq, uint32_t Hkv,
                                  uint32_t D, uint32_t N_mlp, float attn_scale, int norm_type, float norm_eps,
                                  int rope, float rope_theta, uint32_t rope_offset, int rope_traditional);

/* Dequantize W [N, K] to fp16 [N, K] with the kernels' own decoders (the
 * registry's dequantize hook, src/router/quant_registry.h:24). Formats 0..7. */
M4_API int m4_bridge_dequantize(void* W_ptr, size_t W_bytes, void* out_ptr, size_t out_bytes, int format,
                         uint32_t K, uint32_t N);

/* No counterpart in the reference.  For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): m4_bridge_dispatch_gemm's projection with the same
 * arguments, validation and results, but its split-K partials live in a
 * fixed 32 MiB device scratch array of the library (one per GPU, held until
 * the process ends) and no device memory is allocated or freed.  X, W and Y
 * must be device memory (X and W 16-byte aligned): -2 otherwise, since host
 * or misaligned buffers would need staging copies.  -4 when the shape needs
 * more split-K partials than the scratch holds (ksplit * M * N <= 8 Mi
 * floats: every tiled launch fits; small-M launches with long K and wide N,
 * e.g. M = 48, K = 16384, N = 12288, do not).  Calls on one GPU share the scratch: calls
 * that overlap in time (other streams, other threads' streams) race. */
M4_API int m4_bridge_dispatch_gemm_noalloc(void* X_ptr, size_t X_bytes, void* W_ptr, size_t W_bytes, void* Y_ptr,
                                           size_t Y_bytes, int format, uint32_t M, uint32_t K, uint32_t N);

/* No counterpart in the reference: which kernel a projection of [M, K]
 * activations runs here, from the same choice that the dispatches make (host
 * arithmetic only, no GPU and no initialization needed).  N holds the widths of
 * `groups` projections launched together (1, or 3 for a layer's Q, K and V);
 * `swiglu`: the fused gate and up projection.  0, -2 (null), -3 (format), -4. */
enum { M4_KERNEL_FEW_ROWS = 0, M4_KERNEL_SMALL_M = 1, M4_KERNEL_TILED = 2, M4_KERNEL_WIDE = 3 };
typedef struct {
    int kernel;                   /* M4_KERNEL_* */
    uint32_t tile_rows, tile_cols; /* outputs of one workgroup */
    uint32_t k_groups;            /* K groups inside a workgroup */
    uint32_t k_splits;            /* K splits over workgroups (> 1: a reduction kernel follows) */
} m4_projection_plan_t;
M4_API int m4_bridge_projection_plan(int format, uint32_t M, uint32_t K, const uint32_t* N, uint32_t groups, int swiglu,
                                     m4_projection_plan_t* plan);

/* ---- serving: a paged, quantized KV cache, read and written by batches of
 *      sequences of any lengths.  No counterpart in the reference, whose cache
 *      is one prompt's ([Hkv, M, D] Q8_0 blocks).  All buffers are device
 *      memory of the stream's device; nothing is staged, allocated or waited
 *      for, so every call can be captured into a graph.  A call's outputs do
 *      not overlap its other buffers, but where one may be the other. ------ */

/* A cache of num_pages pages of page_size tokens (16, 32, 64, 128 or 256),
 * Hkv heads, D = 64 or 128, in format QUANT_Q8_0 (6) or QUANT_Q4_0 (0), one
 * fp16 scale per 32 dims of a token.  A page holds, for each head, K codes
 * [page_size][D], V codes [page_size / 4][D][4 tokens], K scales
 * [page_size][D / 32], V scales [page_size / 4][D / 32][4 tokens].  Q8_0 codes
 * are stored plus 128; of Q4_0 codes a byte holds two dims: of K, byte 4 m + i
 * dims 8 m + i (low) and 8 m + 4 + i, of V dims 2 x (low) and 2 x + 1.  Values are
 * half(q * half(d)) and half((c - 8) * half(d)), as in the router's blocks; scales
 * of Q4_0 at most 8188, as those of fp16 rows are.
 * `pages` 16-byte aligned, at least m4_bridge_kv_cache_bytes. */
typedef struct {
    void* pages;
    size_t bytes;
    int format;
    uint32_t num_pages, page_size, Hkv, D;
} m4_kv_cache_t;

/* B sequences.  The rows of a call's Q, K, V and O (T of them) are the sequences'
 * new tokens: rows q_start[b] .. q_start[b + 1] (int32 [B + 1], not decreasing) are
 * the last keys of sequence b, which has kv_len[b] (int32 [B]) keys with them:
 * row i of n has position kv_len[b] - n + i.  Position p is token p % page_size
 * of page page_table[b][p / page_size] (int32 [B][table_stride], table_pages of
 * a row used).  All three are device memory, read by the kernels: entries out
 * of range (a page that is not there, more keys than the table holds, a
 * negative position, rows past T) are never followed -- such a token is not
 * written and not seen, and the others keep the positions that this gives them
 * (a start below 0 or past T counts rows that the call does not have).
 * Rows behind the last sequence are left as they are.
 * Two tokens of a call that fall on one place of the cache leave it undefined.
 * max_new and max_kv are what the caller expects of the longest sequence: they
 * choose kernels and the size of a workspace; the results hold for any.  T at
 * most 2^26, a table row's pages at most 0x7fff0000 tokens (else -4). */
typedef struct {
    uint32_t B;
    const int32_t *q_start, *kv_len, *page_table;
    uint32_t table_pages, table_stride;
    uint32_t max_new, max_kv;
} m4_kv_batch_t;

/* fp16 rows [T][heads][D]: element strides of a token and of a head (multiples
 * of 8; rows of an output must not overlap), D contiguous, 16-byte aligned.
 * `bytes` is what the buffer holds from ptr on. */
typedef struct {
    void* ptr;
    size_t bytes;
    int64_t token_stride, head_stride;
} m4_rows_t;

/* Rotary positions with several axes (time, height, width): pair i of `pairs`
 * (a multiple of 8, at most 128) turns by positions[axis of i][token] times its
 * inverse frequency; pairs are dims (i, i + pairs), or (2 i, 2 i + 1) when
 * traditional; dims from 2 * pairs on stay.  `table`: device memory, 16-byte
 * aligned, that holds what m4_bridge_rope_axes_table wrote for these pairs and
 * axes; a program keeps it as it keeps weights. */
enum { M4_ROPE_MAX_PAIRS = 128, M4_ROPE_PAIR_BYTES = 12 };
typedef struct {
    uint32_t pairs, axes;
    int traditional;
    const void* table;
    size_t table_bytes;
} m4_rope_axes_t;

/* Writes the table of `pairs` inverse frequencies (radians per position, finite)
 * and their axes (each below `axes`) to host memory: M4_ROPE_PAIR_BYTES a pair.
 * The frequencies come first, in turns as 64-bit fractions, then the axes, 32 bits
 * each; angles keep their precision at any int32 position.  Host arithmetic only.  0, -2 (null), -4. */
M4_API int m4_bridge_rope_axes_table(const double* inv_freq, const uint8_t* pair_axis, uint32_t pairs, uint32_t axes,
                                     void* table);

/* Bytes of a cache, 0 for a format or dimension that it does not take. */
M4_API size_t m4_bridge_kv_cache_bytes(int format, uint32_t num_pages, uint32_t page_size, uint32_t Hkv, uint32_t D);

/* Rotates the rows X [T][H][D] (D % 8 == 0, at most 256) into Y, which may be X
 * itself; positions int32 [axes][position_stride], a stride of 0 for one row
 * that all axes read.  Codes: -1, -2 (null,
 * misaligned, short or not device memory), -4 (dims, strides), -6.  T = 0 is 0. */
M4_API int m4_bridge_rope_axes(const m4_rope_axes_t* rope, const int32_t* positions, uint32_t position_stride,
                               const m4_rows_t* X, const m4_rows_t* Y, uint32_t T, uint32_t H, uint32_t D);

/* Writes the batch's rows of K and V [T][Hkv][D] to the cache, quantized as
 * m4_bridge_quantize_kv_q8_0 does (Q8_0) or with d = m / -8 of the value m of
 * largest magnitude, code floor(x / d + 8.5) (Q4_0).  With `rope`, K is rotated
 * first, and so are the rows Q [T][H][D] into Q_out (may be Q), in the same
 * launch; positions NULL with one axis: each token's place in its sequence.
 * The results are those of m4_bridge_rope_axes followed by a write.  Rows of Q
 * whose token has no place in the cache are left.  rope NULL: Q must be NULL.
 * Codes as m4_bridge_rope_axes, and -3 (format). */
M4_API int m4_bridge_kv_cache_append(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                     const m4_rows_t* K, const m4_rows_t* V, const m4_rope_axes_t* rope,
                                     const int32_t* positions, uint32_t position_stride, const m4_rows_t* Q,
                                     const m4_rows_t* Q_out, uint32_t H);

/* The inverse: the values of the batch's rows into K and V [T][Hkv][D] fp16
 * (with q_start the running sum of kv_len, whole sequences).  Rows that have no
 * place in the cache are left. */
M4_API int m4_bridge_kv_cache_read(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                   const m4_rows_t* K, const m4_rows_t* V);

/* Causal attention of the batch's rows Q [T][H][D] over the cached keys of their
 * sequences (their own included: append first), O [T][H][D]: query head h reads
 * KV head h / (H / Hkv); a row at position p sees keys up to p, and with `window`
 * > 0 only the last `window` of them.  A row that sees no key, or none that
 * scores above -infinity, is zero.  A cached value that is not finite (of a
 * row with 65504 in it, half(127 half(65504 / 127)) is infinity) reaches its
 * dim of the rows that see its key, and no others.  Both products are of fp16
 * operands, the cached values and the weights, and are summed in fp32, as are the
 * softmax's sums: 1.6 to 2.8e-4 of the result's norm from the same in 64 bits
 * (the rounding of O alone: up to 2.1e-4), 2.8 to 4.2e-4 over unrounded q * half(d).  Any number of rows a sequence, from one
 * decoded token to a prompt.  `ws`: m4_bridge_paged_attn_workspace bytes of
 * device memory, 16-byte aligned, whose contents do not matter; calls that may
 * run at the same time need one each.  scale finite.  Codes as above. */
M4_API size_t m4_bridge_paged_attn_workspace(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                             uint32_t H, uint32_t window);
M4_API int m4_bridge_dispatch_paged_attn(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                         const m4_rows_t* Q, const m4_rows_t* O, uint32_t H, float scale,
                                         uint32_t window, void* ws, size_t ws_bytes);

/* ---- trees of drafted tokens over the cache.  The new tokens of a sequence --
 *      its rows, as far as the call has them -- are the nodes of a tree, numbered
 *      from the first of them; a node comes behind its parent.  Places in the
 *      cache are the rows' own, node by node: append them as any rows. ------- */

/* What each row sees of its sequence's new tokens: bit j % 32 of word j / 32 of its
 * words of `mask` [T][words] for node j; nodes past 32 * words are seen by none.
 * positions int32 [T]: a node's place in the text, behind its ancestors'. */
typedef struct {
    uint32_t* mask;
    size_t mask_bytes;
    int32_t* positions;
    size_t positions_bytes;
    uint32_t words;
} m4_draft_tree_t;

/* Fills mask and positions of the batch's rows from their parents (int32 [T], node
 * numbers; one that is not an earlier node stands for none): a row sees itself and
 * its ancestors, its position is that of the sequence's first new token plus
 * their number.  Once a step, for all layers: m4_bridge_kv_cache_append takes the
 * positions.  Rows behind the last sequence are left.  Codes: -1, -2, -4, -6. */
M4_API int m4_bridge_draft_tree(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents,
                                const m4_draft_tree_t* tree);

/* m4_bridge_dispatch_paged_attn where a row sees, of its sequence's new tokens, those
 * that the mask says (any: not only earlier ones), and all keys before them; with
 * `window` > 0 those whose position is among the last `window` up to its own
 * (positions below the first new token's, or past the last one's, count as these;
 * without a window they may be NULL).  tree NULL: as there, up to itself.
 * lse (may be NULL): fp32 [T][H] by strides of any size, the natural logarithm of
 * the sum of exp(scale q . k) over the keys that a row sees, -infinity if none, of
 * unrounded weights.  O is divided by the sum of the rounded ones as in the other
 * call, and differs from its results by their rounding at most; with neither tree nor lse
 * it is that call. */
M4_API int m4_bridge_dispatch_paged_attn_tree(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                              const m4_rows_t* Q, const m4_rows_t* O, uint32_t H, float scale,
                                              uint32_t window, const m4_draft_tree_t* tree, const m4_rows_t* lse, void* ws,
                                              size_t ws_bytes);

/* The path that the model takes down each tree: node 0 (the newest token that is
 * certain), then again and again the first node whose parent is the last one and
 * whose token is the model's choice behind it.  parents, tokens, targets int32
 * [T], targets[i] the model's choice behind row i.  path int32 [T]: a sequence's
 * rows hold its nodes in order, then -1; count int32 [B]; next int32 [B]: the
 * choice behind the last of them.  A sequence without rows: 0 and -1; so all of them
 * where T is 0, whose other pointers, and those of the two that are not wanted, may be NULL. */
M4_API int m4_bridge_tree_accept(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents, const int32_t* tokens,
                                 const int32_t* targets, int32_t* path, int32_t* count, int32_t* next);

/* Keeps of each sequence's new tokens the first count[b] of the list in its rows
 * of `keep` (int32 [T], node numbers, rising, as m4_bridge_tree_accept writes
 * them): K and V of node keep[i] move to the place of new token i.  Then the
 * sequence has kv_len_out[b] keys: those before the tree and count[b] (int32 [B],
 * may be the batch's kv_len, may be NULL).  Entries that are no nodes, and places
 * that are not there, move nothing; a list that does not rise leaves the
 * sequence's new tokens undefined.  Once a layer.  T = 0 needs nothing but the cache's
 * description and, for kv_len_out, the batch's kv_len, which it gets. */
M4_API int m4_bridge_kv_cache_keep(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const int32_t* keep,
                                   const int32_t* count, int32_t* kv_len_out);

/* ---- bounded caches: the attention weight that each key has received -------- */

/* sums, fp32 [num_pages][Hkv][page_size] (16-byte aligned, as the pages lie): adds to
 * each key's the weights exp(scale q . k - lse) of the batch's rows Q [T][H][D] and
 * of the H / Hkv query heads of its KV head that see it, as m4_bridge_dispatch_paged_attn
 * does with the same window; for the batch's new tokens it sets them, whatever
 * they held.  lse as that call's tree form writes it (append, attend, then weigh; a
 * row whose lse is infinite gives nothing, whatever its Q holds).
 * Products are of fp16 operands, the cached values, summed in fp32; no order changes.
 * A page that two sequences of a call share: its sums are undefined.  A call without
 * rows writes nothing.  B x Hkv, and T x H / Hkv, below 2^31. */
M4_API int m4_bridge_kv_cache_weigh(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* Q,
                                    const m4_rows_t* lse, uint32_t H, float scale, uint32_t window, float* sums,
                                    size_t sums_bytes);

/* Evicts keys: of each sequence and KV head the first `sinks` places, the last
 * `recent` and the ones with the largest sums among the others stay, `budget` in all
 * (at least sinks + recent; equal sums: the lower place; NaN above all numbers), or
 * all if there are no more.  They are copied in their order, codes, scales and sums,
 * to the pages of table_out (int32 [B][out_stride], out_pages of a row used, at
 * least `budget` tokens), whose sequences have kv_len_out[b] keys (int32 [B]);
 * kept int32 [B][Hkv][budget]: the places that they had, then -1.  The old
 * pages stay as they are, also where sequences share them; those of table_out are
 * others, and no two alike.  Heads keep keys of their own, so a place no longer
 * stands for a position: what is appended next takes explicit positions, and a
 * window counts places.  Those of m4_bridge_draft_tree are formed from kv_len, so they are
 * places then: attention takes them as they are, an append with what was evicted added.  Keys on pages that are not there count as gone;
 * kept ones whose new page is not there are not copied.  q_start is not read (but
 * not NULL). */
M4_API int m4_bridge_kv_cache_evict(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, float* sums, size_t sums_bytes,
                                    const int32_t* table_out, uint32_t out_pages, uint32_t out_stride, uint32_t budget,
                                    uint32_t sinks, uint32_t recent, int32_t* kept, size_t kept_bytes, int32_t* kv_len_out,
                                    void* ws, size_t ws_bytes);
/* Bytes of its workspace, device memory of any contents, 16-byte aligned; 0 for many or
 * short sequences (ws may be NULL then).  Calls that may run at the same time need one each. */
M4_API size_t m4_bridge_kv_evict_workspace(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch);

/* A transformer block over the cache: m4_bridge_prefill_layer_ex with the
 * batch's rows as its prompt and the paged cache in place of one call's keys --
 * RMSNorm -> Q, K, V -> m4_bridge_kv_cache_append (K and Q turned by `rope`, NULL:
 * not) -> m4_bridge_dispatch_paged_attn -> O-projection + residual -> RMSNorm ->
 * SwiGLU -> down-projection + residual.  X, X_out fp16 [T, d_model], X_out not
 * X; weights as there, in `format`; KV heads and head width are the cache's.
 * Device pointers, 16-byte aligned.  Scratch is the bridge's: a size must have
 * run once before it is captured, calls run one after the other, and the stream
 * is of the device that was current at m4_bridge_init (else -2).  Rows of
 * X_out behind the last sequence hold nothing of use.  Codes as
 * m4_bridge_prefill_layer_ex. */
M4_API int m4_bridge_paged_layer(void* X_ptr, void* w_attn, void* Wq, void* Wk, void* Wv, void* Wo, void* w_ffn,
                                 void* Wg, void* Wu, void* Wd, void* X_out, const m4_kv_cache_t* cache,
                                 const m4_kv_batch_t* batch, uint32_t T, const m4_rope_axes_t* rope,
                                 const int32_t* positions, uint32_t position_stride, int format, uint32_t d_model,
                                 uint32_t Hq, uint32_t N_mlp, float attn_scale, uint32_t window, int norm_type,
                                 float norm_eps);

/* Validation only, as m4_bridge_validate_gemm: the code that the call would
 * return on an initialized bridge (0 if it would launch) but for the check that
 * the pointers are device memory. */
M4_API int m4_bridge_validate_rope_axes(const m4_rope_axes_t* rope, const int32_t* positions, uint32_t position_stride,
                                        const m4_rows_t* X, const m4_rows_t* Y, uint32_t T, uint32_t H, uint32_t D);
M4_API int m4_bridge_validate_kv_cache_append(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                              const m4_rows_t* K, const m4_rows_t* V, const m4_rope_axes_t* rope,
                                              const int32_t* positions, uint32_t position_stride, const m4_rows_t* Q,
                                              const m4_rows_t* Q_out, uint32_t H);
M4_API int m4_bridge_validate_kv_cache_read(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                            const m4_rows_t* K, const m4_rows_t* V);
M4_API int m4_bridge_validate_paged_attn(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                         const m4_rows_t* Q, const m4_rows_t* O, uint32_t H, float scale,
                                         uint32_t window, const void* ws, size_t ws_bytes);
M4_API int m4_bridge_validate_draft_tree(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents,
                                         const m4_draft_tree_t* tree);
M4_API int m4_bridge_validate_paged_attn_tree(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                              const m4_rows_t* Q, const m4_rows_t* O, uint32_t H, float scale,
                                              uint32_t window, const m4_draft_tree_t* tree, const m4_rows_t* lse,
                                              const void* ws, size_t ws_bytes);
M4_API int m4_bridge_validate_tree_accept(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents,
                                          const int32_t* tokens, const int32_t* targets, const int32_t* path,
                                          const int32_t* count, const int32_t* next);
M4_API int m4_bridge_validate_kv_cache_keep(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                            const int32_t* keep, const int32_t* count, const int32_t* kv_len_out);
M4_API int m4_bridge_validate_kv_cache_weigh(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T,
                                             const m4_rows_t* Q, const m4_rows_t* lse, uint32_t H, float scale,
                                             uint32_t window, const float* sums, size_t sums_bytes);
M4_API int m4_bridge_validate_kv_cache_evict(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, const float* sums,
                                             size_t sums_bytes, const int32_t* table_out, uint32_t out_pages,
                                             uint32_t out_stride, uint32_t budget, uint32_t sinks, uint32_t recent,
                                             const int32_t* kept, size_t kept_bytes, const int32_t* kv_len_out,
                                             const void* ws, size_t ws_bytes);

/* Run subsequent work on `stream` (a hipStream_t, e.g. torch's current
 * stream); NULL restores the bridge's own stream.  Returns 0 or -1. */
M4_API int m4_bridge_set_stream(void* stream);
/* The hipStream_t work is issued on. */
M4_API void* m4_bridge_get_stream(void);
/* Text of the last error this thread's bridge calls saw ("" if none); per
 * thread, like errno, so a caller reads the message of its own failed call. */
M4_API const char* m4_bridge_last_error(void);

/* ---- roofline probes (quant_router_kernels.metal:71-104, timed as in
 *      bench_universal_router.mm:645-717) ------------------------------- */

/* probe_memory_bandwidth: HBM GB/s of a read-only stream over `bytes` (> the
 * 256 MB Infinity Cache to measure HBM) and of the reference's dst = src + 1
 * copy (bytes read + written), best of `reps` timed runs after one warmup.
 * Allocates its own buffers; runs on the null stream.  0, -2, -4 or -6. */
M4_API int m4_probe_hbm_bandwidth(size_t bytes, int reps, double* read_gbs, double* copy_gbs);
/* probe_fma_roofline, on the matrix pipe: dense fp16 TFLOP/s of back-to-back
 * v_mfma_f32_32x32x16_f16 on every SIMD (`iters` rounds of 4 independent
 * chains per wave), best of `reps`, and the average shader clock (GHz) the
 * waves saw (shader-cycle counter over the 100 MHz real-time counter).
 * `iters` >= 64 and a multiple of 4.  0, -2, -4 or -6. */
M4_API int m4_probe_mfma_f16(uint32_t iters, int reps, double* tflops, double* clock_ghz);
/* The same with random fp16 operands (four A and four B fragments per lane,
 * values in [-1, 1)): the matrix pipe draws more power when more operand bits
 * toggle, and the part lowers its clock, so this is the dense ceiling real
 * activations and weights can reach.  No counterpart in the reference (its
 * FMA probe is operand-independent).  `iters` a multiple of 4.  0, -2, -4, -6. */
M4_API int m4_probe_mfma_f16_random(uint32_t iters, int reps, double* tflops, double* clock_ghz);

/* ---- format registry (src/router/quant_registry.h:14-65) ---------------- */

typedef struct {
    int format;
    const char* name;
    const char* description;
    uint32_t block_size;
    uint64_t struct_size;
    double bits_per_weight;
    const char* gemm_kernel_name;
    const char* head_gemm_kernel_name;
} m4_quant_codec_info;

/* QuantRegistry::get -- 0 and *out filled, or -3 if unknown. */
M4_API int m4_registry_get(int format, m4_quant_codec_info* out);
/* QuantRegistry::get_by_name -- format id or -3. */
M4_API int m4_registry_get_by_name(const char* name);
/* QuantRegistry::available_formats -- count; ids written to out[0..cap). */
M4_API int m4_registry_available_formats(int* out, int cap);
/* QuantRegistry::compute_weight_bytes -- 0 for an unknown format. */
M4_API uint64_t m4_registry_compute_weight_bytes(int format, uint64_t num_elements);
/* QuantRegistry::has_format */
M4_API bool m4_registry_has_format(int format);
/* QuantRegistry::register_codec (e.g. QUANT_CUSTOM = 99); strings are copied. */
M4_API int m4_registry_register_codec(const m4_quant_codec_info* info);

#ifdef __cplusplus
}
#endif

#endif /* M4_MLX_BRIDGE_H */
