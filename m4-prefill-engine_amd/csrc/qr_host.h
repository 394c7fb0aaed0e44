// qr_host.h -- host-only helpers of the C-ABI (qr_host.cpp).
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../include/m4_mlx_bridge.h"
#include "qr_formats.h"

namespace qr {

// Whether every page of the host range [p, p + bytes) is readable (and, when
// `write`, writable) by this process; probed without raising a signal.
bool host_range_ok(const void* p, size_t bytes, bool write);

// Formats m4_bridge_dispatch_gemm accepts, and every format with kernels.
bool is_projection_format(int f);
bool has_kernels(int f);

// Argument validation of a projection: 0, or the reference's codes -2 / -3 /
// -4 in its order (core/bridge/m4_mlx_bridge.mm:204-230, minus the init
// check); `ext` widens the format range to every format with kernels.
int validate(const void* X, size_t Xb, const void* W, size_t Wb, const void* Y, size_t Yb, int format,
             uint32_t M, uint32_t K, uint32_t N, bool ext = false);

// The table of a rotary embedding (m4_bridge_rope_axes_table).
int rope_axes_table(const double* inv_freq, const uint8_t* pair_axis, uint32_t pairs, uint32_t axes, void* table);
// Bytes of a paged cache (0: not a cache), and the codes that the serving entry
// points return for their arguments; *empty: valid, with no rows to work on.
size_t kv_cache_bytes(int format, uint32_t num_pages, uint32_t page_size, uint32_t Hkv, uint32_t D);
int validate_rope_axes(const m4_rope_axes_t* rope, const int32_t* positions, uint32_t position_stride,
                       const m4_rows_t* X, const m4_rows_t* Y, uint32_t T, uint32_t H, uint32_t D, bool* empty);
int validate_append(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* K, const m4_rows_t* V,
                    const m4_rope_axes_t* rope, const int32_t* positions, uint32_t position_stride,
                    const m4_rows_t* Q, const m4_rows_t* Q_out, uint32_t H, bool* empty);
int validate_read(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* K, const m4_rows_t* V,
                  bool* empty);
int validate_attn(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* Q, const m4_rows_t* O,
                  uint32_t H, float scale, const void* ws, bool* empty);
// lse may be null, and the tree
int validate_attn_tree(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* Q, const m4_rows_t* O,
                       uint32_t H, float scale, uint32_t window, const m4_draft_tree_t* tree, const m4_rows_t* lse,
                       const void* ws, bool* empty);
int validate_draft_tree(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents, const m4_draft_tree_t* tree, bool* empty);
int validate_tree_accept(const m4_kv_batch_t* batch, uint32_t T, const int32_t* parents, const int32_t* tokens,
                         const int32_t* targets, const int32_t* path, const int32_t* count, const int32_t* next, bool* empty);
int validate_keep(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const int32_t* keep,
                  const int32_t* count, const int32_t* kv_len_out, bool* empty);
int validate_weigh(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* Q, const m4_rows_t* lse,
                   uint32_t H, float scale, const float* sums, size_t sums_bytes, bool* empty);
int validate_evict(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, const float* sums, size_t sums_bytes,
                   const int32_t* table_out, uint32_t out_pages, uint32_t out_stride, uint32_t budget, uint32_t sinks,
                   uint32_t recent, const int32_t* kept, size_t kept_bytes, const int32_t* kv_len_out, const void* ws, bool* empty);
// all of a layer's arguments but its tensors
int validate_layer(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rope_axes_t* rope,
                   const int32_t* positions, uint32_t position_stride, int format, uint32_t d_model, uint32_t Hq,
                   uint32_t N_mlp, float scale, bool norms, int norm_type, bool* empty);

}  // namespace qr
