// qr_paged.h -- paged, quantized KV cache: page geometry, batch and view
// descriptors (host and device) and the launch interface of its kernels.
//
// A page holds P tokens (16 .. 256, a power of two) of every KV head.  Per
// head: K codes [P][D], V codes [P / 4][D][4 tokens], K scales [P][D / 32]
// fp16, V scales [P / 4][D / 32][4 tokens] fp16, one scale per 32 dims of a
// token.  Q8_0 codes are stored plus 128 (one byte per dim); Q4_0 codes are
// 0 .. 15, two dims to a byte: of K, byte 4 m + i holds dims 8 m + i (low) and
// 8 m + 4 + i (high), of V dims 2 x and 2 x + 1.  Why: a lane's MFMA operands
// are then whole 16- or 32-byte runs of both K (dims of a token) and V (tokens
// of a dim), with no transposition on the way.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qr_formats.h"

namespace qr {

struct PageGeom {
    uint8_t* pages;
    uint32_t num_pages, log2_page, Hkv;
    // bytes of a head's share of a page, and of its parts before V and the scales
    uint32_t head_bytes, v_off, ks_off, vs_off;
};

inline PageGeom page_geom(void* pages, int format, uint32_t num_pages, uint32_t P, uint32_t Hkv, uint32_t D) {
    PageGeom g{};
    g.pages = static_cast<uint8_t*>(pages);
    g.num_pages = num_pages;
    while ((1u << g.log2_page) < P) g.log2_page++;
    g.Hkv = Hkv;
    const uint32_t codes = P * (format == QUANT_Q8_0 ? D : D / 2), scales = P * (D / 32) * 2;
    g.v_off = codes;
    g.ks_off = 2 * codes;
    g.vs_off = 2 * codes + scales;
    g.head_bytes = 2 * codes + 2 * scales;
    return g;
}

// New tokens of sequence b: rows q_start[b] .. q_start[b + 1], the last of its
// kv_len[b] keys.  Values on the device are clamped to T and to the table, so
// none of them reaches past a buffer.
struct BatchView {
    uint32_t B, T;
    const int32_t *q_start, *kv_len, *table;
    uint32_t table_pages, table_stride;
};

// Rows [T][H][D] of fp16 by strides in elements.
struct RowsView {
    _Float16* p;
    int64_t ts, hs;
};

// Pairs' frequencies in turns per position, as 64-bit fractions (a position times
// one, modulo 2^64, is the angle's fraction of a turn, exact at any position), then
// their axes, 32 bits each.  In device memory: as a kernel argument (host memory)
// a table's latency showed in every short call (64 tokens 6.4 us, now 4.6).
struct RopeView {
    const uint64_t* table;
    uint32_t pairs, axes;
    int traditional;
    const int32_t* positions;  // [axes][stride], or null: the place in the sequence
    uint32_t position_stride;
};

// Rotates Q (H heads; Qo may be Q) and, when the cache is given, rotates K and
// writes K and V to it.  rope.pairs = 0: no rotation.  D <= 256 without a cache.
struct AppendParams {
    RowsView Q, Qo, K, V;
    uint32_t H, T, D;
    int format;
    PageGeom geom;   // pages null: no cache
    BatchView batch;
    RopeView rope;
};
hipError_t launch_kv_append(const AppendParams& p, hipStream_t st);

struct ReadParams {
    RowsView K, V;
    uint32_t D;
    int format;
    PageGeom geom;
    BatchView batch;
};
hipError_t launch_kv_read(const ReadParams& p, hipStream_t st);

// One fp32 value per row and head, by strides in elements.
struct ValuesView {
    float* p;
    int64_t ts, hs;
};

// What each new token sees of its sequence's new tokens: bit j of its words of the
// mask [T][words] for the j-th of them; places [T]: their positions (for a window).
struct TreeView {
    const uint32_t* mask;
    uint32_t words;
    const int32_t* places;
};

struct PagedAttnParams {
    RowsView Q, O;
    uint32_t H, G, D;  // query heads, those of a KV head, head width
    int format;
    float scale;
    uint32_t window;  // keys a row sees at most (the newest), 0: all
    PageGeom geom;
    BatchView batch;
    uint32_t max_new, max_kv;  // what the plan expects; any value is right
    // a launch's: sequences of that many rows a KV head, [min_rows, max_rows)
    uint32_t min_rows, max_rows;
    uint8_t* ws;
    TreeView tree;   // launch_paged_attn_tree only
    ValuesView lse;  // and launch_paged_attn_lse; p null: not wanted
};
size_t paged_attn_workspace(const PagedAttnParams& p);
hipError_t launch_paged_attn(const PagedAttnParams& p, hipStream_t st);
// the same with the logarithm of each row's sum of exponentials, and with a tree's mask (lse or none)
hipError_t launch_paged_attn_lse(const PagedAttnParams& p, hipStream_t st);
hipError_t launch_paged_attn_tree(const PagedAttnParams& p, hipStream_t st);


// ---- trees of drafted tokens ----
// Masks and places of the batch's new tokens from their parents (launch interface of qr_paged_tree.hip).
struct DraftParams {
    BatchView batch;  // no table
    const int32_t* parents;
    uint32_t* mask;
    uint32_t words;
    int32_t* places;
};
hipError_t launch_draft_tree(const DraftParams& p, hipStream_t st);

struct AcceptParams {
    BatchView batch;  // no table
    const int32_t *parents, *tokens, *targets;
    int32_t *path, *count, *next;
};
hipError_t launch_tree_accept(const AcceptParams& p, hipStream_t st);

struct KeepParams {
    uint32_t D;
    int format;
    PageGeom geom;
    BatchView batch;
    const int32_t *keep, *count;
    int32_t* len_out;
};
hipError_t launch_kv_keep(const KeepParams& p, hipStream_t st);

// ---- bounded caches ----
// Division of numbers below 2^31 by a number that is known before, in three instructions.
struct Divider {
    uint32_t by, mul, shift;
};
inline Divider divider(uint32_t by) {
    Divider d{by, 0, 0};
    while ((1ull << d.shift) < by) d.shift++;
    d.mul = (uint32_t)(((1ull << 32) * ((1ull << d.shift) - by)) / by + 1);
    return d;
}

struct WeighParams {
    RowsView Q;
    ValuesView lse;
    uint32_t H, G, D;
    Divider of_group;
    int format;
    float scale;
    uint32_t window;
    PageGeom geom;
    BatchView batch;
    uint32_t max_new, max_kv;
    // a launch's: sequences of that many rows a KV head, [min_rows, max_rows)
    uint32_t min_rows, max_rows;
    uint32_t tile_shift;
    float* sums;  // [num_pages][Hkv][page]
};
hipError_t launch_kv_weigh(const WeighParams& p, hipStream_t st);

struct EvictParams {
    uint32_t D;
    int format;
    PageGeom geom;
    BatchView batch;  // no rows
    uint32_t max_kv;
    uint32_t budget, sinks, recent;
    float* sums;
    const int32_t* table_out;
    uint32_t out_pages, out_stride;
    int32_t *kept, *len_out;
    uint8_t* ws;
};
size_t kv_evict_workspace(const EvictParams& p);
hipError_t launch_kv_evict(const EvictParams& p, hipStream_t st);

// The rows of sequence b that a call has, and the position of the first of them.
struct NewRows {
    int q0, n, first;
};
__host__ __device__ inline NewRows new_rows(const BatchView& v, uint32_t b) {
    const int T = (int)v.T, start = v.q_start[b], end = v.q_start[b + 1], len = v.kv_len[b];
    NewRows r;
    r.q0 = start < 0 ? 0 : (start > T ? T : start);
    r.n = (end < 0 ? 0 : (end > T ? T : end)) - r.q0;
    if (r.n < 0) r.n = 0;
    // rows past T count: those before them keep their positions
    r.first = r.n ? (len < 0 ? 0 : len) - (end - r.q0) : 0;
    return r;
}

}  // namespace qr
