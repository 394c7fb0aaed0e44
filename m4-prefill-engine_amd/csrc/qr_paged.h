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
};
size_t paged_attn_workspace(const PagedAttnParams& p);
hipError_t launch_paged_attn(const PagedAttnParams& p, hipStream_t st);

}  // namespace qr
