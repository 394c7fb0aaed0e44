// qr_paged_attn.hip -- causal attention of new tokens over a paged, quantized
// KV cache: softmax over the keys a row sees of scale q . k, times v.
//
// Rows of a KV head are (token, query head of its group) pairs; a tile takes
// R = 16 NR of them.  A wave takes 32 keys at a time with v_mfma_f32_16x16x32_f16:
// S^T = K . Q^T and O^T += V^T . P^T, so a lane owns one row, its softmax state
// is lane-local but for the four lanes that share the row, and P goes from the
// first product's result into the second's operand without leaving the lane:
// lane (j, g) gets the scores of keys 16 t + 4 g + r, and takes as its k index
// 8 g + 4 t + r of V^T the same key.  The contraction runs over dims in the order
// in which lane group g owns dims D/4 g .. of a key, one run of bytes of the page.
#include "qr_device.h"
#include "qr_paged.h"

namespace qr {

constexpr uint32_t kWaves = 4;     // of a workgroup
constexpr uint32_t kStep = 32;     // keys of a step
// What an item costs beside its steps, in steps: its descriptors, queries and
// the write of its rows.  us with 2 / 3 / 4: drafted tokens 19.3 / 18.2 / 18.9, a
// chunk of 300 among single tokens 23.7 / 25.3 / 25.0, 64 requests of D = 64
// 21.7 / 19.1 / 19.0.
constexpr uint32_t kItemCost = 3;
// Waves: two per SIMD where each gets kLongShare of the line (four requests of
// 131072 keys: 132 us on one, 118 on two when this was chosen), else one: fewer items are cut and fewer
// parts joined (drafted tokens 18.7 us, on two 19.8; one token over 16384 keys 16.7
// and 19.5).  A count between the two leaves some SIMDs with two and the rest
// waiting.  Three are slower: with the next step's tiles in flight the registers
// of most variants hold two.
constexpr uint32_t kMaxWaves = 2048, kFewWaves = 1024, kLongShare = 16, kMinSteps = 2;
// Chunks: rows of a row tile, workgroups (one a CU), what an item costs beside its
// key tiles and the least of the line that is worth a workgroup.
constexpr uint32_t kChunkTile = 256, kChunkGroups = 256, kChunkCost = 2, kChunkMin = 4;
// Rows times keys of all heads from which chunks of rows are worth it, and the
// tiles through LDS that they share: us of rows / chunks at H = 32, Hkv = 8,
// D = 128, one request unless said: 2^25 64 tokens over 16384 keys 49 / 76, 256
// over 4096 48 / 50, eight of 32 over 4096 57 / 45; 2^26 512 over 4096 72 / 70,
// eight of 256 over 1024 70 / 57; 2^27 256 over 16384 130 / 102.
constexpr uint64_t kChunkWork = (uint64_t)1 << 26;
constexpr float kNone = -3.402823466e38f;  // reference point of a row that has seen no score above -infinity
// Weights are rounded to fp16 for the second product, 2^-11 of each; those below
// 2^-14 lose more.  So a row's reference point is kLift below its largest exponent:
// beside a largest weight of 2^7 or more the small ones keep 2^-32 of it, where
// beside 1 it would be 2^-25, and many light keys next to a heavy one count.  It
// moves when an exponent passes 15 (kTop, as bits), so no weight passes 2^15.  The sum
// is of the rounded weights, so that one that is off moves a row towards its value or
// away from it, and does not scale the row.
constexpr float kLift = 7.0f;
constexpr int kTop = 0x41700000;

// A workgroup's note on its partial rows.  tail: an item begins in its share and
// goes on in the next one's (slot 1, and which rows they are: the KV head, the
// first of its sequence's (token, head) pairs and how many, the sequence's first
// row); head: the first item of its share began before it (slot 0) and ends here
// (1) or goes on (2).
struct alignas(16) ItemNote {
    uint32_t hk, first, rows, q0, tail, head, pad[2];
};

struct WorkPlan {
    uint32_t rows, groups, items;  // of a row tile; workgroups; row tiles of all heads, as expected
};
struct AttnPlan {
    WorkPlan few, many;  // of the sequences of few rows and of those of chunks; no groups: no launch
    bool both;
};

// Operands are the cache's values, half(q half(d)): rounded to fp16 because that is what
// such a cache holds by definition (kv_cache_read returns the same), and what the matrix
// unit takes.  Q8_0: 1024 + 128 + q of four bytes, as pairs.
__device__ __forceinline__ h2_t q8_lo(uint32_t w, h2_t d) {
    const h2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return (as_h2(nib_pair_lo(w)) - off) * d;
}
__device__ __forceinline__ h2_t q8_hi(uint32_t w, h2_t d) {
    const h2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return (as_h2(nib_pair_hi(w)) - off) * d;
}
// values c d - 8 d of Q4_0 codes, n8 = -8 d: one instruction, and one rounding as in
// (c - 8) d since 8 d is exact for scales up to 8188, which fp16 rows do not pass
template <bool HI>
__device__ __forceinline__ h2_t q4_pair(uint32_t codes, h2_t d, h2_t n8) {
    return __builtin_elementwise_fma(code_pair<HI>(codes), d, n8);
}
__device__ __forceinline__ h2_t q4_offset(h2_t d) {
    const h2_t m8 = {(_Float16)-8.0f, (_Float16)-8.0f};
    return d * m8;
}

// Smallest V scale (fp16 bits, without the sign) whose values may not be finite: 512,
// -128 of which is -65536, or 8192, -8 of which is (q4_offset; past what such a cache
// holds).  A row of fp16 reaches 516 in Q8_0: half(127 half(65504 / 127)) is infinite.
template <int FMT>
constexpr uint32_t kOddScale = FMT == QUANT_Q8_0 ? 0x6000u : 0x7000u;

// Hidden keys have weight 0, and 0 times a value that is not finite is NaN.  Where such
// values meet rows that do not see them, the product takes their finite part, and two
// more, in bfloat16, add what is left out: 2^127 or -2^127 for an infinity, both for NaN,
// times 4 for a row that sees the key, which fp32 does not hold, and times 0 for others.
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ h8_t finite_part(h8_t v) {
    u4_t w = __builtin_bit_cast(u4_t, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t lo = (w[i] & 0x7c00u) == 0x7c00u ? 0xffff0000u : 0xffffffffu;
        w[i] &= (w[i] & 0x7c000000u) == 0x7c000000u ? lo & 0xffffu : lo;
    }
    return __builtin_bit_cast(h8_t, w);
}
// DOWN: of -infinities, else of infinities
template <bool DOWN>
__device__ __forceinline__ b8_t marks_of(h8_t v) {
    u4_t w = __builtin_bit_cast(u4_t, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 32; e += 16) {
            const uint32_t h = w[i] >> e & 0xffffu;
            if (h == (DOWN ? 0xfc00u : 0x7c00u) || (h & 0x7fffu) > 0x7c00u) m |= (DOWN ? 0xff00u : 0x7f00u) << e;
        }
        w[i] = m;
    }
    return __builtin_bit_cast(b8_t, w);
}
constexpr uint32_t kSeen = 0x4080u;  // bfloat16 4

template <bool ONCE, typename T>
__device__ __forceinline__ T load_of(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
    return *reinterpret_cast<const T*>(p);
}
template <int W, bool ONCE>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t w[W]) {
    if constexpr (W == 1) {
        w[0] = load_of<ONCE, uint32_t>(p);
    } else if constexpr (W == 2) {
        const u2_t a = load_of<ONCE, u2_t>(p);
        w[0] = a.x;
        w[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; i++) {
            const u4_t a = load_of<ONCE, u4_t>(p + 16 * i);
            w[4 * i] = a.x;
            w[4 * i + 1] = a.y;
            w[4 * i + 2] = a.z;
            w[4 * i + 3] = a.w;
        }
    }
}

// the same through a buffer resource: a lane's offset and a wave's
template <int W>
__device__ __forceinline__ void fetch_words(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff, uint32_t w[W]) {
    if constexpr (W == 1) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, soff, 0);
    } else if constexpr (W == 2) {
        const u2_t a = __builtin_amdgcn_raw_buffer_load_b64(r, off, soff, 0);
        w[0] = a.x;
        w[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; i++) {
            const u4_t a = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, soff, 0);
            w[4 * i] = a.x;
            w[4 * i + 1] = a.y;
            w[4 * i + 2] = a.z;
            w[4 * i + 3] = a.w;
        }
    }
}

// K values of dims 8 kk .. 8 kk + 7 of a run of codes
template <int FMT>
__device__ __forceinline__ h8_t k_octet(const uint32_t* k, int kk, h2_t d) {
    h2_t a, b, c, e;
    if constexpr (FMT == QUANT_Q8_0) {
        a = q8_lo(k[2 * kk], d);
        b = q8_hi(k[2 * kk], d);
        c = q8_lo(k[2 * kk + 1], d);
        e = q8_hi(k[2 * kk + 1], d);
    } else {
        const uint32_t lo = k[kk] & 0x0f0f0f0fu, hi = k[kk] >> 4 & 0x0f0f0f0fu;
        const h2_t n8 = q4_offset(d);
        a = q4_pair<false>(lo, d, n8);
        b = q4_pair<true>(lo, d, n8);
        c = q4_pair<false>(hi, d, n8);
        e = q4_pair<true>(hi, d, n8);
    }
    return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}
// V values of four keys of dim dt of a run of codes, as two pairs
template <int FMT>
__device__ __forceinline__ u2_t v_quad(const uint32_t* v, int dt, u2_t d) {
    const h2_t s0 = as_h2((uint32_t)d.x), s1 = as_h2((uint32_t)d.y);
    if constexpr (FMT == QUANT_Q8_0) return u2_t{as_u32(q8_lo(v[dt], s0)), as_u32(q8_hi(v[dt], s1))};
    const uint32_t w = (dt & 1 ? v[dt / 2] >> 4 : v[dt / 2]) & 0x0f0f0f0fu;
    return u2_t{as_u32(q4_pair<false>(w, s0, q4_offset(s0))), as_u32(q4_pair<true>(w, s1, q4_offset(s1)))};
}

// A lane's share of 16 keys: W words of K codes (D / 4 dims of one key) and of V
// codes (D / 16 dims of four keys), its K scale and four V scales.
template <int FMT, int D>
struct Tile {
    static constexpr int W = FMT == QUANT_Q8_0 ? D / 16 : D / 32;
    static constexpr uint32_t CB = 4 * W * 4, NB = D / 32;  // bytes of a key's codes, blocks
    uint32_t k[W], v[W];
    uint32_t kd;
    u2_t vd;
    bool there;  // its page is one of the cache's

    // a lane's byte offsets of those in a page, but for the tile's first slot
    struct Offsets {
        uint32_t k, v, ks, vs;
        __device__ __forceinline__ Offsets(const PageGeom& g, int lane) {
            const uint32_t j = lane & 15, q = lane >> 4;
            k = j * CB + q * (W * 4);
            v = g.v_off + q * (4 * CB) + j * (W * 4);
            ks = g.ks_off + (j * NB + q * NB / 4) * 2;
            vs = g.vs_off + (q * NB + j * NB / 16) * 8;
        }
    };
    // ONCE: codes that no other wave reads pass the caches by
    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t* head, const Offsets& at, uint32_t slot0) {
        // no buffer resources: through them the four requests of 131072 keys took 145 us, so 128
        load_words<W, ONCE>(head + slot0 * CB + at.k, k);
        load_words<W, ONCE>(head + slot0 * CB + at.v, v);
        kd = *reinterpret_cast<const uint16_t*>(head + slot0 * (NB * 2) + at.ks);
        vd = *reinterpret_cast<const u2_t*>(head + slot0 * (NB * 2) + at.vs);
    }
    // operand of contraction step kk: dims 8 kk .. 8 kk + 7 of the lane's run
    __device__ __forceinline__ h8_t k_frag(int kk) const { return k_octet<FMT>(k, kk, as_h2(kd | kd << 16)); }
    // the four keys of dim dt of the lane's run, as two pairs
    __device__ __forceinline__ u2_t v_pairs(int dt) const { return v_quad<FMT>(v, dt, vd); }
    // of those, `y`, the ones that are not finite become zero: the codes of Q8_0 by finite
    // scales here, the others by their scales
    __device__ __forceinline__ void clear_odd(int dt, u2_t y) {
        if constexpr (FMT == QUANT_Q8_0) {
            const uint32_t h[4] = {y.x & 0x7fffu, y.x >> 16 & 0x7fffu, y.y & 0x7fffu, y.y >> 16 & 0x7fffu};
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (h[r] >= 0x7c00u) v[dt] = (v[dt] & ~(0xffu << 8 * r)) | 0x80u << 8 * r;
        }
    }
    __device__ __forceinline__ void clear_scales() {
        constexpr uint32_t least = FMT == QUANT_Q8_0 ? 0x7c00u : kOddScale<FMT>;
        const uint32_t e[2] = {vd.x, vd.y};
        uint32_t y[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            y[i] = ((e[i] & 0x7fffu) >= least ? 0 : e[i] & 0xffffu) | ((e[i] >> 16 & 0x7fffu) >= least ? 0 : e[i] & 0xffff0000u);
        vd = u2_t{y[0], y[1]};
    }
};

template <int D, int R>
__host__ __device__ constexpr size_t slot_bytes() {
    return (size_t)R * (D + 2) * 4;
}
// workspace: a note per workgroup, then two slots per workgroup of partial rows
// (O [R][D], reference points [R], sums [R], fp32)
template <int D, int R>
__device__ __forceinline__ float* slot_of(uint8_t* ws, uint32_t groups, uint32_t w, int which) {
    return reinterpret_cast<float*>(ws + (size_t)groups * sizeof(ItemNote) + ((size_t)w * 2 + which) * slot_bytes<D, R>());
}

// lane `at`'s value, as a wave-uniform one
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int at) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), at) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, at);
}

// a / b of wave-uniform numbers that nearly always fit in 32 bits, where a
// division takes a fifth of the time
__device__ __forceinline__ uint64_t udiv(uint64_t a, uint64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}
// share w of nw (at most 2^16) of a line of `total`: total w / nw on, in whole
// places, so that as many items as shares, alike in cost, are not cut
__device__ __forceinline__ void share_of(uint64_t total, uint32_t nw, uint32_t w, uint64_t& s0, uint64_t& s1) {
    const uint64_t each = udiv(total, nw);
    const uint32_t more = (uint32_t)(total - each * nw);
    s0 = each * w + more * w / nw;
    s1 = each * (w + 1) + more * (w + 1) / nw;
}

struct Seq {
    int q0, n, first;     // first row, new tokens, position of the first of them
    int keys, lo;         // keys that the table holds and a row may see, first that one sees (a multiple of kStep)
    uint32_t tiles, steps;  // row tiles and key steps per tile
    uint64_t cost;
};
__device__ __forceinline__ Seq seq_of(const PagedAttnParams& p, uint32_t b, uint32_t R) {
    Seq s;
    const int T = (int)p.batch.T;
    const int cap = (int)min((uint64_t)p.batch.table_pages << p.geom.log2_page, (uint64_t)0x7fff0000);  // a stretch of pages on top fits
    s.q0 = min(max(p.batch.q_start[b], 0), T);
    const int end = p.batch.q_start[b + 1];  // past T: its last rows are not there
    s.n = max(min(max(end, 0), T) - s.q0, 0);
    if ((uint32_t)s.n * p.G < p.min_rows || (uint32_t)s.n * p.G >= p.max_rows) s.n = 0;  // another launch's
    // a sequence may be longer than its row of the table: its tokens have the positions
    // that its length gives them, its keys end where the table does
    s.first = s.n ? max(p.batch.kv_len[b], 0) - (end - s.q0) : 0;
    s.keys = min(max(s.first + s.n, 0), cap);
    s.lo = 0;
    if (p.window) s.lo = (int)min(max((int64_t)s.first + 1 - (int64_t)p.window, (int64_t)0), (int64_t)s.keys) / (int)kStep * (int)kStep;
    const uint32_t G = p.G;
    s.tiles = (uint32_t)(((uint64_t)s.n * G + R - 1) / R);
    s.steps = max((uint32_t)(s.keys - s.lo + (int)kStep - 1) / kStep, 1u);
    s.cost = (uint64_t)p.geom.Hkv * s.tiles * (kItemCost + s.steps);
    return s;
}

// The work is one line: of every sequence, KV head and row tile (an item)
// kItemCost for its overhead, then its key steps.  A wave takes an even share of
// the line wherever it begins and ends, so batches of any lengths fill the chip
// alike and no wave waits for another until the end, when an item that several
// waves of a workgroup took is gathered by the first of them, through LDS; items
// of several workgroups leave partial rows in the workspace, which
// paged_attn_join_kernel joins in order.  The next step's tiles are loaded before
// the present one is computed, and page numbers 32 steps ahead, a lane each.
// Bound by the cache's bytes once there are enough of them: four requests of
// 131072 keys (Q4_0, D = 128, 604 MB) 110 us, 5.5 TB/s (with codes less 8, then times
// the scale, 6 more: vector instructions count there too); 64 requests of 1 .. 8192
// keys (Q8_0, 110 MB) 31 us, 24 of them this kernel; one of 1000 keys 12 us, a chain
// of descriptor, page table, key and join latencies; drafted tokens and short
// chunks (two row blocks) by turning codes into fp16 on one wave per SIMD.
template <int FMT, int D, int NR>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PagedAttnParams p, uint32_t groups) {
    constexpr uint32_t R = 16 * NR;
    constexpr int DT = D / 16, KK = D / 32;
    constexpr int RUN = D / 4;  // dims of a lane's run
    // Codes past the caches: one row tile, Q4_0.  us without / with: four requests of
    // 131072 keys 113.5 / 109, one 40 / 37.6, 64 of 8192 113 / 108.5.  Q8_0, whose lines
    // are longer runs: 64 of 1 .. 8192 30.4 / 31.0, 64 of 1024 36.0 / 35.3, one of 131072
    // 62.7 / 63.6.  Two row blocks (more tiles that read them again): Q4_0 24.4 / 24.8.
    constexpr bool kOnce = FMT == QUANT_Q4_0 && NR == 1;

    const int lane = threadIdx.x & 63;
    const int j = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = blockIdx.x * kWaves + wave;
    const uint32_t workers = groups * kWaves;
    ItemNote* note = reinterpret_cast<ItemNote*>(p.ws) + blockIdx.x;
    // rows of waves 1 .. 3 that finish or carry on an item of the wave before them
    __shared__ __attribute__((aligned(16))) f4_t xo[kWaves - 1][NR][DT][64];
    __shared__ float xs[kWaves - 1][NR][64][2];
    __shared__ int head_of[kWaves];  // 0: none, 1: it ends in that wave's share, 2: it goes on

    // ---- this wave's share [s0, s1) and the item in which it begins ----
    const uint32_t per = (p.batch.B + 63) / 64;
    const uint32_t b_lo = min(lane * per, p.batch.B), b_hi = min(b_lo + per, p.batch.B);
    uint64_t mine = 0;
    Seq held{};  // up to 64 sequences: a lane's own, to be taken from it
    for (uint32_t x = b_lo; x < b_hi; x++) {
        held = seq_of(p, x, R);
        mine += held.cost;
    }
    uint64_t incl = mine;
    for (uint32_t o = 1; o < min(p.batch.B, 64u); o <<= 1) {
        const uint64_t x = __shfl_up((unsigned long long)incl, o);
        if ((uint32_t)lane >= o) incl += x;
    }
    const uint64_t total = lane_u64(incl, (int)min(p.batch.B, 64u) - 1);
    const uint64_t nw = min((uint64_t)workers, total >= (uint64_t)kLongShare * kMaxWaves ? kMaxWaves : min(total, (uint64_t)kFewWaves));
    if (threadIdx.x == 0) *note = ItemNote{};
    if (lane == 0) head_of[wave] = 0;
    uint64_t s0 = 0, s1 = 0;
    if (w < nw) share_of(total, (uint32_t)nw, w, s0, s1);
    uint32_t b = 0;
    uint64_t off = 0;
    if (incl - mine <= s0 && s0 < incl) {
        off = s0 - (incl - mine);
        for (b = b_lo; b + 1 < b_hi; b++) {
            const uint64_t cost = seq_of(p, b, R).cost;
            if (off < cost) break;
            off -= cost;
        }
    }
    const int at = max(__ffsll((unsigned long long)__ballot(incl - mine <= s0 && s0 < incl)) - 1, 0);
    b = __builtin_amdgcn_readlane(b, at);
    off = lane_u64(off, at);

    float c = p.scale * 1.4426950408889634f;  // log2 units
    const bool neg = c < 0.0f;
    if (neg) c = -c;
    c = fmaxf(c, 1.17549435e-38f);  // a scale of zero weighs seen keys alike, and hidden ones (-infinity times it) not
    const uint32_t G = p.G;
    const h2_t one2 = {(_Float16)1.0f, (_Float16)1.0f};
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;

    const typename Tile<FMT, D>::Offsets at_lane(p.geom, lane);

    // the item at work: its rows, and their running state
    f4_t o[NR][DT];
    float m_run[NR], l_run[NR];
    Seq s{};
    uint32_t hk = 0, rt = 0, rows = 0;
    bool open = false, begun = false;  // it goes on in the next wave's share; its first step was here

    auto row_of = [&](const RowsView& v, uint32_t r) {
        const uint32_t f = rt * R + r;
        return v.p + (int64_t)(s.q0 + (int)(f / G)) * v.ts + (int64_t)(hk * G + f % G) * v.hs;
    };
    // lane (j, g): row j of each 16, dims RUN g + DT r + dt
    auto emit = [&]() {
#pragma unroll
        for (int q = 0; q < NR; q++) {
            const uint32_t r = 16 * q + j;
            if (r >= rows) continue;
            _Float16* dst = row_of(p.O, r) + g * RUN;
            const float inv = l_run[q] == 0.0f ? 0.0f : 1.0f / l_run[q];
#pragma unroll
            for (int e = 0; e < RUN; e += 8) {
                h8_t y;
#pragma unroll
                for (int x = 0; x < 8; x++) y[x] = (_Float16)(o[q][(e + x) % DT][(e + x) / DT] * inv);
                *reinterpret_cast<h8_t*>(dst + e) = y;
            }
        }
    };
    auto leave = [&](int which) {
        float* slot = slot_of<D, R>(p.ws, groups, blockIdx.x, which);
#pragma unroll
        for (int q = 0; q < NR; q++) {
            const uint32_t r = 16 * q + j;
            if (r >= rows) continue;
#pragma unroll
            for (int e = 0; e < RUN; e += 4)
                *reinterpret_cast<f4_t*>(slot + r * D + g * RUN + e) =
                    f4_t{o[q][e % DT][e / DT], o[q][(e + 1) % DT][(e + 1) / DT], o[q][(e + 2) % DT][(e + 2) / DT],
                         o[q][(e + 3) % DT][(e + 3) / DT]};
            if (g == 0) {
                slot[R * D + r] = m_run[q];
                slot[R * D + R + r] = l_run[q];
            }
        }
    };

    for (uint64_t cur = s0; cur < s1 && b < p.batch.B;) {
        if (per == 1) {
            s.q0 = __builtin_amdgcn_readlane(held.q0, b);
            s.n = __builtin_amdgcn_readlane(held.n, b);
            s.first = __builtin_amdgcn_readlane(held.first, b);
            s.keys = __builtin_amdgcn_readlane(held.keys, b);
            s.lo = __builtin_amdgcn_readlane(held.lo, b);
            s.tiles = __builtin_amdgcn_readlane(held.tiles, b);
            s.steps = __builtin_amdgcn_readlane(held.steps, b);
            s.cost = lane_u64(held.cost, b);
        } else {
            s = seq_of(p, b, R);
        }
        if (off >= s.cost) {
            b++;
            off = 0;
            continue;
        }
        // this share of the item: its line from o0 on, steps u0 .. u0 + nu
        const uint32_t line = kItemCost + s.steps;
        const uint32_t item = (uint32_t)udiv(off, line), o0 = (uint32_t)(off - (uint64_t)item * line);
        const uint32_t o1 = (uint32_t)min((uint64_t)line, o0 + (s1 - cur));
        cur += o1 - o0;
        off += o1 - o0;
        if (o1 <= kItemCost) continue;
        const uint32_t u0 = o0 > kItemCost ? o0 - kItemCost : 0, nu = o1 - kItemCost - u0;
        hk = s.tiles == 1 ? item : item / s.tiles;
        rt = item - hk * s.tiles;

        // ---- rows: the last key that each sees (none behind the table), and the first ----
        auto last_seen = [&](int i) { return min(s.first + i, s.keys - 1); };
        auto first_seen = [&](int i) { return p.window ? (int)max((int64_t)s.first + i + 1 - (int64_t)p.window, (int64_t)0) : 0; };
        rows = min(R, (uint32_t)s.n * G - rt * R);
        const int i_first = (int)(rt * R / G), i_last = (int)((rt * R + rows - 1) / G);
        int lim[NR], low[NR];
        h8_t qf[NR][KK];
#pragma unroll
        for (int q = 0; q < NR; q++) {
            const uint32_t r = 16 * q + j;
            const uint32_t f = rt * R + min(r, rows - 1);
            const int i = (int)(f / G);
            const uint32_t h = hk * G + f % G;
            lim[q] = last_seen(i);
            low[q] = first_seen(i);
            const _Float16* src = p.Q.p + (int64_t)(s.q0 + i) * p.Q.ts + (int64_t)h * p.Q.hs + g * RUN;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                qf[q][kk] = *reinterpret_cast<const h8_t*>(src + 8 * kk);
                if (neg) qf[q][kk] = -qf[q][kk];
            }
        }
        const int lim_min = last_seen(i_first), lim_max = last_seen(i_last);
        const int low_min = first_seen(i_first), low_max = first_seen(i_last);

#pragma unroll
        for (int q = 0; q < NR; q++) {
            m_run[q] = kNone;
            l_run[q] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[q][dt] = f4_t{};
        }

        // ---- steps that some row sees something of: keys s.lo + kStep u .. + 31 ----
        const int key_base = s.lo;
        int ua = (int)u0, ub = (int)(u0 + nu);
        if (lim_max < key_base) ub = ua;
        else ub = min(ub, (lim_max - key_base) / (int)kStep + 1);
        if (low_min > key_base + 31) ua = max(ua, (low_min - key_base - 31 + (int)kStep - 1) / (int)kStep);
        // page numbers of the next 32 steps, a lane each 16 keys
        uint32_t page_ids = 0xffffffffu;
        int ids_from = ua - 32;
        auto fetch = [&](Tile<FMT, D> tile[2], int u) {
            if (u >= ids_from + 32) {
                ids_from = u;
                const int k0 = key_base + (u + (lane >> 1)) * (int)kStep + 16 * (lane & 1);
                page_ids = k0 < s.keys ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)k0 >> p.geom.log2_page)]
                                      : 0xffffffffu;
            }
            const int key0 = key_base + u * (int)kStep;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t page = __builtin_amdgcn_readlane(page_ids, 2 * (u - ids_from) + t);
                tile[t].there = page < p.geom.num_pages;
                const uint8_t* head = p.geom.pages + ((size_t)(tile[t].there ? page : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                tile[t].template load<kOnce>(head, at_lane, (uint32_t)(key0 + 16 * t) & pmask);
            }
        };
        auto step = [&](Tile<FMT, D> tile[2], int u) {
            const int key0 = key_base + u * (int)kStep;
            bool odd = false;  // some row does not see all keys, and some V value may not be finite
            f4_t sc[NR][2];
#pragma unroll
            for (int q = 0; q < NR; q++) sc[q][0] = sc[q][1] = f4_t{};
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    const h8_t a = tile[t].k_frag(kk);
#pragma unroll
                    for (int q = 0; q < NR; q++)
                        sc[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[q][kk], sc[q][t], 0, 0, 0);
                }
            if (key0 + 31 > lim_min || key0 < low_max || !tile[0].there || !tile[1].there) {
                // Some row does not see some key.  V scales of keys that nobody sees are
                // cleared: what was never written may be anything.
                uint32_t large = 0;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    uint32_t e[4] = {tile[t].vd.x & 0xffffu, tile[t].vd.x >> 16, tile[t].vd.y & 0xffffu, tile[t].vd.y >> 16};
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if (!tile[t].there || key0 + 16 * t + 4 * g + r >= s.keys) e[r] = 0;
                        large = max(large, e[r] & 0x7fffu);
                    }
                    tile[t].vd = u2_t{e[0] | e[1] << 16, e[2] | e[3] << 16};
#pragma unroll
                    for (int q = 0; q < NR; q++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int key = key0 + 16 * t + 4 * g + r;
                            if (!tile[t].there || key > lim[q] || key < low[q]) sc[q][t][r] = -INFINITY;
                        }
                }
                odd = __any(large >= kOddScale<FMT>);
            }
            h8_t pf[NR];
#pragma unroll
            for (int q = 0; q < NR; q++) {
                // Positive floats compare as integers do and negative ones are negative
                // integers, so an integer maximum (three at a time, no quieting of NaNs) tells
                // whether the reference point has to move.
                float ex[8];
                int top = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) ex[e] = __builtin_fmaf(sc[q][e >> 2][e & 3], c, -m_run[q]);
#pragma unroll
                for (int e = 0; e < 8; e += 2) top = max(max(top, (int)f32_bits(ex[e])), (int)f32_bits(ex[e + 1]));
                if (__any(top > kTop)) {
                    float mx = sc[q][0].x;
#pragma unroll
                    for (int e = 1; e < 8; e++) mx = fmaxf(mx, sc[q][e >> 2][e & 3]);
                    mx = __builtin_fmaf(mx, c, -kLift);
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m_new = fmaxf(m_run[q], mx);
                    const float alpha = __builtin_amdgcn_exp2f(m_run[q] - m_new);
                    m_run[q] = m_new;
                    l_run[q] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[q][dt] *= alpha;
#pragma unroll
                    for (int e = 0; e < 8; e++) ex[e] = __builtin_fmaf(sc[q][e >> 2][e & 3], c, -m_run[q]);
                }
                uint32_t pk[4];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const f2_t e = {__builtin_amdgcn_exp2f(ex[4 * t + r]), __builtin_amdgcn_exp2f(ex[4 * t + r + 1])};
                        const h2_t pp = __builtin_convertvector(e, h2_t);
                        pk[2 * t + r / 2] = as_u32(pp);
                        l_run[q] = __builtin_amdgcn_fdot2(pp, one2, l_run[q], false);
                    }
                pf[q] = __builtin_bit_cast(h8_t, u4_t{pk[0], pk[1], pk[2], pk[3]});
            }
            if (__builtin_expect(odd, 0)) {
                auto seen = [&](int q) {
                    u4_t w{};
                    int l = lim[q] - key0, f = low[q] - key0;
                    asm volatile("" : "+v"(l), "+v"(f));  // formed anew for each dt: kept, registers would spill
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        const int key = 16 * (x >> 2) + 4 * g + (x & 3);
                        if (tile[x >> 2].there && key <= l && key >= f) w[x / 2] |= kSeen << (x & 1) * 16;
                    }
                    return __builtin_bit_cast(b8_t, w);
                };
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const u2_t a = tile[0].v_pairs(dt), e = tile[1].v_pairs(dt);
                    const h8_t vf = __builtin_bit_cast(h8_t, u4_t{a.x, a.y, e.x, e.y});
#pragma unroll
                    for (int q = 0; q < NR; q++) {
                        o[q][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(marks_of<false>(vf), seen(q), o[q][dt], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        o[q][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(marks_of<true>(vf), seen(q), o[q][dt], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    tile[0].clear_odd(dt, a);
                    tile[1].clear_odd(dt, e);
                    __builtin_amdgcn_sched_barrier(0);
                }
                tile[0].clear_scales();
                tile[1].clear_scales();
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u2_t a = tile[0].v_pairs(dt), e = tile[1].v_pairs(dt);
                const h8_t vf = __builtin_bit_cast(h8_t, u4_t{a.x, a.y, e.x, e.y});
#pragma unroll
                for (int q = 0; q < NR; q++) o[q][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[q], o[q][dt], 0, 0, 0);
            }
        };
        Tile<FMT, D> ta[2], tb[2];
        if (ua < ub) fetch(ta, ua);
#pragma unroll 1
        for (int u = ua; u < ub; u++) {
            if (u + 1 < ub) fetch(tb, u + 1);
            step(ta, u);
            ta[0] = tb[0];
            ta[1] = tb[1];
        }
#pragma unroll
        for (int q = 0; q < NR; q++) {
            l_run[q] += __shfl_xor(l_run[q], 16);
            l_run[q] += __shfl_xor(l_run[q], 32);
        }
        const bool ends = u0 + nu == s.steps;
        begun = u0 == 0;
        open = !ends;
        if (begun && ends) {
            emit();
        } else if (!begun && wave > 0) {
#pragma unroll
            for (int q = 0; q < NR; q++) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) xo[wave - 1][q][dt][lane] = o[q][dt];
                xs[wave - 1][q][lane][0] = m_run[q];
                xs[wave - 1][q][lane][1] = l_run[q];
            }
            if (lane == 0) head_of[wave] = ends ? 1 : 2;
            open = false;  // the wave before gathers it
        } else if (!begun && ends) {
            leave(0);
            if (lane == 0) note->head = 1;
        }
    }

    // ---- an item that goes on takes the rows of the waves after this one, in order ----
    __syncthreads();
    if (!open) return;
    bool ended = false;
    for (uint32_t v = wave + 1; v < kWaves && !ended; v++) {
#pragma unroll
        for (int q = 0; q < NR; q++) {
            const float m2 = xs[v - 1][q][lane][0], l2 = xs[v - 1][q][lane][1];
            const float m = fmaxf(m_run[q], m2);
            const float fa = __builtin_amdgcn_exp2f(m_run[q] - m), fb = __builtin_amdgcn_exp2f(m2 - m);
            m_run[q] = m;
            l_run[q] = l_run[q] * fa + l2 * fb;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[q][dt] = o[q][dt] * fa + xo[v - 1][q][dt][lane] * fb;
        }
        ended = __builtin_amdgcn_readfirstlane(head_of[v]) == 1;
    }
    if (ended && begun) {
        emit();
        return;
    }
    leave(begun ? 1 : 0);
    if (lane != 0) return;
    if (begun) {
        note->hk = hk;
        note->first = rt * R;
        note->rows = rows;
        note->q0 = (uint32_t)s.q0;
        note->tail = 1;
    } else {
        note->head = ended ? 1 : 2;
    }
}

// Joins the partial rows of the items that begin in the shares of this block's
// workgroups: slot 1 of the first, then slot 0 of those after it.  D / 4 lanes hold
// a row; rows side by side while an item has few parts, else the parts of a row
// are split over the lane groups, whose sums meet in LDS in a fixed order.
constexpr uint32_t kJoinBlocks = 512;
template <int D, int R>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PagedAttnParams p, uint32_t groups) {
    constexpr int L = D / 4, GROUPS = 256 / L, U = 4;
    __shared__ f4_t part_sum[256];
    const uint32_t per = (groups + gridDim.x - 1) / gridDim.x, w1 = min((blockIdx.x + 1) * per, groups);
    const ItemNote* notes = reinterpret_cast<const ItemNote*>(p.ws);
    const uint32_t tid = threadIdx.x, lane = tid & 63, l4 = tid % L, group = tid / L;
    const uint32_t G = p.G;
    // 32 notes at a time to begin at, and those behind them to end at, a lane each
    for (uint32_t base = blockIdx.x * per; base < w1; base += 32) {
        ItemNote mine{};
        if (base + lane < groups) mine = notes[base + lane];
        uint64_t todo = __ballot(lane < 32 && base + lane < w1 && mine.tail);
        const uint64_t stops = __ballot(mine.head != 2);
        while (todo) {
            const int at = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            const uint32_t w = base + at;
            const uint32_t hk = __builtin_amdgcn_readlane(mine.hk, at), first = __builtin_amdgcn_readlane(mine.first, at);
            const uint32_t rows = __builtin_amdgcn_readlane(mine.rows, at), q0 = __builtin_amdgcn_readlane(mine.q0, at);
            // parts: up to the first workgroup in which it ends
            uint32_t parts = 0;
            const uint64_t behind = at < 63 ? stops >> (at + 1) : 0;
            if (behind) parts = __ffsll((unsigned long long)behind) + 1;
            for (uint32_t k = base + 64; parts == 0 && k < groups; k += 64) {
                const uint64_t end = __ballot(k + lane >= groups || notes[k + lane].head != 2);
                if (end) parts = k - w + __ffsll((unsigned long long)end);
            }
            parts = parts ? min(parts, groups - w) : groups - w;
            auto slot = [&](uint32_t k) { return slot_of<D, R>(p.ws, groups, w + k, k == 0 ? 1 : 0); };
            uint32_t split = 1;
            while (split < GROUPS && parts > U * split) split *= 2;
            const uint32_t side = GROUPS / split, mine0 = group % split;
            for (uint32_t r0 = blockIdx.y * side; r0 < rows; r0 += gridDim.y * side) {
                const uint32_t r = r0 + group / split;
                const bool live = r < rows;
                // reference points and sums, a lane each part, and the first rows, all under way together
                float m = kNone, l = 0.0f, mk[U];
                f4_t v[U], o{};
                if (live && l4 < parts) {
                    m = slot(l4)[R * D + r];
                    l = slot(l4)[R * D + R + r];
                }
#pragma unroll
                for (int i = 0; i < U; i++) {
                    v[i] = f4_t{};
                    mk[i] = -INFINITY;
                    const uint32_t k = mine0 + i * split;
                    if (live && k < parts) {
                        v[i] = *reinterpret_cast<const f4_t*>(slot(k) + r * D + 4 * l4);
                        mk[i] = slot(k)[R * D + r];
                    }
                }
                if (live)
                    for (uint32_t k = l4 + L; k < parts; k += L) {
                        const float m2 = slot(k)[R * D + r], m_new = fmaxf(m, m2);
                        l = l * __builtin_amdgcn_exp2f(m - m_new) + slot(k)[R * D + R + r] * __builtin_amdgcn_exp2f(m2 - m_new);
                        m = m_new;
                    }
                const float m_lane = m;
#pragma unroll
                for (int x = L / 2; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
                l *= __builtin_amdgcn_exp2f(m_lane - m);
#pragma unroll
                for (int x = L / 2; x >= 1; x >>= 1) l += __shfl_xor(l, x);
#pragma unroll
                for (int i = 0; i < U; i++)
                    if (live && mine0 + i * split < parts) o += v[i] * __builtin_amdgcn_exp2f(mk[i] - m);
                if (live) {
#pragma unroll 4
                    for (uint32_t k = mine0 + U * split; k < parts; k += split) {
                        const float* x = slot(k);
                        o += *reinterpret_cast<const f4_t*>(x + r * D + 4 * l4) * __builtin_amdgcn_exp2f(x[R * D + r] - m);
                    }
                }
                if (split > 1) {
                    __syncthreads();
                    part_sum[tid] = o;
                    __syncthreads();
                    if (mine0 == 0)
                        for (uint32_t k = 1; k < split; k++) o += part_sum[tid + k * L];
                }
                if (live && mine0 == 0) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const uint32_t f = first + r;
                    _Float16* dst = p.O.p + (int64_t)(q0 + f / G) * p.O.ts + (int64_t)(hk * G + f % G) * p.O.hs;
                    const f2_t a = {o.x * inv, o.y * inv}, b = {o.z * inv, o.w * inv};
                    *reinterpret_cast<u2_t*>(dst + 4 * l4) =
                        u2_t{as_u32(__builtin_convertvector(a, h2_t)), as_u32(__builtin_convertvector(b, h2_t))};
                }
            }
        }
    }
}

// ---- chunks: 32 rows a wave, the keys' tiles shared through LDS ----------------

struct Chunk {
    uint32_t tile_tokens, tiles;  // tokens of a row tile, row tiles
};

// Steps (key tiles of KT) of row tile rt, and its first key.
template <int KT>
__device__ __forceinline__ uint32_t steps_of(const PagedAttnParams& p, const Seq& s, uint32_t tokens, uint32_t rt, int& lo) {
    const int64_t first = (int64_t)s.first + rt * tokens;
    const int end = (int)min(first + tokens, (int64_t)s.keys);
    lo = p.window ? (int)min(max(first + 1 - (int64_t)p.window, (int64_t)0), (int64_t)s.keys) / KT * KT : 0;
    return end <= lo ? 1u : (uint32_t)(end - lo + KT - 1) / KT;
}

// A workgroup of NW waves takes 32 NW rows (whole tokens' query heads) and an even
// share of the line of all row tiles' key tiles, as above.  Key tiles of 16 NW
// keys: every thread turns 32 bytes of K and of V codes (Q4_0: 16) into fp16 in a
// double-buffered LDS tile, the codes loaded two tiles ahead; then each wave
// takes its rows over the tile, 32 x 32 scores at a time.  256 rows share the work
// of turning codes (128 rows: 1306 us where 256 take 1140).  2048 tokens over 30000
// keys (D = 128, 972 GFLOP) 1067 us with the join, 0.91 PFLOP/s.  Counters: the matrix
// pipe 44% busy, 8.1 vector operations per MFMA beside it, LDS bank conflicts in 0.23 M
// of a CU's 1.98 M cycles (V's tile is stored by lanes four rows apart), at 1.9 GHz of 2.2.
template <int FMT, int D, int NW>
__global__ void __launch_bounds__(64 * NW, 2) paged_attn_chunk_kernel(PagedAttnParams p, uint32_t groups) {
    constexpr int R = 32 * NW, KT = 16 * NW, UNITS = KT / 32;
    constexpr int DT = D / 32, KK = D / 16;
    constexpr int KU = D / 8, VU = KT / 8;       // 16-byte units of a K row (a key), of a V^T row (a dim)
    constexpr int KB = KT * D * 2, TB = 2 * KB;  // bytes of a K tile, of a tile
    constexpr int RUN = D / 4;                   // dims of a K task: a quarter of a key
    constexpr int DV = D / 32;                   // dims of a V task: 8 keys of each
    constexpr int KW = FMT == QUANT_Q8_0 ? RUN / 4 : RUN / 8, VW = FMT == QUANT_Q8_0 ? DV : DV / 2;
    constexpr uint32_t CB = 4 * KW * 4, NB = D / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    // of each 16 keys: 1, their page is one of the cache's; 2, not all rows see all keys of
    // the tile, and some V value of these may not be finite
    __shared__ int there[2][NW];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 5, j = lane & 31;
    ItemNote* note = reinterpret_cast<ItemNote*>(p.ws) + blockIdx.x;
    const uint32_t G = p.G, tokens = R / G;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;

    // ---- this workgroup's share [s0, s1) ----
    auto heads_cost = [&](const Seq& s) {  // of one KV head's row tiles
        uint64_t c = 0;
        int lo;
        const uint32_t tiles = ((uint32_t)s.n + tokens - 1) / tokens;
        for (uint32_t rt = 0; rt < tiles; rt++) c += kChunkCost + steps_of<KT>(p, s, tokens, rt, lo);
        return c;
    };
    const uint32_t per = (p.batch.B + 63) / 64;
    const uint32_t b_lo = min(lane * per, p.batch.B), b_hi = min(b_lo + per, p.batch.B);
    uint64_t mine = 0;
    for (uint32_t x = b_lo; x < b_hi; x++) mine += heads_cost(seq_of(p, x, R)) * p.geom.Hkv;
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up((unsigned long long)incl, o);
        if (lane >= o) incl += x;
    }
    const uint64_t total = lane_u64(incl, 63);
    const uint64_t nw = max(min((uint64_t)groups, total / kChunkMin), (uint64_t)1);
    if (tid == 0) *note = ItemNote{};
    if (blockIdx.x >= nw || total == 0) return;
    uint64_t s0, s1;
    share_of(total, (uint32_t)nw, blockIdx.x, s0, s1);
    uint32_t b = 0;
    uint64_t off = 0;
    const bool here = incl - mine <= s0 && s0 < incl;
    if (here) {
        off = s0 - (incl - mine);
        for (b = b_lo; b + 1 < b_hi; b++) {
            const uint64_t cost = heads_cost(seq_of(p, b, R)) * p.geom.Hkv;
            if (off < cost) break;
            off -= cost;
        }
    }
    const int at = max(__ffsll((unsigned long long)__ballot(here)) - 1, 0);
    b = __builtin_amdgcn_readlane(b, at);
    off = lane_u64(off, at);

    float c = p.scale * 1.4426950408889634f;  // log2 units
    const bool neg = c < 0.0f;
    if (neg) c = -c;
    c = fmaxf(c, 1.17549435e-38f);

    // Unit u of row r of a tile sits at u ^ swz(r).  A row's units differ from one
    // base by the exclusive or of 16 times their number: the bases alone are kept
    // (hidden from the compiler, which would keep every sum).
    auto swz = [](int units, uint32_t r) -> uint32_t { return units == 16 ? (r & 15u) : ((r ^ (r >> 3)) & 7u); };
    auto place = [&](int units, uint32_t r, uint32_t u) { return r * (units * 16u) + 16u * (u ^ swz(units, r & 31u)); };
    uint32_t kof = place(KU, (uint32_t)j, (uint32_t)g), vof = place(VU, (uint32_t)j, (uint32_t)g);
    // tasks: K, a quarter of key 16 wave + lane / 4; V, dims DV (lane % 32) .. of
    // unit 2 wave + lane / 32, i.e. keys 16 wave + 4 g + {0 .. 3, 8 .. 11}
    const uint32_t kkey = lane >> 2, kq = lane & 3, vdim = DV * (uint32_t)j;
    uint32_t kst = place(KU, 16 * wave + kkey, kq * (RUN / 8)), vst = place(VU, vdim, 2 * wave + g);
    uint32_t kld = kkey * CB + kq * (KW * 4), vld = p.geom.v_off + g * (4 * CB) + vdim * (4 * CB / D);
    uint32_t ksl = p.geom.ks_off + (kkey * NB + kq * NB / 4) * 2, vsl = p.geom.vs_off + (g * NB + vdim / 32) * 8;
    const h2_t one2 = {(_Float16)1.0f, (_Float16)1.0f};

    f16v_t o[DT];
    float m_run = kNone, l_run = 0.0f;
    Seq s{};
    uint64_t row_cost = 0;  // of a KV head of the sequence at work
    uint32_t at_b = 0xffffffffu;

    for (uint64_t cur = s0; cur < s1 && b < p.batch.B;) {
        if (b != at_b) {
            s = seq_of(p, b, R);
            row_cost = lane_u64(heads_cost(s), 0);
            at_b = b;
        }
        if (off >= row_cost * p.geom.Hkv) {
            b++;
            off = 0;
            continue;
        }
        const uint32_t hk = (uint32_t)udiv(off, row_cost);
        uint64_t in_row = off - hk * row_cost;
        uint32_t rt = 0, steps;
        int lo;
        for (;; rt++) {  // the row tile at this place
            steps = __builtin_amdgcn_readfirstlane(steps_of<KT>(p, s, tokens, rt, lo));
            if (in_row < kChunkCost + steps) break;
            in_row -= kChunkCost + steps;
        }
        const uint32_t line = kChunkCost + steps, o0 = (uint32_t)in_row;
        const uint32_t o1 = (uint32_t)min((uint64_t)line, o0 + (s1 - cur));
        cur += o1 - o0;
        off += o1 - o0;
        if (o1 <= kChunkCost) continue;
        const int u0 = (int)(o0 > kChunkCost ? o0 - kChunkCost : 0), u1 = (int)(o1 - kChunkCost);
        const bool begun = u0 == 0, ends = u1 == (int)steps;

        // ---- rows ----
        const uint32_t rows = min(tokens * G, ((uint32_t)s.n - rt * tokens) * G);
        const int i0 = (int)(rt * tokens);  // the tile's first token
        const uint32_t r = 32 * wave + j, rc = min(r, rows - 1);
        const bool wave_live = 32u * wave < rows;
        // the last key that a row sees (none behind the table), and the first
        auto last_seen = [&](uint32_t r) { return min(s.first + i0 + (int)(r / G), s.keys - 1); };
        auto first_seen = [&](uint32_t r) {
            return p.window ? (int)max((int64_t)s.first + i0 + (int)(r / G) + 1 - (int64_t)p.window, (int64_t)0) : 0;
        };
        const int lim = last_seen(rc), low = first_seen(rc);
        // of this wave's rows, and of all
        const uint32_t r0 = min(32u * wave, rows - 1), r1 = min(32u * wave + 31, rows - 1);
        const int lim0 = last_seen(r0), lim1 = last_seen(r1), low0 = first_seen(r0), low1 = first_seen(r1);
        const int all0 = last_seen(0), all_low1 = first_seen(rows - 1);
        h8_t qf[KK];
        {
            const _Float16* src = p.Q.p + (int64_t)(s.q0 + (int)(rt * tokens + rc / G)) * p.Q.ts +
                                  (int64_t)(hk * G + rc % G) * p.Q.hs + 8 * g;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                qf[kk] = *reinterpret_cast<const h8_t*>(src + 16 * kk);
                if (neg) qf[kk] = -qf[kk];
            }
        }
        m_run = kNone;
        l_run = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) o[t] = f16v_t{};

        // ---- codes of a tile into registers, and from there into LDS ----
        uint32_t kw[KW], vw[2][VW], kd = 0;
        u2_t vd[2];
        bool mine_there = false;
        uint32_t page_ids = 0;
        int ids_from = u0 - 64;
        auto fetch = [&](int u) {
            if (u >= ids_from + 64) {
                ids_from = u;
                const int k0 = lo + (u + lane) * KT + 16 * wave;
                page_ids = k0 < s.keys ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)k0 >> p.geom.log2_page)]
                                      : 0xffffffffu;
            }
            const uint32_t page = __builtin_amdgcn_readlane(page_ids, u - ids_from);
            mine_there = page < p.geom.num_pages;
            const uint32_t slot = (uint32_t)(lo + u * KT + 16 * wave) & pmask;
            const uint8_t* head = p.geom.pages + ((size_t)(mine_there ? page : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
            const auto rs = make_rsrc(head, p.geom.head_bytes);
            fetch_words<KW>(rs, kld, slot * CB, kw);
            kd = __builtin_amdgcn_raw_buffer_load_b16(rs, ksl, slot * (NB * 2), 0);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                fetch_words<VW>(rs, vld + 2 * h * (4 * CB), slot * CB, vw[h]);
                vd[h] = __builtin_amdgcn_raw_buffer_load_b64(rs, vsl + 2 * h * NB * 8, slot * (NB * 2), 0);
            }
        };
        auto fill = [&](int u) {
            uint8_t* buf = smem + (u & 1) * TB;
            const int k0 = lo + u * KT;
            asm volatile("" : "+v"(kst), "+v"(vst));
            const h2_t d = as_h2(kd | kd << 16);
#pragma unroll
            for (int kk = 0; kk < RUN / 8; kk++)
                *reinterpret_cast<h8_t*>(buf + (kst ^ 16u * kk)) = k_octet<FMT>(kw, kk, d);
            int odd = 0;
            if (k0 + KT - 1 > all0 || k0 < all_low1 || !mine_there) {
                // not all rows see all of the tile's keys: V scales of keys that none sees are cleared
                uint32_t large = 0;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t e[4] = {vd[h].x & 0xffffu, vd[h].x >> 16, vd[h].y & 0xffffu, vd[h].y >> 16};
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        if (!mine_there || k0 + 16 * wave + 4 * g + 8 * h + x >= s.keys) e[x] = 0;
                        large = max(large, e[x] & 0x7fffu);
                    }
                    vd[h] = u2_t{e[0] | e[1] << 16, e[2] | e[3] << 16};
                }
                odd = __any(large >= kOddScale<FMT>) ? 2 : 0;
            }
            if (lane == 0) there[u & 1][wave] = odd | (mine_there || k0 + 16 * wave >= s.keys);
#pragma unroll
            for (int x = 0; x < DV; x++) {
                const u2_t a = v_quad<FMT>(vw[0], x, vd[0]), e = v_quad<FMT>(vw[1], x, vd[1]);
                *reinterpret_cast<u4_t*>(buf + KB + x * (VU * 16) + (vst ^ 16u * x)) = u4_t{a.x, a.y, e.x, e.y};
            }
        };

        // ---- this wave's rows over a tile, 32 keys (a unit) at a time ----
        auto scores = [&](const uint8_t* buf, int x) {
            const uint8_t* kb = buf + x * 32 * (KU * 16);
            f16v_t sc{};
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8_t*>(kb + (kof ^ 32u * kk)), qf[kk], sc, 0, 0, 0);
            return sc;
        };
        // Exponents of a unit's weights, beside the reference point; whether that has to
        // move, an integer maximum tells, as above.
        auto settle = [&](const f16v_t& sc, float ex[16], int top) {
            if (__any(top > kTop)) {
                float mx = sc[0];
#pragma unroll
                for (int e = 1; e < 16; e++) mx = fmaxf(mx, sc[e]);
                mx = __builtin_fmaf(mx, c, -kLift);
                const float m_new = fmaxf(m_run, fmaxf(mx, __shfl_xor(mx, 32)));
                const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int t = 0; t < DT; t++) o[t] *= alpha;
#pragma unroll
                for (int e = 0; e < 16; e++) ex[e] = __builtin_fmaf(sc[e], c, -m_run);
            }
        };
        auto exponents = [&](const f16v_t& sc, float ex[16]) {
            int top = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) ex[e] = __builtin_fmaf(sc[e], c, -m_run);
#pragma unroll
            for (int e = 0; e < 16; e += 2) top = max(max(top, (int)f32_bits(ex[e])), (int)f32_bits(ex[e + 1]));
            settle(sc, ex, top);
        };
        auto weigh = [&](const float ex[16], uint32_t pk[8]) {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const f2_t w = {__builtin_amdgcn_exp2f(ex[e]), __builtin_amdgcn_exp2f(ex[e + 1])};
                const h2_t pp = __builtin_convertvector(w, h2_t);
                pk[e >> 1] = as_u32(pp);
                l_run = __builtin_amdgcn_fdot2(pp, one2, l_run, false);
            }
        };
        auto add = [&](const uint8_t* buf, int x, const uint32_t pk[8]) {
#pragma unroll
            for (int t2 = 0; t2 < 2; t2++) {
                const h8_t pf = __builtin_bit_cast(h8_t, u4_t{pk[4 * t2], pk[4 * t2 + 1], pk[4 * t2 + 2], pk[4 * t2 + 3]});
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    const h8_t va = *reinterpret_cast<const h8_t*>(buf + KB + t * 32 * (VU * 16) + (vof ^ 32u * (2 * x + t2)));
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pf, o[t], 0, 0, 0);
                }
            }
        };
        // the same where some values may not be finite, and rows do not see all keys
        auto add_marked = [&](const uint8_t* buf, int x, const uint32_t pk[8], int u) {
            const int key0 = lo + u * KT + 32 * x;
#pragma unroll
            for (int t2 = 0; t2 < 2; t2++) {
                const h8_t pf = __builtin_bit_cast(h8_t, u4_t{pk[4 * t2], pk[4 * t2 + 1], pk[4 * t2 + 2], pk[4 * t2 + 3]});
                u4_t seen{};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = key0 + 16 * t2 + 8 * (e >> 2) + 4 * g + (e & 3);
                    if ((there[u & 1][2 * x + t2] & 1) && key <= lim && key >= low) seen[e / 2] |= kSeen << (e & 1) * 16;
                }
                const b8_t sf = __builtin_bit_cast(b8_t, seen);
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    const h8_t va = *reinterpret_cast<const h8_t*>(buf + KB + t * 32 * (VU * 16) + (vof ^ 32u * (2 * x + t2)));
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(marks_of<false>(va), sf, o[t], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(marks_of<true>(va), sf, o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(finite_part(va), pf, o[t], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        auto attend = [&](int u) {
            const uint8_t* buf = smem + (u & 1) * TB;
            asm volatile("" : "+v"(kof), "+v"(vof));
            const int k0 = lo + u * KT;
            if (!wave_live || k0 > lim1 || k0 + KT - 1 < low0) return;
            int every = 1, some = 0;
#pragma unroll
            for (int x = 0; x < NW; x++) {
                every &= there[u & 1][x];
                some |= there[u & 1][x];
            }
            const bool all_there = every & 1;
            if (!(k0 + KT - 1 > all0 || k0 < all_low1 || !all_there)) {
                // every row sees every key.  Each line below ends at a barrier for the scheduler:
                // one MFMA, the loads of operands four MFMAs ahead, and the vector work that
                // runs beside it -- a unit's exponentials beside the next one's scores (the
                // matrix pipe leaves the transcendental unit free), the next one's exponents
                // beside this one's values.
                auto key = [&](int x, int kk) {
                    return *reinterpret_cast<const h8_t*>(buf + x * 32 * (KU * 16) + (kof ^ 32u * kk));
                };
                auto value = [&](int x, int i) {
                    return *reinterpret_cast<const h8_t*>(buf + KB + (i % DT) * 32 * (VU * 16) + (vof ^ 32u * (2 * x + i / DT)));
                };
                constexpr int NV = 2 * DT;
                h8_t kf[4], vf[4];
#pragma unroll
                for (int i = 0; i < 4; i++) kf[i] = key(0, i);
                f16v_t sc{};
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kk & 3], qf[kk], sc, 0, 0, 0);
                    kf[kk & 3] = kk + 4 < KK ? key(0, kk + 4) : key(1, kk + 4 - KK);
                }
                float ex[16];
                exponents(sc, ex);
#pragma unroll
                for (int x = 0; x < UNITS; x++) {
                    uint32_t pk[8];
                    auto pair = [&](int e) {
                        const f2_t w = {__builtin_amdgcn_exp2f(ex[2 * e]), __builtin_amdgcn_exp2f(ex[2 * e + 1])};
                        const h2_t pp = __builtin_convertvector(w, h2_t);
                        pk[e] = as_u32(pp);
                        l_run = __builtin_amdgcn_fdot2(pp, one2, l_run, false);
                    };
                    __builtin_amdgcn_sched_barrier(0);
                    if (x + 1 < UNITS) {
                        sc = f16v_t{};
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) {
                            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kk & 3], qf[kk], sc, 0, 0, 0);
                            if (kk + 4 < KK) kf[kk & 3] = key(x + 1, kk + 4);
                            else vf[kk + 4 - KK] = value(x, kk + 4 - KK);
#pragma unroll
                            for (int e = 0; e < 8 / KK; e++) pair(kk * (8 / KK) + e);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) vf[i] = value(x, i);
#pragma unroll
                        for (int e = 0; e < 8; e++) pair(e);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    int top = 0;
#pragma unroll
                    for (int i = 0; i < NV; i++) {
                        const int t2 = i / DT, t = i % DT;
                        const h8_t pf = __builtin_bit_cast(h8_t, u4_t{pk[4 * t2], pk[4 * t2 + 1], pk[4 * t2 + 2], pk[4 * t2 + 3]});
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i & 3], pf, o[t], 0, 0, 0);
                        if (i + 4 < NV) vf[i & 3] = value(x, i + 4);
                        else if (x + 2 < UNITS) kf[i + 4 - NV] = key(x + 2, i + 4 - NV);
                        if (x + 1 < UNITS)
#pragma unroll
                            for (int e = i * (16 / NV); e < (i + 1) * (16 / NV); e += 2) {
                                ex[e] = __builtin_fmaf(sc[e], c, -m_run);
                                ex[e + 1] = __builtin_fmaf(sc[e + 1], c, -m_run);
                                top = max(max(top, (int)f32_bits(ex[e])), (int)f32_bits(ex[e + 1]));
                            }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (x + 1 < UNITS) settle(sc, ex, top);
                }
                return;
            }
            auto unit = [&](int x, bool marks) {
                const int key0 = k0 + 32 * x;
                if (key0 > lim1 || key0 + 31 < low0) return;
                f16v_t sc = scores(buf, x);
                if (key0 + 31 > lim0 || key0 < low1 || !all_there) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int key = key0 + 8 * (e >> 2) + 4 * g + (e & 3);
                        if (key > lim || key < low || !(there[u & 1][2 * x + (e >> 3)] & 1)) sc[e] = -INFINITY;
                    }
                }
                float ex[16];
                exponents(sc, ex);
                uint32_t pk[8];
                weigh(ex, pk);
                if (marks) add_marked(buf, x, pk, u);
                else add(buf, x, pk);
            };
            if (__builtin_amdgcn_readfirstlane(some) & 2) {
#pragma unroll 1
                for (int x = 0; x < UNITS; x++) unit(x, true);
                return;
            }
#pragma unroll
            for (int x = 0; x < UNITS; x++) unit(x, false);
        };

        fetch(u0);
        fill(u0);
        if (u0 + 1 < u1) fetch(u0 + 1);
        __syncthreads();
        for (int u = u0; u < u1; u++) {
            if (u + 1 < u1) fill(u + 1);
            if (u + 2 < u1) fetch(u + 2);
            attend(u);
            __syncthreads();
        }

        l_run += __shfl_xor(l_run, 32);
        // lane (j, g): row 32 wave + j, dims 32 t + 8 (e / 4) + 4 g + e % 4
        if (begun && ends) {
            if (r < rows) {
                const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
                _Float16* dst = p.O.p + (int64_t)(s.q0 + (int)(rt * tokens + r / G)) * p.O.ts + (int64_t)(hk * G + r % G) * p.O.hs;
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f2_t x = {o[t][4 * q] * inv, o[t][4 * q + 1] * inv}, y = {o[t][4 * q + 2] * inv, o[t][4 * q + 3] * inv};
                        *reinterpret_cast<u2_t*>(dst + 32 * t + 8 * q + 4 * g) =
                            u2_t{as_u32(__builtin_convertvector(x, h2_t)), as_u32(__builtin_convertvector(y, h2_t))};
                    }
            }
        } else {
            float* slot = slot_of<D, R>(p.ws, groups, blockIdx.x, begun ? 1 : 0);
            if (r < rows) {
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        *reinterpret_cast<f4_t*>(slot + r * D + 32 * t + 8 * q + 4 * g) =
                            f4_t{o[t][4 * q], o[t][4 * q + 1], o[t][4 * q + 2], o[t][4 * q + 3]};
                if (g == 0) {
                    slot[R * D + r] = m_run;
                    slot[R * D + R + r] = l_run;
                }
            }
            if (tid == 0) {
                if (begun) {
                    note->hk = hk;
                    note->first = rt * tokens * G;
                    note->rows = rows;
                    note->q0 = (uint32_t)s.q0;
                    note->tail = 1;
                } else {
                    note->head = ends ? 1 : 2;
                }
            }
        }
    }
}

// Row tiles by the rows of the longest chunk, workgroups by the length of the line
// expected.  Any expectation is right, so every product stays within 64 bits.  A
// batch whose chunks are worth theirs, but not all of whose sequences are as long (T
// says so), is taken apart, sequences of kChunkTile / 2 rows and more for chunks: a
// row tile there is as much work for one token as for 64.  us of chunks alone / both:
// 2048 tokens beside 63 single ones 523 / 387, four of 512 beside 60 270 / 178, 512
// beside 31 (Q4_0) 199 / 113; three prompts of 700 .. 2048, for which the other
// kernels run in vain, 119 / 124.  From a little more work than chunks alone: 512
// beside 63 (9/8 of kChunkWork) by rows altogether 100, both 116; prompts of 1500
// and 700 (12/8) 99 and 82.
static AttnPlan plan_of(const PagedAttnParams& p) {
    auto at_most = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
    const uint64_t G = p.G, max_new = p.max_new ? p.max_new : 1, rows = max_new * G;
    uint64_t keys = p.max_kv ? p.max_kv : 1;
    if (p.window) keys = at_most(keys, (uint64_t)p.window + max_new);
    const bool mixed = p.batch.T < p.batch.B * max_new && p.batch.B > 1;
    const uint64_t least = mixed ? kChunkWork * 5 / 4 : kChunkWork;
    const bool chunks = rows >= kChunkTile / 2 && G <= kChunkTile && (uint64_t)p.batch.T * p.H >= (least + keys - 1) / keys;
    const uint64_t heads = at_most((uint64_t)p.batch.B * p.geom.Hkv, 1u << 31);
    auto tiles_of = [&](uint32_t of) { return heads * at_most((rows + of - 1) / of, 1u << 31); };
    AttnPlan a{};
    a.both = chunks && mixed;
    if (chunks) {
        const uint64_t tiles = tiles_of(kChunkTile), some = at_most(tiles, kChunkGroups * kChunkMin);
        const uint64_t want = some * (keys / (kChunkTile / 2) + 1 + kChunkCost) / kChunkMin + 1;
        a.many = {kChunkTile, (uint32_t)at_most(want, kChunkGroups), (uint32_t)at_most(tiles, 0xffffffffu)};
    }
    if (!chunks || mixed) {
        const uint32_t of = (chunks ? G : rows) <= 16 ? 16 : 32;
        const uint64_t tiles = chunks ? heads : tiles_of(of), some = at_most(tiles, kMaxWaves * kMinSteps);
        const uint64_t want = (some * (keys / kStep + 1 + kItemCost) + kMinSteps - 1) / kMinSteps;
        a.few = {of, (uint32_t)(at_most(want, kMaxWaves) + kWaves - 1) / kWaves, (uint32_t)at_most(tiles, 0xffffffffu)};
    }
    return a;
}

template <int D>
static size_t ws_bytes(const WorkPlan& w) {
    const size_t slot = w.rows == 16 ? slot_bytes<D, 16>() : (w.rows == 32 ? slot_bytes<D, 32>() : slot_bytes<D, kChunkTile>());
    return (size_t)w.groups * (sizeof(ItemNote) + 2 * slot);
}

size_t paged_attn_workspace(const PagedAttnParams& p) {
    const AttnPlan a = plan_of(p);
    return p.D == 64 ? ws_bytes<64>(a.few) + ws_bytes<64>(a.many) : ws_bytes<128>(a.few) + ws_bytes<128>(a.many);
}

template <int D, int R>
static hipError_t launch_join(const PagedAttnParams& p, const WorkPlan& w, hipStream_t st) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Blocks for each few workgroups, over which the rows of an item are spread: more
    // where items have many parts.  us of the whole call with 4 / 16 of them: 64 tokens
    // over 16384 keys (32 parts an item) 82 / 42, one token 27 / 23, 64 requests (one
    // part) 34 / 40.
    const uint32_t parts = w.groups / w.items, across = R > 32 ? 32 : (parts >= 16 ? 16 : (parts >= 8 ? 8 : 4));
    const uint32_t most = 4 * kJoinBlocks / across;
    const dim3 grid(w.groups < most ? w.groups : most, across);
    hipLaunchKernelGGL((paged_attn_join_kernel<D, R>), grid, dim3(256), 0, st, p, w.groups);
    return hipGetLastError();
}

template <int FMT, int D>
static hipError_t launch_format(PagedAttnParams p, hipStream_t st) {
    const AttnPlan a = plan_of(p);
    constexpr uint32_t cut = kChunkTile / 2;
    p.min_rows = 0;
    p.max_rows = a.both ? cut : 0xffffffffu;
    if (a.few.groups) {
        const dim3 grid(a.few.groups), block(64 * kWaves);
        hipError_t e;
        if (a.few.rows == 16) {
            hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 1>), grid, block, 0, st, p, a.few.groups);
            e = launch_join<D, 16>(p, a.few, st);
        } else {
            hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 2>), grid, block, 0, st, p, a.few.groups);
            e = launch_join<D, 32>(p, a.few, st);
        }
        if (e != hipSuccess) return e;
    }
    if (!a.many.groups) return hipSuccess;
    p.ws += ws_bytes<D>(a.few);
    p.min_rows = a.both ? cut : 0;
    p.max_rows = 0xffffffffu;
    constexpr int NW = kChunkTile / 32;
    constexpr size_t lds = 2 * 2 * 16 * NW * D * 2;
    static size_t attr[kMaxDevices] = {};  // more than the default 64 KB of LDS
    const hipError_t e = lds_limit_once((const void*)paged_attn_chunk_kernel<FMT, D, NW>, lds, attr);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_attn_chunk_kernel<FMT, D, NW>), dim3(a.many.groups), dim3(64 * NW), lds, st, p, a.many.groups);
    return launch_join<D, kChunkTile>(p, a.many, st);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, hipStream_t st) {
    if (p.batch.B == 0 || p.batch.T == 0) return hipSuccess;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_format<QUANT_Q8_0, 64>(p, st) : launch_format<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_format<QUANT_Q4_0, 64>(p, st) : launch_format<QUANT_Q4_0, 128>(p, st);
}

}  // namespace qr
