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
// the write of its rows.  64 requests of 1 .. 8192 keys: 4 and 8 the same within
// noise; shares by steps alone, with a join of four waves an item, 44 us, now 33.
constexpr uint32_t kItemCost = 4;
// Waves of a launch: two per SIMD, what the registers allow with the next step's
// tiles in flight (three without them: 47 us there), at least kMinSteps of the
// line each.
constexpr uint32_t kMaxWaves = 2048, kMinSteps = 2;
constexpr float kNone = -3.402823466e38f;  // reference point of a row that has seen no score above -infinity

// A workgroup's note of an item that begins in its share of the work and ends in
// later ones': how many workgroups took part.
struct ItemNote {
    uint32_t b, hk, rt, parts;
};

struct WorkPlan {
    uint32_t nr, groups;
};

// values 1024 + 128 + q of four Q8_0 bytes, as pairs
__device__ __forceinline__ h2_t q8_lo(uint32_t w, h2_t d) {
    const h2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return (as_h2(nib_pair_lo(w)) - off) * d;
}
__device__ __forceinline__ h2_t q8_hi(uint32_t w, h2_t d) {
    const h2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return (as_h2(nib_pair_hi(w)) - off) * d;
}
template <bool HI>
__device__ __forceinline__ h2_t q4_pair(uint32_t codes, h2_t d) {
    const h2_t off = {(_Float16)8.0f, (_Float16)8.0f};
    return (code_pair<HI>(codes) - off) * d;
}

// A lane's share of 16 keys: W words of K codes (D / 4 dims of one key) and of V
// codes (D / 16 dims of four keys), its K scale and four V scales.
template <int FMT, int D>
struct Tile {
    static constexpr int W = FMT == QUANT_Q8_0 ? D / 16 : D / 32;
    uint32_t k[W], v[W];
    uint32_t kd;
    u2_t vd;
    bool there;  // its page is one of the cache's

    __device__ __forceinline__ void load(const uint8_t* head, const PageGeom& g, uint32_t slot0, int lane) {
        constexpr uint32_t CB = 4 * W * 4, NB = D / 32;  // bytes of a key's codes, blocks
        const uint32_t j = lane & 15, q = lane >> 4;
        const uint8_t* kp = head + (slot0 + j) * CB + q * (W * 4);
        const uint8_t* vp = head + g.v_off + ((slot0 >> 2) + q) * (4 * CB) + j * (W * 4);
        load_words(kp, k);
        load_words(vp, v);
        kd = *reinterpret_cast<const uint16_t*>(head + g.ks_off + ((slot0 + j) * NB + q * NB / 4) * 2);
        vd = *reinterpret_cast<const u2_t*>(head + g.vs_off + (((slot0 >> 2) + q) * NB + j * NB / 16) * 8);
    }
    __device__ __forceinline__ static void load_words(const uint8_t* p, uint32_t w[W]) {
        if constexpr (W == 2) {
            const u2_t a = *reinterpret_cast<const u2_t*>(p);
            w[0] = a.x;
            w[1] = a.y;
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; i++) {
                const u4_t a = reinterpret_cast<const u4_t*>(p)[i];
                w[4 * i] = a.x;
                w[4 * i + 1] = a.y;
                w[4 * i + 2] = a.z;
                w[4 * i + 3] = a.w;
            }
        }
    }
    // operand of contraction step kk: dims 8 kk .. 8 kk + 7 of the lane's run
    __device__ __forceinline__ h8_t k_frag(int kk) const {
        const h2_t d = as_h2(kd | kd << 16);
        h2_t a, b, c, e;
        if constexpr (FMT == QUANT_Q8_0) {
            a = q8_lo(k[2 * kk], d);
            b = q8_hi(k[2 * kk], d);
            c = q8_lo(k[2 * kk + 1], d);
            e = q8_hi(k[2 * kk + 1], d);
        } else {
            const uint32_t lo = k[kk] & 0x0f0f0f0fu, hi = k[kk] >> 4 & 0x0f0f0f0fu;
            a = q4_pair<false>(lo, d);
            b = q4_pair<true>(lo, d);
            c = q4_pair<false>(hi, d);
            e = q4_pair<true>(hi, d);
        }
        return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
    }
    // the four keys of dim dt of the lane's run, as two pairs
    __device__ __forceinline__ u2_t v_pairs(int dt) const {
        const uint32_t s0 = vd.x, s1 = vd.y;
        if constexpr (FMT == QUANT_Q8_0)
            return u2_t{as_u32(q8_lo(v[dt], as_h2(s0))), as_u32(q8_hi(v[dt], as_h2(s1)))};
        const uint32_t w = (dt & 1 ? v[dt / 2] >> 4 : v[dt / 2]) & 0x0f0f0f0fu;
        return u2_t{as_u32(q4_pair<false>(w, as_h2(s0))), as_u32(q4_pair<true>(w, as_h2(s1)))};
    }
};

template <int D, int NR>
__host__ __device__ constexpr size_t slot_bytes() {
    return (size_t)16 * NR * (D + 2) * 4;
}
// workspace: a note per workgroup, then two slots per workgroup of partial rows
// (O [R][D], reference points [R], sums [R], fp32)
template <int D, int NR>
__device__ __forceinline__ float* slot_of(uint8_t* ws, uint32_t groups, uint32_t w, int which) {
    return reinterpret_cast<float*>(ws + (size_t)groups * sizeof(ItemNote) + ((size_t)w * 2 + which) * slot_bytes<D, NR>());
}

// lane `at`'s value, as a wave-uniform one
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int at) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), at) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, at);
}

struct Seq {
    int q0, n, len, lo;   // first row, new tokens, keys, first key that any row sees (a multiple of kStep)
    uint32_t tiles, steps;  // row tiles and key steps per tile
    uint64_t cost;
};
__device__ __forceinline__ Seq seq_of(const PagedAttnParams& p, uint32_t b, uint32_t R) {
    Seq s;
    const int T = (int)p.batch.T;
    const int cap = (int)min((uint64_t)p.batch.table_pages << p.geom.log2_page, (uint64_t)0x7fffffff);
    s.q0 = min(max(p.batch.q_start[b], 0), T);
    s.n = max(min(max(p.batch.q_start[b + 1], 0), T) - s.q0, 0);
    s.len = min(max(p.batch.kv_len[b], 0), cap);
    s.lo = 0;
    if (p.window) s.lo = (int)(max((int64_t)s.len - s.n + 1 - (int64_t)p.window, (int64_t)0) / kStep * kStep);
    const uint32_t G = p.H / p.geom.Hkv;
    s.tiles = (uint32_t)(((uint64_t)s.n * G + R - 1) / R);
    s.steps = max((uint32_t)(s.len - s.lo + (int)kStep - 1) / kStep, 1u);
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
// 131072 keys (Q4_0, D = 128, 604 MB) 127 us, 4.8 TB/s; 64 requests of 1 .. 8192
// keys (Q8_0, 110 MB) 33 us of which 4 are the join; one of 1000 keys 13.6 us, a
// chain of descriptor, page table, key and join latencies.
template <int FMT, int D, int NR>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PagedAttnParams p, uint32_t groups) {
    constexpr uint32_t R = 16 * NR;
    constexpr int DT = D / 16, KK = D / 32;
    constexpr int RUN = D / 4;  // dims of a lane's run

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
    for (uint32_t x = b_lo; x < b_hi; x++) mine += seq_of(p, x, R).cost;
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up((unsigned long long)incl, o);
        if (lane >= o) incl += x;
    }
    const uint64_t total = lane_u64(incl, 63);
    const uint64_t nw = min((uint64_t)workers, total);
    if (threadIdx.x == 0) *note = ItemNote{0, 0, 0, 0};
    if (lane == 0) head_of[wave] = 0;
    const uint64_t s0 = w < nw ? total * w / nw : 0, s1 = w < nw ? total * (w + 1) / nw : 0;
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
    const uint32_t G = p.H / p.geom.Hkv;
    const h2_t one2 = {(_Float16)1.0f, (_Float16)1.0f};
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;

    // the item at work: its rows, and their running state
    f4_t o[NR][DT];
    float m_run[NR], l_run[NR];
    Seq s{};
    uint32_t b_open = 0, hk = 0, rt = 0, rows = 0;
    uint64_t last = 0;            // its last place on the line
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
        float* slot = slot_of<D, NR>(p.ws, groups, blockIdx.x, which);
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
        s = seq_of(p, b, R);
        if (off >= s.cost) {
            b++;
            off = 0;
            continue;
        }
        // this share of the item: its line from o0 on, steps u0 .. u0 + nu
        const uint32_t line = kItemCost + s.steps;
        const uint32_t o0 = (uint32_t)(off % line), item = (uint32_t)(off / line);
        const uint32_t o1 = (uint32_t)min((uint64_t)line, o0 + (s1 - cur));
        cur += o1 - o0;
        off += o1 - o0;
        if (o1 <= kItemCost) continue;
        const uint32_t u0 = o0 > kItemCost ? o0 - kItemCost : 0, nu = o1 - kItemCost - u0;
        hk = item / s.tiles;
        rt = item % s.tiles;
        b_open = b;
        last = cur - o1 + line - 1;
        const int p0 = s.len - s.n;  // position of the first new token

        // ---- rows ----
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
            lim[q] = p0 + i;
            low[q] = p.window ? (int)max((int64_t)lim[q] + 1 - (int64_t)p.window, (int64_t)0) : 0;
            const _Float16* src = p.Q.p + (int64_t)(s.q0 + i) * p.Q.ts + (int64_t)h * p.Q.hs + g * RUN;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                qf[q][kk] = *reinterpret_cast<const h8_t*>(src + 8 * kk);
                if (neg) qf[q][kk] = -qf[q][kk];
            }
        }
        const int lim_min = p0 + i_first, lim_max = p0 + i_last;
        const int low_min = p.window ? (int)max((int64_t)lim_min + 1 - (int64_t)p.window, (int64_t)0) : 0;
        const int low_max = p.window ? (int)max((int64_t)lim_max + 1 - (int64_t)p.window, (int64_t)0) : 0;

        uint32_t poison = 0;  // bit q: the row saw a V scale that is not finite
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
                page_ids = k0 < s.len ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)k0 >> p.geom.log2_page)]
                                      : 0xffffffffu;
            }
            const int key0 = key_base + u * (int)kStep;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t page = __builtin_amdgcn_readlane(page_ids, 2 * (u - ids_from) + t);
                tile[t].there = page < p.geom.num_pages;
                const uint8_t* head = p.geom.pages + ((size_t)(tile[t].there ? page : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                tile[t].load(head, p.geom, (uint32_t)(key0 + 16 * t) & pmask, lane);
            }
        };
        auto step = [&](Tile<FMT, D> tile[2], int u) {
            const int key0 = key_base + u * (int)kStep;
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
            if (key0 + 31 > lim_min || key0 < low_max || key0 + 31 >= s.len || !tile[0].there || !tile[1].there) {
                // Some row does not see some key.  What such a key's V holds must
                // not reach that row through 0 times infinity: V scales of keys
                // that nobody sees are cleared, and scales that are not finite
                // are cleared and noted for the rows that do see them.
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    uint32_t bad = 0;
                    uint32_t e[4] = {tile[t].vd.x & 0xffffu, tile[t].vd.x >> 16, tile[t].vd.y & 0xffffu, tile[t].vd.y >> 16};
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int key = key0 + 16 * t + 4 * g + r;
                        const bool dead = !tile[t].there || key >= s.len;
                        if (!dead && (e[r] & 0x7c00u) == 0x7c00u) bad |= 1u << r;
                        if (dead || (bad >> r & 1)) e[r] = 0;
                    }
                    tile[t].vd = u2_t{e[0] | e[1] << 16, e[2] | e[3] << 16};
                    if (__any(bad != 0)) {
                        // lane (j, g) owns output dims of block g NB / 4 of its row; the scales
                        // of block i are lanes j = i * 16 / NB's
                        constexpr int NB = D / 32;
                        for (int key = 0; key < 16; key++) {
                            const uint32_t theirs = (uint32_t)__shfl((int)bad, (key >> 2) * 16 + (g * NB / 4) * (16 / NB));
                            if (!(theirs >> (key & 3) & 1)) continue;
                            const int at = key0 + 16 * t + key;
#pragma unroll
                            for (int q = 0; q < NR; q++)
                                if (at <= lim[q] && at >= low[q]) poison |= 1u << q;
                        }
                    }
#pragma unroll
                    for (int q = 0; q < NR; q++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int key = key0 + 16 * t + 4 * g + r;
                            if (!tile[t].there || key > lim[q] || key < low[q]) sc[q][t][r] = -INFINITY;
                        }
                }
            }
            h8_t pf[NR];
#pragma unroll
            for (int q = 0; q < NR; q++) {
                // the reference point moves only when a score exceeds it by 2^8
                float mx = fmaxf(fmaxf(fmaxf(sc[q][0].x, sc[q][0].y), fmaxf(sc[q][0].z, sc[q][0].w)),
                                 fmaxf(fmaxf(sc[q][1].x, sc[q][1].y), fmaxf(sc[q][1].z, sc[q][1].w))) * c;
                if (__any(mx > m_run[q] + 8.0f)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m_new = fmaxf(m_run[q], mx);
                    const float alpha = __builtin_amdgcn_exp2f(m_run[q] - m_new);
                    m_run[q] = m_new;
                    l_run[q] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[q][dt] *= alpha;
                }
                uint32_t pk[4];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const f2_t e = {__builtin_amdgcn_exp2f(__builtin_fmaf(sc[q][t][r], c, -m_run[q])),
                                        __builtin_amdgcn_exp2f(__builtin_fmaf(sc[q][t][r + 1], c, -m_run[q]))};
                        const h2_t pp = __builtin_convertvector(e, h2_t);
                        pk[2 * t + r / 2] = as_u32(pp);
                        l_run[q] = __builtin_amdgcn_fdot2(pp, one2, l_run[q], false);
                    }
                pf[q] = __builtin_bit_cast(h8_t, u4_t{pk[0], pk[1], pk[2], pk[3]});
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
        if (poison) {
#pragma unroll
            for (int q = 0; q < NR; q++)
                if (poison >> q & 1)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[q][dt] = f4_t{NAN, NAN, NAN, NAN};
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
    if (begun && lane == 0)
        *note = ItemNote{b_open, hk, rt, (uint32_t)((((last + 1) * nw - 1) / total) / kWaves) - blockIdx.x + 1};
}

// Joins the partial rows of the items that begin in the shares of this block's
// workgroups: slot 1 of the first, then slot 0 of those after it.  D / 4 lanes hold
// a row; rows side by side while an item has few parts, else the parts of a row
// are split over the lane groups, whose sums meet in LDS in a fixed order.
constexpr uint32_t kJoinBlocks = 512;
template <int D, int NR>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PagedAttnParams p, uint32_t groups) {
    constexpr uint32_t R = 16 * NR;
    constexpr int L = D / 4, GROUPS = 256 / L;
    __shared__ f4_t part_sum[256];
    const uint32_t per = (groups + gridDim.x - 1) / gridDim.x, w0 = blockIdx.x * per;
    const uint32_t w1 = min(w0 + per, groups);
    const ItemNote* notes = reinterpret_cast<const ItemNote*>(p.ws);
    const uint32_t tid = threadIdx.x, l4 = tid % L, group = tid / L;
    const uint32_t G = p.H / p.geom.Hkv;
    for (uint32_t base = w0; base < w1; base += 64) {
        const uint32_t mine = base + (tid & 63);
        uint64_t todo = __ballot(mine < w1 && notes[mine].parts >= 2);
        while (todo) {
            const uint32_t w = base + __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            const ItemNote note = notes[w];
            const Seq s = seq_of(p, note.b, R);
            const uint32_t rows = min(R, (uint32_t)s.n * G - note.rt * R), parts = note.parts;
            auto slot = [&](uint32_t k) { return slot_of<D, NR>(p.ws, groups, w + k, k == 0 ? 1 : 0); };
            uint32_t split = 1;
            while (split < GROUPS && parts > 4 * split) split *= 2;
            const uint32_t side = GROUPS / split;
            for (uint32_t r0 = blockIdx.y * side; r0 < rows; r0 += gridDim.y * side) {
                const uint32_t r = r0 + group / split;
                const bool live = r < rows;
                float m = kNone, l = 0.0f;
                f4_t o{};
                if (live)
                    for (uint32_t k = l4; k < parts; k += L) m = fmaxf(m, slot(k)[R * D + r]);
#pragma unroll
                for (int x = L / 2; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
                if (live) {
                    for (uint32_t k = l4; k < parts; k += L)
                        l += slot(k)[R * D + R + r] * __builtin_amdgcn_exp2f(slot(k)[R * D + r] - m);
#pragma unroll 4
                    for (uint32_t k = group % split; k < parts; k += split) {
                        const float* x = slot(k);
                        o += *reinterpret_cast<const f4_t*>(x + r * D + 4 * l4) * __builtin_amdgcn_exp2f(x[R * D + r] - m);
                    }
                }
#pragma unroll
                for (int x = L / 2; x >= 1; x >>= 1) l += __shfl_xor(l, x);
                if (split > 1) {
                    __syncthreads();
                    part_sum[tid] = o;
                    __syncthreads();
                    if (group % split == 0)
                        for (uint32_t k = 1; k < split; k++) o += part_sum[tid + k * L];
                }
                if (live && group % split == 0) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const uint32_t f = note.rt * R + r;
                    _Float16* dst = p.O.p + (int64_t)(s.q0 + (int)(f / G)) * p.O.ts + (int64_t)(note.hk * G + f % G) * p.O.hs;
                    const f2_t a = {o.x * inv, o.y * inv}, b = {o.z * inv, o.w * inv};
                    *reinterpret_cast<u2_t*>(dst + 4 * l4) =
                        u2_t{as_u32(__builtin_convertvector(a, h2_t)), as_u32(__builtin_convertvector(b, h2_t))};
                }
            }
        }
    }
}

// Row tiles by the rows of the longest chunk, workgroups by the length of the line expected.
static WorkPlan plan_of(const PagedAttnParams& p) {
    const uint64_t G = p.H / p.geom.Hkv, rows = (uint64_t)(p.max_new ? p.max_new : 1) * G;
    WorkPlan w;
    w.nr = rows <= 16 ? 1 : 2;
    const uint64_t R = 16 * w.nr;
    uint64_t keys = p.max_kv ? p.max_kv : 1;
    if (p.window) keys = keys < (uint64_t)p.window + p.max_new ? keys : (uint64_t)p.window + p.max_new;
    const uint64_t tiles = (rows + R - 1) / R;
    const uint64_t line = (uint64_t)p.batch.B * p.geom.Hkv * tiles * (keys / kStep + 1 + kItemCost);
    const uint64_t want = (line + kMinSteps - 1) / kMinSteps;
    w.groups = (uint32_t)((want < kMaxWaves ? want : kMaxWaves) + kWaves - 1) / kWaves;
    return w;
}

template <int D>
static size_t ws_bytes(const WorkPlan& w) {
    const size_t slot = w.nr == 1 ? slot_bytes<D, 1>() : slot_bytes<D, 2>();
    return (size_t)w.groups * (sizeof(ItemNote) + 2 * slot);
}

size_t paged_attn_workspace(const PagedAttnParams& p) {
    const WorkPlan w = plan_of(p);
    return p.D == 64 ? ws_bytes<64>(w) : ws_bytes<128>(w);
}

template <int FMT, int D, int NR>
static hipError_t launch_rows(const PagedAttnParams& p, uint32_t groups, hipStream_t st) {
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, NR>), dim3(groups), dim3(64 * kWaves), 0, st, p, groups);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // four blocks for each few workgroups: the rows of an item in several parts are spread over them
    const dim3 join(groups < kJoinBlocks ? groups : kJoinBlocks, 4);
    hipLaunchKernelGGL((paged_attn_join_kernel<D, NR>), join, dim3(256), 0, st, p, groups);
    return hipGetLastError();
}

template <int FMT, int D>
static hipError_t launch_format(const PagedAttnParams& p, hipStream_t st) {
    const WorkPlan w = plan_of(p);
    return w.nr == 1 ? launch_rows<FMT, D, 1>(p, w.groups, st) : launch_rows<FMT, D, 2>(p, w.groups, st);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, hipStream_t st) {
    if (p.batch.B == 0 || p.batch.T == 0) return hipSuccess;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_format<QUANT_Q8_0, 64>(p, st) : launch_format<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_format<QUANT_Q4_0, 64>(p, st) : launch_format<QUANT_Q4_0, 128>(p, st);
}

}  // namespace qr
