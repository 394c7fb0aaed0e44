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

constexpr int kWaves = 4;
constexpr uint32_t kUnit = 32 * kWaves;  // keys that a workgroup takes per step
constexpr float kNone = -3.402823466e38f;  // reference point of a row that has seen no score above -infinity

// A worker's note of an item that begins in its share of the work and ends in
// later ones': how many workers took part.
struct ItemNote {
    uint32_t b, hk, rt, workers;
};

struct WorkPlan {
    uint32_t nr, workers;
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
// workspace: a note per worker, then two slots per worker of partial rows
// (O [R][D], reference points [R], sums [R], fp32)
template <int D, int NR>
__device__ __forceinline__ float* slot_of(uint8_t* ws, uint32_t workers, uint32_t w, int which) {
    return reinterpret_cast<float*>(ws + (size_t)workers * sizeof(ItemNote) + ((size_t)w * 2 + which) * slot_bytes<D, NR>());
}

struct Seq {
    int q0, n, len, lo;   // first row, new tokens, keys, first key that any row sees (a multiple of kUnit)
    uint32_t tiles, units;  // row tiles and key steps per tile
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
    if (p.window) s.lo = (int)(max((int64_t)s.len - s.n + 1 - (int64_t)p.window, (int64_t)0) / kUnit * kUnit);
    const uint32_t G = p.H / p.geom.Hkv;
    s.tiles = (uint32_t)(((uint64_t)s.n * G + R - 1) / R);
    s.units = max((uint32_t)(s.len - s.lo + (int)kUnit - 1) / kUnit, 1u);
    s.cost = (uint64_t)p.geom.Hkv * s.tiles * s.units;
    return s;
}

// The work is one line of key steps: of every sequence, KV head and row tile.
// A workgroup takes an even share of it wherever it begins and ends, so batches
// of any lengths fill the chip alike; items that cross a boundary leave
// partial rows in the workspace, which paged_attn_join_kernel joins in order.
template <int FMT, int D, int NR>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PagedAttnParams p, uint32_t workers) {
    constexpr uint32_t R = 16 * NR;
    constexpr int DT = D / 16, KK = D / 32;
    constexpr int RUN = D / 4;  // dims of a lane's run
    __shared__ uint64_t wave_sum[kWaves];
    __shared__ uint64_t start_off;
    __shared__ uint32_t start_b;
    __shared__ __attribute__((aligned(16))) float xo[2][NR][DT][64][4];
    __shared__ float xs[2][NR][64][2];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, g = lane >> 4;
    const uint32_t w = blockIdx.x;
    ItemNote* note = reinterpret_cast<ItemNote*>(p.ws) + w;

    // ---- this worker's share [s0, s1) ----
    const uint32_t per = (p.batch.B + 255) / 256;
    const uint32_t b_lo = min(tid * per, p.batch.B), b_hi = min(b_lo + per, p.batch.B);
    uint64_t mine = 0;
    for (uint32_t b = b_lo; b < b_hi; b++) mine += seq_of(p, b, R).cost;
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up((unsigned long long)incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint64_t total = 0, before = incl - mine;
    for (int k = 0; k < kWaves; k++) {
        if (k < wave) before += wave_sum[k];
        total += wave_sum[k];
    }
    const uint64_t nw = min((uint64_t)workers, total);
    if (tid == 0) *note = ItemNote{0, 0, 0, 0};
    if (w >= nw) return;
    const uint64_t s0 = total * w / nw, s1 = total * (w + 1) / nw;
    if (before <= s0 && s0 < before + mine) {
        uint64_t at = before;
        for (uint32_t b = b_lo; b < b_hi; b++) {
            const uint64_t c = seq_of(p, b, R).cost;
            if (s0 < at + c) {
                start_b = b;
                start_off = s0 - at;
                break;
            }
            at += c;
        }
    }
    __syncthreads();
    uint32_t b = __builtin_amdgcn_readfirstlane(start_b);
    uint64_t off = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(start_off >> 32)) << 32 |
                   __builtin_amdgcn_readfirstlane((uint32_t)start_off);

    float c = p.scale * 1.4426950408889634f;  // log2 units
    const bool neg = c < 0.0f;
    if (neg) c = -c;
    c = fmaxf(c, 1.17549435e-38f);  // a scale of zero weighs seen keys alike, and hidden ones (-infinity times it) not
    const uint32_t G = p.H / p.geom.Hkv;
    const h2_t one2 = {(_Float16)1.0f, (_Float16)1.0f};
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;

    for (uint64_t cur = s0; cur < s1 && b < p.batch.B;) {
        const Seq s = seq_of(p, b, R);
        if (off >= s.cost) {
            b++;
            off = 0;
            continue;
        }
        const uint32_t u0 = (uint32_t)(off % s.units);
        const uint32_t item = (uint32_t)(off / s.units), hk = item / s.tiles, rt = item % s.tiles;
        const uint32_t nu = (uint32_t)min((uint64_t)(s.units - u0), s1 - cur);
        const int p0 = s.len - s.n;  // position of the first new token

        // ---- rows ----
        const uint32_t rows = min(R, (uint32_t)s.n * G - rt * R);
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

        f4_t o[NR][DT];
        float m_run[NR], l_run[NR];
        uint32_t poison = 0;  // bit q: the row saw a V scale that is not finite
#pragma unroll
        for (int q = 0; q < NR; q++) {
            m_run[q] = kNone;
            l_run[q] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[q][dt] = f4_t{};
        }

        for (uint32_t u = u0; u < u0 + nu; u++) {
            const int key0 = s.lo + (int)(u * kUnit) + 32 * wave;
            if (key0 > lim_max || key0 + 31 < low_min || key0 >= s.len) continue;
            Tile<FMT, D> tile[2];
            bool there[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int k0 = key0 + 16 * t;
                const uint32_t pi = (uint32_t)k0 >> p.geom.log2_page;
                uint32_t page = 0xffffffffu;
                if (k0 < s.len) page = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + pi];
                there[t] = page < p.geom.num_pages;
                const uint8_t* head = p.geom.pages + ((size_t)(there[t] ? page : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                tile[t].load(head, p.geom, (uint32_t)k0 & pmask, lane);
            }
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
            if (key0 + 31 > lim_min || key0 < low_max || key0 + 31 >= s.len || !there[0] || !there[1]) {
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
                        const bool dead = !there[t] || key >= s.len;
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
                            if (!there[t] || key > lim[q] || key < low[q]) sc[q][t][r] = -INFINITY;
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
        }
        if (poison) {
#pragma unroll
            for (int q = 0; q < NR; q++)
                if (poison >> q & 1)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[q][dt] = f4_t{NAN, NAN, NAN, NAN};
        }

        // ---- the four waves' rows join: 2, 3 into 0, 1, then 1 into 0 ----
#pragma unroll
        for (int q = 0; q < NR; q++) {
            l_run[q] += __shfl_xor(l_run[q], 16);
            l_run[q] += __shfl_xor(l_run[q], 32);
        }
#pragma unroll
        for (int half = 2; half >= 1; half /= 2) {
            __syncthreads();
            if (wave >= half && wave < 2 * half) {
                const int x = wave - half;
#pragma unroll
                for (int q = 0; q < NR; q++) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f4_t*>(xo[x][q][dt][lane]) = o[q][dt];
                    xs[x][q][lane][0] = m_run[q];
                    xs[x][q][lane][1] = l_run[q];
                }
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int q = 0; q < NR; q++) {
                    const float m2 = xs[wave][q][lane][0], l2 = xs[wave][q][lane][1];
                    const float m = fmaxf(m_run[q], m2);
                    const float fa = __builtin_amdgcn_exp2f(m_run[q] - m), fb = __builtin_amdgcn_exp2f(m2 - m);
                    m_run[q] = m;
                    l_run[q] = l_run[q] * fa + l2 * fb;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        o[q][dt] = o[q][dt] * fa + *reinterpret_cast<const f4_t*>(xo[wave][q][dt][lane]) * fb;
                }
            }
        }
        const bool whole = nu == s.units;
        if (wave == 0) {
            // lane (j, g): row j of the tile's 16, dims RUN g + DT r + dt
            if (whole) {
#pragma unroll
                for (int q = 0; q < NR; q++) {
                    const uint32_t r = 16 * q + j;
                    if (r >= rows) continue;
                    const uint32_t f = rt * R + r;
                    _Float16* dst = p.O.p + (int64_t)(s.q0 + (int)(f / G)) * p.O.ts + (int64_t)(hk * G + f % G) * p.O.hs + g * RUN;
                    const float inv = l_run[q] == 0.0f ? 0.0f : 1.0f / l_run[q];
#pragma unroll
                    for (int e = 0; e < RUN; e += 8) {
                        h8_t y;
#pragma unroll
                        for (int x = 0; x < 8; x++) y[x] = (_Float16)(o[q][(e + x) % DT][(e + x) / DT] * inv);
                        *reinterpret_cast<h8_t*>(dst + e) = y;
                    }
                }
            } else {
                float* slot = slot_of<D, NR>(p.ws, workers, w, u0 == 0 ? 1 : 0);
#pragma unroll
                for (int q = 0; q < NR; q++) {
                    const uint32_t r = 16 * q + j;
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
                if (u0 == 0 && lane == 0) {
                    const uint64_t last = cur + s.units - 1;  // this item's last step, and who takes it
                    *note = ItemNote{b, hk, rt, (uint32_t)(((last + 1) * nw - 1) / total) - w + 1};
                }
            }
        }
        cur += nu;
        off += nu;
    }
}

// Joins the partial rows of the item that begins in worker blockIdx.x's share:
// its slot 1, then slot 0 of the workers after it.  One wave per row: lanes over
// the workers for their reference points and sums, then over dims.
template <int D, int NR>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PagedAttnParams p, uint32_t workers) {
    constexpr uint32_t R = 16 * NR;
    constexpr int E = D / 64;
    const uint32_t w = blockIdx.x;
    const ItemNote note = reinterpret_cast<const ItemNote*>(p.ws)[w];
    if (note.workers < 2) return;
    const int lane = threadIdx.x & 63;
    const uint32_t r = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t G = p.H / p.geom.Hkv;
    const int T = (int)p.batch.T, q0 = min(max(p.batch.q_start[note.b], 0), T);
    const uint32_t f = note.rt * R + r;
    if (q0 + (int)(f / G) >= min(max(p.batch.q_start[note.b + 1], 0), T)) return;
    auto slot = [&](uint32_t k) { return slot_of<D, NR>(p.ws, workers, w + k, k == 0 ? 1 : 0); };
    float m = kNone;
    for (uint32_t k = lane; k < note.workers; k += 64) m = fmaxf(m, slot(k)[R * D + r]);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    float l = 0.0f, o[E] = {};
    for (uint32_t k0 = 0; k0 < note.workers; k0 += 64) {
        const uint32_t n = min(64u, note.workers - k0);
        float weight = 0.0f;
        if ((uint32_t)lane < n) {
            const float* s = slot(k0 + lane) + R * D + r;
            weight = __builtin_amdgcn_exp2f(s[0] - m);
            l += s[R] * weight;
        }
#pragma unroll 4
        for (uint32_t k = 0; k < n; k++) {
            const float fa = bits_f32(__builtin_amdgcn_readlane(f32_bits(weight), k));
            const float* s = slot(k0 + k) + r * D;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] += s[64 * e + lane] * fa;
        }
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    _Float16* dst = p.O.p + (int64_t)(q0 + (int)(f / G)) * p.O.ts + (int64_t)(note.hk * G + f % G) * p.O.hs;
#pragma unroll
    for (int e = 0; e < E; e++) dst[64 * e + lane] = (_Float16)(o[e] * inv);
}

// Row tiles by the rows of the longest chunk, workers by the steps expected.
static WorkPlan plan_of(const PagedAttnParams& p) {
    const uint64_t G = p.H / p.geom.Hkv, rows = (uint64_t)(p.max_new ? p.max_new : 1) * G;
    WorkPlan w;
    w.nr = rows <= 16 ? 1 : 2;
    const uint64_t R = 16 * w.nr;
    uint64_t keys = p.max_kv ? p.max_kv : 1;
    if (p.window) keys = keys < (uint64_t)p.window + p.max_new ? keys : (uint64_t)p.window + p.max_new;
    const uint64_t units = (keys + kUnit - 1) / kUnit + 1;
    const uint64_t tiles = (rows + R - 1) / R;
    const uint64_t steps = (uint64_t)p.batch.B * p.geom.Hkv * tiles * units;
    w.workers = (uint32_t)(steps < 512 ? steps : 512);
    return w;
}

template <int D>
static size_t ws_bytes(const WorkPlan& w) {
    const size_t slot = w.nr == 1 ? slot_bytes<D, 1>() : slot_bytes<D, 2>();
    return (size_t)w.workers * (sizeof(ItemNote) + 2 * slot);
}

size_t paged_attn_workspace(const PagedAttnParams& p) {
    const WorkPlan w = plan_of(p);
    return p.D == 64 ? ws_bytes<64>(w) : ws_bytes<128>(w);
}

template <int FMT, int D, int NR>
static hipError_t launch_rows(const PagedAttnParams& p, uint32_t workers, hipStream_t st) {
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, NR>), dim3(workers), dim3(256), 0, st, p, workers);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_attn_join_kernel<D, NR>), dim3(workers, 4 * NR), dim3(256), 0, st, p, workers);
    return hipGetLastError();
}

template <int FMT, int D>
static hipError_t launch_format(const PagedAttnParams& p, hipStream_t st) {
    const WorkPlan w = plan_of(p);
    return w.nr == 1 ? launch_rows<FMT, D, 1>(p, w.workers, st) : launch_rows<FMT, D, 2>(p, w.workers, st);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, hipStream_t st) {
    if (p.batch.B == 0 || p.batch.T == 0) return hipSuccess;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_format<QUANT_Q8_0, 64>(p, st) : launch_format<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_format<QUANT_Q4_0, 64>(p, st) : launch_format<QUANT_Q4_0, 128>(p, st);
}

}  // namespace qr
