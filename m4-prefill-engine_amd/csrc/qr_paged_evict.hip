// qr_paged_evict.hip -- a bounded cache: the attention weight that each cached key has
// received, and eviction of the lightest.
#include <algorithm>

#include "qr_device.h"
#include "qr_paged.h"
#include "qr_paged_decode.h"

namespace qr {

// ---- weights received ----------------------------------------------------------
//
// sums[key] += sum over the rows of a KV head of exp(scale q . k - lse(row)), or = for a key
// of the call's own.  A row's lse is known, so nothing has to be joined over the keys: a wave
// holds its keys as fp16 operands in registers and takes the rows past them, S = Q . K^T with
// the keys as columns, so that a column's sum is lane-local but for the lanes that share it.
// Each sum is formed in one order by one wave or workgroup: no atomics.

// Keys of a wave of the rows kernel.
constexpr uint32_t kWaveKeys = 64;

struct WeighSeq {
    int q0, n, first, keys, lo;  // keys that the table holds and a row sees; the first that one sees
};
__device__ __forceinline__ WeighSeq weigh_seq(const WeighParams& p, uint32_t b) {
    const NewRows r = new_rows(p.batch, b);
    WeighSeq s{r.q0, r.n, r.first, 0, 0};
    if ((uint32_t)s.n * p.G < p.min_rows || (uint32_t)s.n * p.G >= p.max_rows) s.n = 0;  // another launch's
    const int cap = (int)min((uint64_t)p.batch.table_pages << p.geom.log2_page, (uint64_t)0x7fff0000);
    s.keys = s.n ? min(max(s.first + s.n, 0), cap) : 0;
    if (p.window) s.lo = (int)min(max((int64_t)s.first + 1 - (int64_t)p.window, (int64_t)0), (int64_t)s.keys);
    return s;
}

// Row f of a KV head's rows (token, query head): its offset in a view, in elements.
template <typename VIEW>
__device__ __forceinline__ int64_t row_offset(const WeighParams& p, const VIEW& v, int q0, uint32_t hk, uint32_t f) {
    const uint32_t i = (__umulhi(f, p.of_group.mul) + f) >> p.of_group.shift, q = f - i * p.G;
    return (int64_t)(q0 + (int)i) * v.ts + (int64_t)(hk * p.G + q) * v.hs;
}
// The new tokens that see a key are [lo, hi).
struct Range {
    int lo, hi;
};
__device__ __forceinline__ Range tokens_of(const WeighParams& p, const WeighSeq& s, int key) {
    const int i = key - s.first;  // keys past the last token's are not asked for but for a tile's width
    // i + window tokens, as far as there are as many: windows reach 2^31 - 1, so it is not formed where it is more
    const int w = (int)p.window;
    return Range{min(max(i, 0), s.n), p.window && i < s.n - w ? max(i + w, 0) : s.n};
}

// Few rows: a wave takes 64 keys of a KV head at a time, 16 rows at a time.  All work is one line
// (per sequence and KV head its tiles of 64 keys), of which each wave has an even share,
// wherever it begins; two tiles' codes are under way while one is computed.  A
// wave does little more than two tiles in a step of 64 requests, so what it does once counts:
// the line is counted in 32 bits (a unit is 64 << tile_shift keys, so that any batch fits).
// 64 requests of up to 8192 keys, 8 KV heads of 128, 8 bit: 20 us (59 MB: 3.0 TB/s); a workgroup
// for each 256 keys of a head, which a quarter of them found empty: 34.
constexpr uint32_t kRowWaves = 2048;  // a power of two: two a SIMD
constexpr float kNoRow = 1e38f;  // lse of a row that is not there: its weights are 0, as those of an infinite one
template <int FMT, int D>
__global__ void __launch_bounds__(256, 2) weigh_rows_kernel(WeighParams p) {
    constexpr int KK = D / 32, RUN = D / 4, W = FMT == QUANT_Q8_0 ? D / 16 : D / 32;
    constexpr uint32_t CB = 4 * W * 4, NB = D / 32;
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t G = p.G, pmask = (1u << p.geom.log2_page) - 1, unit_shift = 6 + p.tile_shift;
    const float c = p.scale * 1.4426950408889634f;  // log2 units

    auto units_of = [&](const WeighSeq& s) {
        return (((uint32_t)s.keys + (1u << unit_shift) - 1) >> unit_shift) - ((uint32_t)s.lo >> unit_shift);
    };
    const uint32_t per = (p.batch.B + 63) / 64;
    const uint32_t b_lo = min(lane * per, p.batch.B), b_hi = min(b_lo + per, p.batch.B);
    uint32_t mine = 0;
#pragma unroll 1
    for (uint32_t x = b_lo; x < b_hi; x++) mine += units_of(weigh_seq(p, x)) * p.geom.Hkv;
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = (uint32_t)__shfl_up((int)incl, o);
        if (lane >= o) incl += x;
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    const uint32_t waves = gridDim.x * 4, log2_waves = 31 - __builtin_clz(waves);
    uint32_t cur = (uint32_t)((uint64_t)total * w >> log2_waves);
    const uint32_t end = (uint32_t)((uint64_t)total * (w + 1) >> log2_waves);
    if (cur == end) return;
    const bool here = incl - mine <= cur && cur < incl;
    uint32_t b = b_lo, off = cur - (incl - mine);
    if (here)
#pragma unroll 1
        for (; b + 1 < b_hi; b++) {
            const uint32_t all = units_of(weigh_seq(p, b)) * p.geom.Hkv;
            if (off < all) break;
            off -= all;
        }
    const int at_lane = __ffsll((unsigned long long)__ballot(here)) - 1;
    b = __builtin_amdgcn_readlane(b, at_lane);
    off = __builtin_amdgcn_readlane(off, at_lane);

#pragma unroll 1
    while (cur < end && b < p.batch.B) {
        const WeighSeq s = weigh_seq(p, b);
        const uint32_t units = units_of(s);
        if (off >= units * p.geom.Hkv) {
            b++;
            off = 0;
            continue;
        }
        const uint32_t rows = (uint32_t)s.n * G;
        // this share's units of one KV head
        const uint32_t hk = off / units, u = off - hk * units, nu = min(units - u, end - cur);
        cur += nu;
        off += nu;
        const int first_key = (int)((((uint32_t)s.lo >> unit_shift) + u) << unit_shift);
        const uint32_t last_key = (uint32_t)first_key + (nu << unit_shift);  // up to 2^31
        const int key_end = last_key < (uint32_t)s.keys ? (int)last_key : s.keys;

        h8_t qf[KK];
        float l[4];
        auto load_rows = [&](uint32_t r0) {
            const _Float16* src = p.Q.p + row_offset(p, p.Q, s.q0, hk, min(r0 + j, rows - 1)) + g * RUN;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) qf[kk] = *reinterpret_cast<const h8_t*>(src + 8 * kk);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t f = r0 + 4 * g + e;
                l[e] = kNoRow;
                if (f < rows) l[e] = p.lse.p[row_offset(p, p.lse, s.q0, hk, f)];
            }
        };
        // page numbers of the next 16 tiles, a lane each 16 keys
        uint32_t ids = 0;
        int ids_from = first_key - 1024;
        uint32_t kw[2][4][W], kd[2][4], page[2][4];
        const uint32_t at_code = j * CB + g * (W * 4), at_scale = p.geom.ks_off + (j * NB + g * NB / 4) * 2;
        auto fetch = [&](int buf, int key0) {
            if (key0 - ids_from >= 1024) {
                ids_from = key0;
                const int k = key0 + 16 * lane;  // past the last key at most by these
                ids = k < s.keys ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)k >> p.geom.log2_page)] : 0xffffffffu;
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                page[buf][t] = __builtin_amdgcn_readlane(ids, (key0 - ids_from) / 16 + t);
                const uint32_t slot = (uint32_t)(key0 + 16 * t) & pmask;
                const uint8_t* base = p.geom.pages + ((size_t)(page[buf][t] < p.geom.num_pages ? page[buf][t] : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                load_words<W, false>(base + slot * CB + at_code, kw[buf][t]);
                kd[buf][t] = *reinterpret_cast<const uint16_t*>(base + slot * (NB * 2) + at_scale);
            }
        };
        // a tile from buffer `buf`, which is filled again with the next but one
        auto tile = [&](int buf, int key0) {
            // a lane's key when the sums are written, and what it has so far
            const uint32_t at = g == 0 ? page[buf][0] : (g == 1 ? page[buf][1] : (g == 2 ? page[buf][2] : page[buf][3]));
            const int key = key0 + 16 * g + j;
            float* to = nullptr;
            float old = 0.0f;
            if (key < s.keys && at < p.geom.num_pages)
                to = p.sums + (((size_t)at * p.geom.Hkv + hk) << p.geom.log2_page) + ((uint32_t)key & pmask);
            h8_t kf[4][KK];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int kk = 0; kk < KK; kk++) kf[t][kk] = k_octet<FMT>(kw[buf][t], kk, as_h2(kd[buf][t] | kd[buf][t] << 16));
            if (to && key < s.first) old = *to;
            if (key0 + 2 * (int)kWaveKeys < key_end) fetch(buf, key0 + 2 * kWaveKeys);
            float sum[4] = {};
            const bool whole = key0 + (int)kWaveKeys - 1 <= s.first && !p.window;  // every row sees every key
#pragma unroll 1
            for (uint32_t r0 = 0; r0 < rows; r0 += 16) {
                if (rows > 16 && (r0 || key0 > first_key)) load_rows(r0);
                f4_t sc[4];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    sc[t] = f4_t{};
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[kk], kf[t][kk], sc[t], 0, 0, 0);
                }
                float less[4];  // a row that sees nothing gives nothing (asked here: the products do not wait for lse)
#pragma unroll
                for (int e = 0; e < 4; e++) less[e] = l[e] == -INFINITY ? -INFINITY : l[e] * -1.4426950408889634f;
                // its products may be NaN or infinite, and so may those of what is no row, which is the last one again
                const bool without = __any(fminf(fminf(less[0], less[1]), fminf(less[2], less[3])) == -INFINITY);
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[t][e] = __builtin_fmaf(sc[t][e], c, less[e]);
                if (without)
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (less[e] <= -kNoRow) sc[t][e] = -INFINITY;
                if (!whole)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const Range see = tokens_of(p, s, key0 + 16 * t + j);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (r0 + 4 * g + e < see.lo * G || r0 + 4 * g + e >= see.hi * G) sc[t][e] = -INFINITY;
                    }
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[t] += __builtin_amdgcn_exp2f(sc[t][e]);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                sum[t] += __shfl_xor(sum[t], 16);
                sum[t] += __shfl_xor(sum[t], 32);
            }
            if (to) *to = old + (g == 0 ? sum[0] : (g == 1 ? sum[1] : (g == 2 ? sum[2] : sum[3])));
        };
        fetch(0, first_key);
        if (first_key + (int)kWaveKeys < key_end) fetch(1, first_key + kWaveKeys);
        load_rows(0);
#pragma unroll 1
        for (int key0 = first_key; key0 < key_end; key0 += 2 * kWaveKeys) {
            tile(0, key0);
            if (key0 + (int)kWaveKeys < key_end) tile(1, key0 + kWaveKeys);
        }
    }
}

// Many rows: a workgroup's waves hold the same 32 NT keys and share the rows, 32 at a time, which
// each brings into LDS of its own by loads of whole rows (operands straight from the rows
// touch 64 lines a load; a row's address by division and 64-bit products cost as much as a
// tile's weights, so all offsets are formed once); their sums meet in LDS.  A tile's products run
// beside the exponentials of the one before.  8 heads, 2048 rows of 32 query heads on 30000 keys of
// 128: 540 us, 0.90 PFLOP/s.  By itself that loop takes 350 cycles a tile of 32 x 32 (256 of products,
// 256 of fused multiplies, exponentials and sums, at 1.65 GHz under this load), 390 us; bringing
// the rows (3.8 GB through the L2s) costs 100 more.  Eight waves of D = 64 are held to the 128
// registers with which two workgroups fit a CU.
template <int FMT, int D, int NT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, D == 64 && NT == 2 ? 4 : 2) weigh_chunk_kernel(WeighParams p) {
    constexpr int KK = D / 16, W = FMT == QUANT_Q8_0 ? 2 : 1;  // words of an octet of codes
    constexpr uint32_t CB = 2 * KK * W * 4, NB = D / 32;
    constexpr int KT = 32 * NT;
    constexpr uint32_t U = D / 8, BLOCK = 32 * D * 2, LOADS = BLOCK / 1024;  // 16-byte units of a row; bytes of 32 rows
    extern __shared__ __attribute__((aligned(16))) uint8_t qs[];             // a wave's 32 rows
    __shared__ __attribute__((aligned(16))) float l2[WAVES][32];
    __shared__ float lse[WAVES][64];  // as it is, twice
    __shared__ __attribute__((aligned(16))) int at_of[WAVES][32];  // tokens from the first of the 32 rows on, far for one that gives nothing
    __shared__ int rel_of[32];
    // what each lane loads of 32 rows, and where a row's lse is, from their first row on (bytes)
    __shared__ int64_t q_off[LOADS * 64], l_off[32];
    __shared__ float part[WAVES][KT];
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hk = blockIdx.x % p.geom.Hkv, G = p.G;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;
    const float c = p.scale * 1.4426950408889634f;  // log2 units
    // 32 rows: some tokens' heads of the group, or of one token 32 at a time, so that what
    // follows is a whole number of tokens on
    const int heads = (int)min(G, 32u), tokens = 32 / heads, subs = (int)(G + 31) / 32;
    const int rel = min(j / heads, tokens), head = j - rel * heads;
    // unit u of row r sits at u ^ swz(r): no two of 16 rows in the same banks
    auto swz = [](uint32_t r) -> uint32_t { return U == 16 ? (r & 15u) : (r >> 1 & 7u); };
    uint8_t* block = qs + wave * BLOCK;
    const uint32_t q_at = j * (U * 16) + 16 * (g ^ swz(j));
    // rows behind the last token's, where 32 are no whole tokens, are its own again and weigh nothing
    for (uint32_t x = tid; x < LOADS * 64; x += 64 * WAVES) {
        const uint32_t r = x / U;
        const int t = min((int)r / heads, tokens);
        q_off[x] = ((int64_t)min(t, tokens - 1) * p.Q.ts + (int64_t)((int)r - t * heads) * p.Q.hs) * 2 + 16 * (x % U ^ swz(r));
    }
    if (tid < 32) {
        rel_of[tid] = rel < tokens ? rel : 0x40000000;
        l_off[tid] = ((int64_t)min(rel, tokens - 1) * p.lse.ts + (int64_t)head * p.lse.hs) * 4;
    }
    __syncthreads();
    for (uint32_t b = blockIdx.x / p.geom.Hkv; b < p.batch.B; b += gridDim.x / p.geom.Hkv) {
        const WeighSeq s = weigh_seq(p, b);
        const int64_t k_lo = s.lo / KT * (int64_t)KT + (int64_t)blockIdx.y * KT;
        if (k_lo >= s.keys) continue;
        for (int64_t k0 = k_lo; k0 < s.keys; k0 += (int64_t)gridDim.y * KT) {
            const int key0 = (int)k0;
            // tokens that see some of these keys, and those that see them all
            const Range first_key = tokens_of(p, s, key0), last_key = tokens_of(p, s, key0 + KT - 1);
            const int i_lo = first_key.lo + (int)wave * tokens, i_hi = last_key.hi;
            auto from_head = [&](int sub) { return min(32 * sub, (int)G - heads); };  // the last ones: some again
            // rows straight into LDS, each load a run of whole ones
            auto bring = [&](int i, int sub) {
                const int64_t row = s.q0 + i, h = hk * G + from_head(sub);
                const uint64_t q = reinterpret_cast<uint64_t>(p.Q.p + row * p.Q.ts + h * p.Q.hs);
                const uint64_t l = reinterpret_cast<uint64_t>(p.lse.p + row * p.lse.ts + h * p.lse.hs);
                const int there = s.n - i;
                const bool all = there >= tokens;  // else again the last token's where there is none
                const int64_t l_at = all ? l_off[j] : ((int64_t)min(rel, there - 1) * p.lse.ts + (int64_t)head * p.lse.hs) * 4;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(l + l_at),
                                                 (__attribute__((address_space(3))) void*)lse[wave], 4, 0, 0);
                int of = lane;
                asm volatile("" : "+v"(of));
                auto load = [&](uint32_t n, int64_t at) {
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(q + at),
                                                     (__attribute__((address_space(3))) void*)(block + n * 1024), 16, 0, 0);
                };
                if (all) {
#pragma unroll
                    for (uint32_t n = 0; n < LOADS; n++) load(n, q_off[n * 64 + of]);
                } else {
#pragma unroll 1
                    for (uint32_t n = 0; n < LOADS; n++) {
                        const uint32_t r = (n * 64 + of) / U;
                        const int t = min(rel_of[r], tokens);
                        load(n, ((int64_t)min(t, there - 1) * p.Q.ts + (int64_t)((int)r - t * heads) * p.Q.hs) * 2 + 16 * (of % U ^ swz(r)));
                    }
                }
            };
            if (i_lo < i_hi) bring(i_lo, 0);
            uint32_t page_id = 0xffffffffu;
            if (lane < 2 * NT && key0 + 16 * lane < s.keys)
                page_id = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)(key0 + 16 * lane) >> p.geom.log2_page)];
            h8_t kf[NT][KK];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t at = (uint32_t)__shfl((int)page_id, 2 * t + (j >> 4));
                const uint32_t slot = (uint32_t)(key0 + 32 * t + j) & pmask;
                const uint8_t* head_of = p.geom.pages + ((size_t)(at < p.geom.num_pages ? at : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    uint32_t kw[W];
                    load_words<W, false>(head_of + slot * CB + (2 * kk + g) * (W * 4), kw);
                    const uint32_t kd = *reinterpret_cast<const uint16_t*>(head_of + p.geom.ks_off + (slot * NB + kk / 2) * 2);
                    kf[t][kk] = k_octet<FMT>(kw, 0, as_h2(kd | kd << 16));
                }
            }
            float sum[NT] = {};
            int i = i_lo, sub = 0;
#pragma unroll 1
            while (i < i_hi && sub < subs) {
                int i_next = i + tokens * WAVES, sub_next = sub;
                if (i_next >= i_hi) {
                    i_next = i_lo;
                    sub_next++;
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // these rows have landed
                // a row that sees nothing gives nothing, nor one that is not there or not of this turn
                const bool live = rel < min(tokens, s.n - i) && from_head(sub) + head >= 32 * sub;
                const float mine = lse[wave][lane];
                const bool without = fabsf(mine) == INFINITY;
                if (g == 0) {
                    l2[wave][j] = without || !live ? INFINITY : mine * 1.4426950408889634f;
                    at_of[wave][j] = without || !live ? 0x40000000 : rel;
                }
                h8_t qf[KK];
#pragma unroll
                for (int kk = 0; kk < KK; kk++) qf[kk] = *reinterpret_cast<const h8_t*>(block + (q_at ^ 32u * kk));
                float l[16];
#pragma unroll
                for (int y = 0; y < 4; y++) *reinterpret_cast<f4_t*>(l + 4 * y) = *reinterpret_cast<const f4_t*>(&l2[wave][8 * y + 4 * g]);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and are read: the next ones may take their place
                if (sub_next < subs) bring(i_next, sub_next);
                if (i >= last_key.lo && min(i + tokens, s.n) <= first_key.hi && !__any(without)) {
                    // all see all: a tile's scores while those before them are weighed (a row of an infinite lse
                    // may hold anything, so it is left out by choice: infinity less infinity would be NaN)
                    f16v_t sc[2];
#pragma unroll
                    for (int t = 0; t <= NT; t++) {
                        if (t < NT) sc[t & 1] = f16v_t{};
                        float of_rows = 0.0f;  // apart from what there is: many small terms
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) {
                            if (t < NT) sc[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf[kk], kf[t][kk], sc[t & 1], 0, 0, 0);
                            if (t > 0)
#pragma unroll
                                for (int e = kk * 16 / KK; e < (kk + 1) * 16 / KK; e++)
                                    of_rows += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[(t - 1) & 1][e], c, -l[e]));
                            if (t > 0) __builtin_amdgcn_sched_barrier(0);
                        }
                        if (t > 0) sum[t - 1] += of_rows;
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        f16v_t sc{};
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf[kk], kf[t][kk], sc, 0, 0, 0);
                        int key = key0 + 32 * t + j;
                        asm volatile("" : "+v"(key));  // formed anew: kept, these ranges would spill
                        const Range see = tokens_of(p, s, key);
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int at = i + at_of[wave][8 * (e >> 2) + 4 * g + (e & 3)];
                            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -l[e]));
                            sum[t] += at >= see.lo && at < see.hi ? w : 0.0f;
                        }
                    }
                }
                i = i_next;
                sub = sub_next;
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                sum[t] += __shfl_xor(sum[t], 32);
                if (g == 0) part[wave][32 * t + j] = sum[t];
            }
            __syncthreads();
            for (int x = tid; x < KT; x += 64 * WAVES) {
                const int key = key0 + x;
                float mine = 0.0f;
#pragma unroll
                for (int v = 0; v < WAVES; v++) mine += part[v][x];
                const uint32_t at = key < s.keys ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)key >> p.geom.log2_page)] : 0xffffffffu;
                if (at < p.geom.num_pages) {
                    float* to = p.sums + (((size_t)at * p.geom.Hkv + hk) << p.geom.log2_page) + ((uint32_t)key & pmask);
                    *to = key >= s.first ? mine : *to + mine;
                }
            }
            __syncthreads();
        }
    }
}

// Rows of a KV head from which a sequence is the chunk kernel's.
constexpr uint32_t kWeighChunk = 128;
// 128 keys to four waves where there are as many workgroups as the chip holds, else 64 to eight.
// us of the two: 8 prompts of 2048 (D = 128, 1024 workgroups of the first kind) 188 / 240, four of
// them 118 / 125, two 103 / 69; 512 rows on 8192 keys (512) 57 / 73; D = 64: 8 prompts 139 / 127, two 80 / 45.
constexpr uint64_t kWeighGroups = 512;

template <int FMT, int D>
static hipError_t launch_weigh(WeighParams p, hipStream_t st) {
    const uint64_t rows = (uint64_t)(p.max_new ? p.max_new : 1) * p.G;
    uint64_t keys = p.max_kv ? p.max_kv : 1;
    if (p.window && keys > (uint64_t)p.window + p.max_new) keys = (uint64_t)p.window + p.max_new;
    // Sequences of few rows among others are the rows kernel's, if there can be any: with as many rows as all
    // but one could have, the last has the rest (three prompts of 809 .. 1739 tokens 41 us, with a launch of the
    // other in vain 45).
    const uint64_t others = (uint64_t)(p.batch.B - 1) * p.max_new, least = (kWeighChunk + p.G - 1) / p.G;
    const bool chunks = rows >= kWeighChunk, both = chunks && p.batch.B > 1 && p.batch.T < others + least;
    p.min_rows = 0;
    p.max_rows = both ? kWeighChunk : 0xffffffffu;
    const uint64_t cap = (uint64_t)p.batch.table_pages << p.geom.log2_page;
    if (!chunks || both) {
        const uint64_t heads = (uint64_t)p.batch.B * p.geom.Hkv;
        p.tile_shift = 0;
        while (heads * ((cap >> (6 + p.tile_shift)) + 1) >= 1ull << 31 && p.tile_shift < 24) p.tile_shift++;
        const uint64_t tiles = (keys + kWaveKeys - 1) / kWaveKeys;
        uint32_t groups = 1;  // a power of two
        while (4ull * groups < kRowWaves && 4ull * groups < heads * tiles) groups *= 2;
        hipLaunchKernelGGL((weigh_rows_kernel<FMT, D>), dim3(groups), dim3(256), 0, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !chunks) return e;
    }
    p.min_rows = both ? kWeighChunk : 0;
    p.max_rows = 0xffffffffu;
    const uint64_t heads = (uint64_t)p.batch.B * p.geom.Hkv, most = std::max(1u << 20, p.geom.Hkv) / p.geom.Hkv * p.geom.Hkv;
    auto launch = [&](auto kernel, uint32_t tile, uint32_t waves, size_t (&attr)[kMaxDevices]) {
        const size_t lds = (size_t)waves * 32 * D * 2;
        const hipError_t e = lds_limit_once((const void*)kernel, lds, attr);
        if (e != hipSuccess) return e;
        // the tiles that most rows see first, of all sequences; no more than the table holds, whatever is
        // expected (a prompt of 2048 in a table for as many, 2^31 expected: 1310 us, so 96)
        const dim3 grid((uint32_t)std::min(heads, most), (uint32_t)std::min((std::min(keys, cap) + tile - 1) / tile, (uint64_t)65535));
        hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), lds, st, p);
        return hipGetLastError();
    };
    if ((keys + 127) / 128 * heads >= kWeighGroups) {
        static size_t attr[kMaxDevices] = {};
        return launch(weigh_chunk_kernel<FMT, D, 4, 4>, 128, 4, attr);
    }
    static size_t attr[kMaxDevices] = {};
    return launch(weigh_chunk_kernel<FMT, D, 2, 8>, 64, 8, attr);
}

hipError_t launch_kv_weigh(const WeighParams& p, hipStream_t st) {
    if (p.batch.B == 0 || p.batch.T == 0) return hipSuccess;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_weigh<QUANT_Q8_0, 64>(p, st) : launch_weigh<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_weigh<QUANT_Q4_0, 64>(p, st) : launch_weigh<QUANT_Q4_0, 128>(p, st);
}

// ---- eviction ------------------------------------------------------------------
//
// Of a sequence's places, per KV head: the first `sinks`, the last `recent` and the heaviest of
// the others, `budget` together, in their order, the lowest first among equals.  One
// kernel finds them, another copies them to pages of their own, so that no copy waits for
// another and pages that sequences share stay as they are.

// Weights as integers of the same order, from 0x007fffff (-infinity) on; 0xffffffff for a place
// that is kept in any case, next to it NaN; 0 for one that is not there.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = f32_bits(w + 0.0f);  // -0 is 0
    const uint32_t k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
    return w != w ? 0xfffffffeu : k;
}

// The budget-th largest key is found by its leading bits: how many keys have each value of 11
// bits is counted in LDS (kCopies counters each, against lanes that meet), which names the value
// that it has.  The keys that share it are few as a rule: up to kList of them are gathered and
// ranked against each other, more are counted again by the next bits.  Then the places that stay
// are written in order.  All loops are kept as loops: unrolled, with the keys in registers,
// most of the 17 KB of code ran once and was waited for (27 us for 64 caches of 8 heads and up to
// 8192 keys).
//
// A workgroup does this for a sequence and KV head, with the keys in LDS (as many as expected,
// up to kHeld; more are formed again for each sweep).  Where these are few and long, it is done
// in three launches by a workgroup every kSegment places: each counts its own and leaves the
// counts (evict_pick_kernel), adds up all and gathers its keys of that value (evict_gather_kernel),
// and ranks what all have gathered and writes its places (evict_place_kernel).  One request of
// 131072 keys: 123 us by one workgroup a head, 5 + 11 + 10 in three launches; 64 requests: 15.
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr uint32_t kCopies = 4, kBins = 2048, kList = 1024, kHeld = 24576;
constexpr uint32_t kSegment = 8192, kGathered = 16384;

// Of a sequence and KV head that is split: the leading bits sought, how many are wanted at or
// below them, how many have them, how many stay.
struct alignas(16) PickNote {
    uint32_t digit, want, share, m;
};
// workspace: a note an item, counts [item][segment][kBins] and how many of a segment lie above
// the bits sought, gathered keys [item][kGathered]
struct PickSpace {
    PickNote* notes;
    uint16_t* counts;
    uint32_t* above;
    uint32_t* keys;
    __host__ __device__ PickSpace(uint8_t* ws, uint64_t items, uint32_t segments) {
        notes = reinterpret_cast<PickNote*>(ws);
        keys = reinterpret_cast<uint32_t*>(notes + items);
        above = keys + items * kGathered;
        counts = reinterpret_cast<uint16_t*>(above + (items * segments + 3) / 4 * 4);
    }
    static size_t bytes(uint64_t items, uint32_t segments) {
        return items * (sizeof(PickNote) + kGathered * 4) + (items * segments + 3) / 4 * 16 + items * segments * kBins * 2;
    }
};

struct PickSeq {
    uint32_t b, hk, n, last, quads;  // places that the table holds; the first of the last `recent`; n in fours
    const int32_t* table;
    __device__ __forceinline__ PickSeq(const EvictParams& p, uint64_t item) {
        b = (uint32_t)(item / p.geom.Hkv);
        hk = (uint32_t)(item % p.geom.Hkv);
        const int len = max(p.batch.kv_len[b], 0);
        n = (uint32_t)min((uint64_t)len, (uint64_t)p.batch.table_pages << p.geom.log2_page);
        last = (uint32_t)max((int64_t)len - (int64_t)p.recent, (int64_t)0);
        quads = (n + 3) / 4;
        table = p.batch.table + (size_t)b * p.batch.table_stride;
    }
    // keys of places 4 q .. 4 q + 3
    __device__ __forceinline__ u4_t keys(const EvictParams& p, uint32_t q) const {
        const uint32_t page = (uint32_t)table[4 * q >> p.geom.log2_page];
        if (page >= p.geom.num_pages) return u4_t{};
        const f4_t w = *reinterpret_cast<const f4_t*>(p.sums + (((size_t)page * p.geom.Hkv + hk) << p.geom.log2_page) +
                                                      (4 * q & ((1u << p.geom.log2_page) - 1)));
        u4_t k;
#pragma unroll
        for (int e = 0; e < 4; e++) k[e] = order_of(w[e]);
        if (4 * q < p.sinks || 4 * q + 4 > min(last, n))
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (4 * q + e < p.sinks || 4 * q + e >= last) k[e] = 0xffffffffu;
                if (4 * q + e >= n) k[e] = 0;
            }
        return k;
    }
    // whether it is split over the workgroups of `segments` segments
    __device__ __forceinline__ bool split(uint32_t segments) const { return n > 2 * kSegment && n <= segments * kSegment; }
};

struct PickShared {
    uint32_t bins[kBins * kCopies];
    uint32_t list[kList];
    uint32_t wave_sum[2][kPickWaves], found[3], listed;
};

__device__ __forceinline__ void clear_bins(PickShared& sh) {
#pragma unroll 1
    for (uint32_t x = threadIdx.x; x < kBins * kCopies / 4; x += kPickThreads) reinterpret_cast<u4_t*>(sh.bins)[x] = u4_t{};
    __syncthreads();
}
// How many keys have the values 2 tid and 2 tid + 1.
__device__ __forceinline__ u2_t bins_of(const PickShared& sh) {
    const u4_t* v = reinterpret_cast<const u4_t*>(sh.bins) + 2 * threadIdx.x;
    return u2_t{v[0].x + v[0].y + v[0].z + v[0].w, v[1].x + v[1].y + v[1].z + v[1].w};
}
// Of values counted a lane two each: found[0] the one that holds the want-th largest key, found[1] how many
// of its keys are wanted, found[2] how many it has.  Returns how many keys were counted; with
// `first` the first value does not count, and nothing is found where the others are at most `want`.
__device__ __forceinline__ uint32_t find_value(PickShared& sh, u2_t c, uint32_t want, bool first) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (first && tid == 0) c.x = 0;
    uint32_t above = c.x + c.y;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const uint32_t y = (uint32_t)__shfl_down((int)above, x);
        if (lane + x < 64) above += y;
    }
    if (lane == 0) sh.wave_sum[0][wave] = above;
    __syncthreads();
    uint32_t all = lane < (uint32_t)kPickWaves ? sh.wave_sum[0][lane] : 0, behind = lane > wave ? all : 0;
#pragma unroll
    for (int x = 1; x < kPickWaves; x <<= 1) {
        all += (uint32_t)__shfl_xor((int)all, x);
        behind += (uint32_t)__shfl_xor((int)behind, x);
    }
    all = (uint32_t)__builtin_amdgcn_readfirstlane((int)all);
    above += (uint32_t)__builtin_amdgcn_readfirstlane((int)behind) - c.x - c.y;
    if (first && all <= want) return all;
    if (above < want && want <= above + c.x + c.y) {
        const bool second = want <= above + c.y;
        sh.found[0] = 2 * tid + second;
        sh.found[1] = want - above - (second ? 0 : c.y);
        sh.found[2] = second ? c.y : c.x;
    }
    __syncthreads();
    return all;
}
// The want-th largest of `share` keys in the list (1 .. kList): found[0], and found[1] how many of those alike are wanted.
__device__ __forceinline__ void rank_list(PickShared& sh, uint32_t share, uint32_t want) {
    const uint32_t tid = threadIdx.x;
    if (tid < (0u - share & 7)) sh.list[share + tid] = 0;
    __syncthreads();
    if (tid / 64 * 64 < share) {
        const uint32_t k = tid < share ? sh.list[tid] : 0;
        uint32_t larger = 0, same = 0;
#pragma unroll 1
        for (uint32_t x = 0; x < share; x += 8) {
            const u4_t u = *reinterpret_cast<const u4_t*>(&sh.list[x]), v = *reinterpret_cast<const u4_t*>(&sh.list[x + 4]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                larger += (u[e] > k ? 1 : 0) + (v[e] > k ? 1 : 0);
                same += (u[e] == k ? 1 : 0) + (v[e] == k ? 1 : 0);
            }
        }
        if (tid < share && larger < want && want <= larger + same) {  // alike in all that are the one sought
            sh.found[0] = k;
            sh.found[1] = want - larger;
        }
    }
    __syncthreads();
}
// Places of fours q0 .. q1 whose keys lie above `least`, and the first `equal` at it (none
// where least is 0), written in order; before them are above0 and equal0.  Sums that another
// stream changes meanwhile give other places, but no more than `room`.
template <typename KEYS>
__device__ __forceinline__ void write_places(PickShared& sh, KEYS keys, uint32_t q0, uint32_t q1, uint32_t least, uint32_t equal,
                                             uint32_t above0, uint32_t equal0, int32_t* out, uint32_t room) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t turn = 0;
#pragma unroll 1
    for (; q0 < q1; q0 += kPickThreads, turn ^= 1) {
        const uint32_t q = q0 + tid;
        const u4_t k = q < q1 ? keys(q) : u4_t{};
        // how many lie above it and, in the high half, at it
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) mine += k[e] > least ? 1u : (k[e] == least && least ? 0x10000u : 0u);
        uint32_t before = mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const uint32_t y = (uint32_t)__shfl_up((int)before, x);
            if (lane >= (uint32_t)x) before += y;
        }
        if (lane == 63) sh.wave_sum[turn][wave] = before;
        __syncthreads();  // the other half may still be read by waves that are behind
        uint32_t sum = lane < (uint32_t)kPickWaves ? sh.wave_sum[turn][lane] : 0, others = lane < wave ? sum : 0;
#pragma unroll
        for (int x = 1; x < kPickWaves; x <<= 1) {
            sum += (uint32_t)__shfl_xor((int)sum, x);
            others += (uint32_t)__shfl_xor((int)others, x);
        }
        sum = (uint32_t)__builtin_amdgcn_readfirstlane((int)sum);
        before += (uint32_t)__builtin_amdgcn_readfirstlane((int)others) - mine;
        uint32_t ne = equal0 + (before >> 16), to = above0 + (before & 0xffffu) + min(ne, equal);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool same = k[e] == least && least, stays = k[e] > least || (same && ne < equal);
            if (stays && to < room) out[to] = (int32_t)(4 * q + e);
            to += stays;
            ne += same;
        }
        above0 += sum & 0xffffu;
        equal0 += sum >> 16;
    }
}
__device__ __forceinline__ void end_places(const EvictParams& p, const PickSeq& s, uint32_t m, int32_t* out) {
#pragma unroll 1
    for (uint32_t x = m + threadIdx.x; x < p.budget; x += kPickThreads) out[x] = -1;
    if (s.hk == 0 && threadIdx.x == 0) p.len_out[s.b] = (int32_t)m;
}

// From the bits of the key sought above `low`, `prefix`, which `share` of the keys have, to all of
// them; want: how many of the largest of these are wanted, then of those alike.
template <typename KEYS>
__device__ __forceinline__ void settle(PickShared& sh, KEYS keys, uint32_t quads, uint32_t low, uint32_t share, uint32_t& prefix,
                                       uint32_t& want) {
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) sh.listed = 0;
    while (low && share > kList) {
        const uint32_t top = low;
        low = low == 21 ? 10 : 0;
        clear_bins(sh);
#pragma unroll 1
        for (uint32_t q = tid; q < quads; q += kPickThreads) {
            const u4_t k = keys(q);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (k[e] >> top == prefix) atomicAdd(&sh.bins[(k[e] >> low & ((1u << (top - low)) - 1)) * kCopies + lane % kCopies], 1u);
        }
        __syncthreads();
        find_value(sh, bins_of(sh), want, false);
        prefix = prefix << (top - low) | sh.found[0];
        want = sh.found[1];
        share = sh.found[2];
    }
    __syncthreads();  // found is read, listed is clear
    if (!low) return;
    uint32_t own = 0;
    asm volatile("" : "+v"(own));  // a lane's own address: lanes that meet are few
#pragma unroll 1
    for (uint32_t q = tid; q < quads; q += kPickThreads) {
        const u4_t k = keys(q);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (k[e] >> low == prefix) {
                const uint32_t at = atomicAdd(&sh.listed + own, 1u);
                if (at < kList) sh.list[at] = k[e];
            }
    }
    __syncthreads();
    rank_list(sh, share, want);
    prefix = sh.found[0];
    want = sh.found[1];
}

// All of it by one workgroup; the keys of up to held_keys places are held.
__device__ __forceinline__ void pick_alone(const EvictParams& p, const PickSeq& s, PickShared& sh, u4_t* held, uint32_t held_keys) {
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const bool hold = s.n <= held_keys;
    auto keys_of = [&](uint32_t q) { return hold ? held[q] : s.keys(p, q); };
    clear_bins(sh);
#pragma unroll 2
    for (uint32_t q = tid; q < s.quads; q += kPickThreads) {
        const u4_t k = s.keys(p, q);
        if (hold) held[q] = k;
#pragma unroll
        for (int e = 0; e < 4; e++) atomicAdd(&sh.bins[(k[e] >> 21) * kCopies + lane % kCopies], 1u);
    }
    __syncthreads();
    // places that are not there have the lowest value to themselves
    const uint32_t there = find_value(sh, bins_of(sh), p.budget, true);
    uint32_t least = 0, equal = 0;
    if (there > p.budget) {
        least = sh.found[0];
        equal = sh.found[1];
        settle(sh, keys_of, s.quads, 21, sh.found[2], least, equal);
    }
    int32_t* out = p.kept + ((size_t)s.b * p.geom.Hkv + s.hk) * p.budget;
    __syncthreads();
    write_places(sh, keys_of, 0, s.quads, least, equal, 0, 0, out, p.budget);
    end_places(p, s, min(there, p.budget), out);
    __syncthreads();
}

// segments > 1: a workgroup a segment of each item, else one an item.
__global__ void __launch_bounds__(kPickThreads, 8) evict_pick_kernel(EvictParams p, uint32_t held_keys, uint32_t segments) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ __attribute__((aligned(16))) PickShared sh;
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    for (uint64_t x = blockIdx.x; x < items * segments; x += gridDim.x) {
        const uint64_t item = x / segments;
        const uint32_t seg = (uint32_t)(x % segments);
        const PickSeq s(p, item);
        if (!s.split(segments)) {
            if (seg == 0) pick_alone(p, s, sh, reinterpret_cast<u4_t*>(smem), held_keys);
            continue;
        }
        clear_bins(sh);
        const uint32_t q1 = min((seg + 1) * (kSegment / 4), s.quads);
#pragma unroll 2
        for (uint32_t q = seg * (kSegment / 4) + threadIdx.x; q < q1; q += kPickThreads) {
            const u4_t k = s.keys(p, q);
#pragma unroll
            for (int e = 0; e < 4; e++) atomicAdd(&sh.bins[(k[e] >> 21) * kCopies + threadIdx.x % kCopies], 1u);
        }
        __syncthreads();
        const u2_t c = bins_of(sh);
        const PickSpace ws(p.ws, items, segments);
        *reinterpret_cast<uint32_t*>(ws.counts + (item * segments + seg) * kBins + 2 * threadIdx.x) = c.x | c.y << 16;
        __syncthreads();
    }
}

// Short sequences: a wave each, four a workgroup, up to 256 FOURS keys in registers.  The budget-th largest
// key is the largest value that as many keys reach, found bit by bit until just as many do; a count is
// four ballots every 256 keys.  us of workgroups (2048 counters to clear and to add up) / waves: one
// request of 260 keys and 4 heads 6.8 / 5.4, 3840 items of up to 89 keys 53 / 6.0; with four fours 2400
// of up to 900 39 / 14, but 512 of them 11.0 / 12.7 and 8 of them 7.6 / 8.3.
constexpr uint32_t kShortKeys = 512, kShortItems = 1024;
// HELD: all keys are in registers; else (sequences longer than expected) they are formed again, and the
// value is found eight bits at a time by counts in LDS.
template <uint32_t FOURS, bool HELD>
__device__ __forceinline__ void pick_short(const EvictParams& p, const PickSeq& s, uint32_t lane, uint32_t (&bins)[256]) {
    u4_t held[FOURS];
    if constexpr (HELD)
#pragma unroll
        for (uint32_t x = 0; x < FOURS; x++) held[x] = 64 * x + lane < s.quads ? s.keys(p, 64 * x + lane) : u4_t{};
    auto each = [&](auto f) {
        if constexpr (HELD) {
#pragma unroll
            for (uint32_t x = 0; x < FOURS; x++) f(64 * x, held[x]);
        } else {
#pragma unroll 1
            for (uint32_t q = 0; q < s.quads; q += 64) f(q, q + lane < s.quads ? s.keys(p, q + lane) : u4_t{});
        }
    };
    auto reach = [&](uint32_t least) {
        uint32_t n = 0;
        each([&](uint32_t, u4_t k) {
#pragma unroll
            for (int e = 0; e < 4; e++) n += (uint32_t)__popcll(__ballot(k[e] >= least));
        });
        return n;
    };
    const uint32_t there = reach(1);
    uint32_t least = 0, equal = 0;
    if (!HELD && there > p.budget) {
        equal = p.budget;
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            *reinterpret_cast<u4_t*>(&bins[4 * lane]) = u4_t{};
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            each([&](uint32_t, u4_t k) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (shift == 24 || k[e] >> (shift + 8 & 31) == least) atomicAdd(&bins[k[e] >> shift & 255], 1u);
            });
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            const u4_t c = *reinterpret_cast<const u4_t*>(&bins[4 * lane]);
            const uint32_t mine = c.x + c.y + c.z + c.w;
            uint32_t above = mine;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                const uint32_t y = (uint32_t)__shfl_down((int)above, x);
                if (lane + x < 64) above += y;
            }
            above -= mine;
            // one lane has it among its four
            uint32_t digit = 4 * lane + 3, left = equal - above;
#pragma unroll
            for (int e = 3; e > 0; e--)
                if (digit == 4 * lane + e && left > c[e]) {
                    left -= c[e];
                    digit--;
                }
            const int at = __ffsll((unsigned long long)__ballot(above < equal && equal <= above + mine)) - 1;
            least = least << 8 | (uint32_t)__builtin_amdgcn_readlane((int)digit, max(at, 0));
            equal = (uint32_t)__builtin_amdgcn_readlane((int)left, max(at, 0));
        }
    } else if (there > p.budget) {
        bool exact = false;  // as many reach it as are wanted: no need to know it better
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit && !exact; bit >>= 1) {
            const uint32_t n = reach(least | bit);
            if (n >= p.budget) least |= bit;
            exact = n == p.budget;
        }
        if (exact) least--;
        else equal = p.budget - (least == 0xffffffffu ? 0 : reach(least + 1));
    }
    int32_t* out = p.kept + ((size_t)s.b * p.geom.Hkv + s.hk) * p.budget;
    uint32_t above0 = 0, equal0 = 0;
    each([&](uint32_t q, u4_t k) {
        uint32_t mine = 0;  // as in write_places
#pragma unroll
        for (int e = 0; e < 4; e++) mine += k[e] > least ? 1u : (k[e] == least && least ? 0x10000u : 0u);
        uint32_t before = mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const uint32_t y = (uint32_t)__shfl_up((int)before, x);
            if (lane >= (uint32_t)x) before += y;
        }
        const uint32_t sum = (uint32_t)__builtin_amdgcn_readlane((int)before, 63);
        before -= mine;
        uint32_t ne = equal0 + (before >> 16), to = above0 + (before & 0xffffu) + min(ne, equal);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool same = k[e] == least && least, stays = k[e] > least || (same && ne < equal);
            if (stays && to < p.budget) out[to] = (int32_t)(4 * (q + lane) + e);
            to += stays;
            ne += same;
        }
        above0 += sum & 0xffffu;
        equal0 += sum >> 16;
    });
    const uint32_t m = min(there, p.budget);
    for (uint32_t x = m + lane; x < p.budget; x += 64) out[x] = -1;
    if (s.hk == 0 && lane == 0) p.len_out[s.b] = (int32_t)m;
}

template <uint32_t FOURS>
__global__ void __launch_bounds__(256) evict_pick_short_kernel(EvictParams p) {
    __shared__ __attribute__((aligned(16))) uint32_t bins[4][256];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    for (uint64_t item = (uint64_t)blockIdx.x * 4 + wave; item < items; item += (uint64_t)gridDim.x * 4) {
        const PickSeq s(p, item);
        if (s.n <= 256 * FOURS) pick_short<FOURS, true>(p, s, lane, bins[wave]);
        else pick_short<FOURS, false>(p, s, lane, bins[wave]);
    }
}

// Sum over the workgroup, by one counter in LDS.
__device__ __forceinline__ uint32_t sum_of_all(PickShared& sh, uint32_t v) {
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    uint32_t own = 0;
    asm volatile("" : "+v"(own));
    if (v) atomicAdd(&sh.listed + own, v);
    __syncthreads();
    const uint32_t sum = sh.listed;
    __syncthreads();
    return sum;
}

__global__ void __launch_bounds__(kPickThreads, 8) evict_gather_kernel(EvictParams p, uint32_t segments) {
    __shared__ __attribute__((aligned(16))) PickShared sh;
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    const uint32_t tid = threadIdx.x;
    const PickSpace ws(p.ws, items, segments);
    for (uint64_t x = blockIdx.x; x < items * segments; x += gridDim.x) {
        const uint64_t item = x / segments;
        const uint32_t seg = (uint32_t)(x % segments);
        const PickSeq s(p, item);
        const uint32_t used = (s.n + kSegment - 1) / kSegment;
        if (!s.split(segments) || seg >= used) continue;
        const uint16_t* counts = ws.counts + item * segments * kBins;
        u2_t c{}, mine{};
#pragma unroll 4
        for (uint32_t y = 0; y < used; y++) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(counts + (size_t)y * kBins + 2 * tid);
            const u2_t w = {v & 0xffffu, v >> 16};
            c += w;
            if (y == seg) mine = w;
        }
        const uint32_t there = find_value(sh, c, p.budget, true);
        PickNote note{0, 0, 0, there};
        if (there > p.budget) note = PickNote{sh.found[0], sh.found[1], sh.found[2], p.budget};
        const uint32_t above = sum_of_all(sh, (2 * tid > note.digit ? mine.x : 0) + (2 * tid + 1 > note.digit ? mine.y : 0));
        if (tid == 0) {
            ws.above[item * segments + seg] = above;
            if (seg == 0) ws.notes[item] = note;
        }
        if (note.share == 0 || note.share > kGathered) continue;
        uint32_t before = 0;
        for (uint32_t y = tid; y < seg; y += kPickThreads) before += counts[(size_t)y * kBins + note.digit];
        uint32_t* to = ws.keys + item * kGathered;
        before = sum_of_all(sh, before);
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        uint32_t own = 0;
        asm volatile("" : "+v"(own));
        const uint32_t q1 = min((seg + 1) * (kSegment / 4), s.quads);
#pragma unroll 2
        for (uint32_t q = seg * (kSegment / 4) + tid; q < q1; q += kPickThreads) {
            const u4_t k = s.keys(p, q);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (k[e] >> 21 == note.digit) {
                    const uint32_t at = before + atomicAdd(&sh.listed + own, 1u);
                    if (at < kGathered) to[at] = k[e];
                }
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kPickThreads, 8) evict_place_kernel(EvictParams p, uint32_t segments) {
    __shared__ __attribute__((aligned(16))) PickShared sh;
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    const uint32_t tid = threadIdx.x;
    const PickSpace ws(p.ws, items, segments);
    for (uint64_t x = blockIdx.x; x < items * segments; x += gridDim.x) {
        const uint64_t item = x / segments;
        const uint32_t seg = (uint32_t)(x % segments);
        const PickSeq s(p, item);
        const uint32_t used = (s.n + kSegment - 1) / kSegment;
        if (!s.split(segments) || seg >= used) continue;
        const PickNote note = ws.notes[item];
        if (note.share > kGathered) {  // too many alike to gather
            if (seg == 0) pick_alone(p, s, sh, nullptr, 0);
            continue;
        }
        uint32_t least = note.digit, equal = note.want;
        const uint32_t* gathered = ws.keys + item * kGathered;
        if (note.share) {
            auto keys = [&](uint32_t q) {
                u4_t k = reinterpret_cast<const u4_t*>(gathered)[q];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * q + e >= note.share) k[e] = 0;
                return k;
            };
            settle(sh, keys, (note.share + 3) / 4, 21, note.share, least, equal);
        }
        // what the segments before this one have above it and at it
        uint32_t above = 0, alike = 0, ahead = 0;
        for (uint32_t y = tid; y < seg; y += kPickThreads) {
            above += ws.above[item * segments + y];
            if (note.share) ahead += ws.counts[(item * segments + y) * kBins + note.digit];
        }
        ahead = sum_of_all(sh, ahead);
        for (uint32_t y = tid; y < min(ahead, kGathered); y += kPickThreads) {
            above += gathered[y] > least;
            alike += gathered[y] == least;
        }
        above = sum_of_all(sh, above);
        alike = sum_of_all(sh, alike);
        int32_t* out = p.kept + ((size_t)s.b * p.geom.Hkv + s.hk) * p.budget;
        write_places(sh, [&](uint32_t q) { return s.keys(p, q); }, seg * (kSegment / 4), min((seg + 1) * (kSegment / 4), s.quads), least,
                     equal, above, alike, out, p.budget);
        if (seg == 0) end_places(p, s, note.m, out);
        __syncthreads();
    }
}

// Kept token i becomes token i of the other table's pages: kCopyTokens of them a workgroup, of one
// head.  Codes of V lie in groups of four tokens, so four sources' bytes make a word; where the
// last group is not full, the others of its tokens keep their own.  Bound by memory: 64 requests cut to
// 1024 tokens (8 heads of 128, 8 bit) 57 .. 64 us, 88 MB read and 114 written; of V each kept
// token's whole group is read, a line in any case.
constexpr uint32_t kCopyTokens = 128;
template <int FMT, int D>
__global__ void __launch_bounds__(256) evict_copy_kernel(EvictParams p, uint32_t tiles) {
    constexpr uint32_t CB = FMT == QUANT_Q8_0 ? D : D / 2, NB = D / 32, KP = CB / 16, VP = CB / 4;
    __shared__ uint32_t src_page[kCopyTokens], src_slot[kCopyTokens], dst_page[kCopyTokens];
    __shared__ uint32_t live[kCopyTokens], some;
    const uint32_t tid = threadIdx.x, hk = blockIdx.x % p.geom.Hkv;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;
    auto head_of = [&](uint32_t page) { return p.geom.pages + ((size_t)page * p.geom.Hkv + hk) * p.geom.head_bytes; };
    for (uint32_t b = blockIdx.y; b < p.batch.B; b += gridDim.y) {
        const int32_t* kept = p.kept + ((size_t)b * p.geom.Hkv + hk) * p.budget;
        for (uint32_t t0 = blockIdx.x / p.geom.Hkv * kCopyTokens; t0 < p.budget; t0 += tiles * kCopyTokens) {
            __syncthreads();
            if (tid < kCopyTokens) {
                const uint32_t i = t0 + tid, pi = i >> p.geom.log2_page;
                int from = i < p.budget ? kept[i] : -1;
                // what the other kernel wrote, unless the caller writes there or to the table meanwhile: nothing outside is read then either
                uint32_t sp = 0xffffffffu;
                if (from >= 0 && (uint32_t)from >> p.geom.log2_page < p.batch.table_pages)
                    sp = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)from >> p.geom.log2_page)];
                if (sp >= p.geom.num_pages) from = -1;
                uint32_t dp = pi < p.out_pages ? (uint32_t)p.table_out[(size_t)b * p.out_stride + pi] : 0xffffffffu;
                if (dp >= p.geom.num_pages) dp = 0xffffffffu;
                dst_page[tid] = dp;
                live[tid] = from >= 0 && dp != 0xffffffffu;
                if (tid == 0) some = from >= 0;
                src_page[tid] = from >= 0 ? sp : dp;
                src_slot[tid] = (uint32_t)(from >= 0 ? from : (int)i) & pmask;
            }
            __syncthreads();
            if (!some) break;  // the kept are the first
            // loaded before anything is stored: the compiler cannot tell that the pages are others
            constexpr int NK = kCopyTokens * KP / 256, NV = kCopyTokens / 4 * VP / 256, NS = kCopyTokens * NB / 256;
            u4_t kv[NK], vv[NV][4];
            uint32_t sv[NS], of_k = 0, of_k2 = 0;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const uint32_t x = tid + 256 * i, t = x / KP, u = x % KP;
                if (live[t]) kv[i] = *reinterpret_cast<const u4_t*>(head_of(src_page[t]) + src_slot[t] * CB + 16 * u);
            }
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t x = tid + 256 * i, t = x / VP * 4, u = x % VP;
                if (live[t])
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        vv[i][e] = *reinterpret_cast<const u4_t*>(head_of(src_page[t + e]) + p.geom.v_off + (src_slot[t + e] >> 2) * (4 * CB) + 16 * u);
            }
            // V's scales block by block, K's and the sum a token
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint32_t x = tid + 256 * i, t = x % kCopyTokens, y = x / kCopyTokens, ss = src_slot[t];
                sv[i] = 0;
                if (live[t]) sv[i] = *reinterpret_cast<const uint16_t*>(head_of(src_page[t]) + p.geom.vs_off + (((ss >> 2) * NB + y) * 4 + (ss & 3)) * 2);
            }
            if (tid < kCopyTokens && live[tid]) {
                const uint32_t* ks = reinterpret_cast<const uint32_t*>(head_of(src_page[tid]) + p.geom.ks_off + src_slot[tid] * (2 * NB));
                of_k = ks[0];
                if constexpr (NB == 4) of_k2 = ks[1];
                sum = p.sums[(((size_t)src_page[tid] * p.geom.Hkv + hk) << p.geom.log2_page) + src_slot[tid]];
            }
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const uint32_t x = tid + 256 * i, t = x / KP, u = x % KP;
                if (live[t]) *reinterpret_cast<u4_t*>(head_of(dst_page[t]) + ((t0 + t) & pmask) * CB + 16 * u) = kv[i];
            }
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t x = tid + 256 * i, t = x / VP * 4, u = x % VP;
                if (!live[t]) continue;
                const uint32_t k0 = src_slot[t] & 3, k1 = src_slot[t + 1] & 3, k2 = src_slot[t + 2] & 3, k3 = src_slot[t + 3] & 3;
                const uint32_t lo = k0 | (4 + k1) << 8 | 0x0c0c0000u, hi = 0x0c0cu | k2 << 16 | (4 + k3) << 24;
                u4_t y;
#pragma unroll
                for (int d = 0; d < 4; d++) y[d] = perm(vv[i][1][d], vv[i][0][d], lo) | perm(vv[i][3][d], vv[i][2][d], hi);
                *reinterpret_cast<u4_t*>(head_of(dst_page[t]) + p.geom.v_off + ((t0 + t) & pmask) / 4 * (4 * CB) + 16 * u) = y;
            }
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint32_t x = tid + 256 * i, t = x % kCopyTokens, y = x / kCopyTokens, ds = (t0 + t) & pmask;
                if (live[t]) *reinterpret_cast<uint16_t*>(head_of(dst_page[t]) + p.geom.vs_off + (((ds >> 2) * NB + y) * 4 + (ds & 3)) * 2) = (uint16_t)sv[i];
            }
            if (tid < kCopyTokens && live[tid]) {
                const uint32_t ds = (t0 + tid) & pmask;
                uint32_t* ks = reinterpret_cast<uint32_t*>(head_of(dst_page[tid]) + p.geom.ks_off + ds * (2 * NB));
                ks[0] = of_k;
                if constexpr (NB == 4) ks[1] = of_k2;
                p.sums[(((size_t)dst_page[tid] * p.geom.Hkv + hk) << p.geom.log2_page) + ds] = sum;
            }
        }
    }
}

template <int FMT, int D>
static hipError_t launch_copy(const EvictParams& p, hipStream_t st) {
    const uint64_t want = ((uint64_t)p.budget + kCopyTokens - 1) / kCopyTokens, most = (1u << 24) / p.geom.Hkv;
    const uint32_t tiles = (uint32_t)(want < most ? want : most), across = p.batch.B < 65535 ? p.batch.B : 65535;
    hipLaunchKernelGGL((evict_copy_kernel<FMT, D>), dim3(tiles * p.geom.Hkv, across), dim3(256), 0, st, p, tiles);
    return hipGetLastError();
}

// Workgroups for a sequence and KV head: several where there are fewer of these than CUs and the
// longest is expected to have places for them.  No more than its row of the table has, whatever is
// expected: 4 KB of workspace each.
static uint32_t pick_segments(const EvictParams& p) {
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    if (items >= 256 || p.max_kv <= 2 * kSegment) return 1;
    const uint64_t held = std::max((uint64_t)p.batch.table_pages << p.geom.log2_page, (uint64_t)2 * kSegment + 1);
    return (uint32_t)((std::min((uint64_t)p.max_kv, held) + kSegment - 1) / kSegment);
}

size_t kv_evict_workspace(const EvictParams& p) {
    const uint32_t segments = pick_segments(p);
    return segments > 1 ? PickSpace::bytes((uint64_t)p.batch.B * p.geom.Hkv, segments) : 0;
}

static hipError_t launch_pick(const EvictParams& p, hipStream_t st) {
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    if (p.max_kv && p.max_kv <= (items > kShortItems ? 2 * kShortKeys : kShortKeys)) {
        const dim3 grid((uint32_t)std::min((items + 3) / 4, (uint64_t)1 << 20));
        if (p.max_kv <= kShortKeys) hipLaunchKernelGGL(evict_pick_short_kernel<kShortKeys / 256>, grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL(evict_pick_short_kernel<2 * kShortKeys / 256>, grid, dim3(256), 0, st, p);
        return hipGetLastError();
    }
    const uint32_t segments = pick_segments(p);
    const uint64_t groups = items * segments;
    const uint32_t held = segments > 1 ? 2 * kSegment : (p.max_kv < kHeld ? (p.max_kv + 1023) / 1024 * 1024 : 0);
    const dim3 grid((uint32_t)(groups < (1u << 20) ? groups : 1u << 20)), block(kPickThreads);
    static size_t attr[kMaxDevices] = {};
    hipError_t e = lds_limit_once((const void*)evict_pick_kernel, kHeld * 4, attr);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(evict_pick_kernel, grid, block, held * 4, st, p, held, segments);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (segments > 1) {
        hipLaunchKernelGGL(evict_gather_kernel, grid, block, 0, st, p, segments);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        hipLaunchKernelGGL(evict_place_kernel, grid, block, 0, st, p, segments);
        e = hipGetLastError();
    }
    return e;
}

hipError_t launch_kv_evict(const EvictParams& p, hipStream_t st) {
    if (p.batch.B == 0) return hipSuccess;
    const hipError_t e = launch_pick(p, st);
    if (e != hipSuccess) return e;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_copy<QUANT_Q8_0, 64>(p, st) : launch_copy<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_copy<QUANT_Q4_0, 64>(p, st) : launch_copy<QUANT_Q4_0, 128>(p, st);
}

}  // namespace qr
