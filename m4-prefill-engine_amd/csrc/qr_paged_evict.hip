// qr_paged_evict.hip -- a bounded cache: the attention weight that each cached key has
// received, and eviction of the lightest.
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

// The rows (token, query head) of a KV head that see a key are [lo, hi).
struct RowRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ RowRange rows_of(const WeighParams& p, const WeighSeq& s, int key) {
    const int64_t i = (int64_t)key - s.first;
    RowRange r;
    r.lo = (uint32_t)min(max(i, (int64_t)0), (int64_t)s.n) * p.G;
    r.hi = p.window ? (uint32_t)min(max(i + p.window, (int64_t)0), (int64_t)s.n) * p.G : (uint32_t)s.n * p.G;
    return r;
}

// Few rows: four waves of 64 keys each, 16 rows at a time.
template <int FMT, int D>
__global__ void __launch_bounds__(256) weigh_rows_kernel(WeighParams p, uint32_t tiles) {
    constexpr int KK = D / 32, RUN = D / 4, W = FMT == QUANT_Q8_0 ? D / 16 : D / 32;
    constexpr uint32_t CB = 4 * W * 4, NB = D / 32;
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t hk = blockIdx.x % p.geom.Hkv, G = p.G;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;
    const float c = p.scale * 1.4426950408889634f;  // log2 units
    for (uint32_t b = blockIdx.y; b < p.batch.B; b += gridDim.y) {
        const WeighSeq s = weigh_seq(p, b);
        const uint32_t rows = (uint32_t)s.n * G;
        for (int64_t k0 = s.lo / (int)kWaveKeys * (int64_t)kWaveKeys + (int64_t)((blockIdx.x / p.geom.Hkv) * 4 + wave) * kWaveKeys; k0 < s.keys;
             k0 += (int64_t)tiles * 4 * kWaveKeys) {
            const int key0 = (int)k0;
            uint32_t page_id = 0xffffffffu;
            if (lane < 4 && key0 + 16 * lane < s.keys)
                page_id = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)(key0 + 16 * lane) >> p.geom.log2_page)];
            uint32_t page[4], kw[4][W], kd[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                page[t] = __builtin_amdgcn_readlane(page_id, t);
                const uint32_t slot = (uint32_t)(key0 + 16 * t) & pmask;
                const uint8_t* head = p.geom.pages + ((size_t)(page[t] < p.geom.num_pages ? page[t] : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                load_words<W, false>(head + (slot + j) * CB + g * (W * 4), kw[t]);
                kd[t] = *reinterpret_cast<const uint16_t*>(head + p.geom.ks_off + ((slot + j) * NB + g * NB / 4) * 2);
            }
            h8_t kf[4][KK];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int kk = 0; kk < KK; kk++) kf[t][kk] = k_octet<FMT>(kw[t], kk, as_h2(kd[t] | kd[t] << 16));
            RowRange see[4];
#pragma unroll
            for (int t = 0; t < 4; t++) see[t] = rows_of(p, s, key0 + 16 * t + j);
            float sum[4] = {};
            for (uint32_t r0 = 0; r0 < rows; r0 += 16) {
                h8_t qf[KK];
                {
                    const uint32_t f = min(r0 + j, rows - 1);
                    const _Float16* src = p.Q.p + (int64_t)(s.q0 + (int)(f / G)) * p.Q.ts + (int64_t)(hk * G + f % G) * p.Q.hs + g * RUN;
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) qf[kk] = *reinterpret_cast<const h8_t*>(src + 8 * kk);
                }
                float l2[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t f = min(r0 + 4 * g + e, rows - 1);
                    l2[e] = p.lse.p[(int64_t)(s.q0 + (int)(f / G)) * p.lse.ts + (int64_t)(hk * G + f % G) * p.lse.hs] * 1.4426950408889634f;
                }
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    f4_t sc{};
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[kk], kf[t][kk], sc, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t f = r0 + 4 * g + e;
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -l2[e]));
                        sum[t] += f >= see[t].lo && f < see[t].hi ? w : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                sum[t] += __shfl_xor(sum[t], 16);
                sum[t] += __shfl_xor(sum[t], 32);
            }
            const float mine = g == 0 ? sum[0] : (g == 1 ? sum[1] : (g == 2 ? sum[2] : sum[3]));
            const uint32_t at = g == 0 ? page[0] : (g == 1 ? page[1] : (g == 2 ? page[2] : page[3]));
            const int key = key0 + 16 * g + j;
            if (key < s.keys && at < p.geom.num_pages) {
                float* to = p.sums + (((size_t)at * p.geom.Hkv + hk) << p.geom.log2_page) + ((uint32_t)key & pmask);
                *to = key >= s.first ? mine : *to + mine;
            }
        }
    }
}

// Many rows: a workgroup's eight waves hold the same 32 NT keys and share the rows, 32 at a
// time; their sums meet in LDS.
constexpr int kWeighWaves = 8;
constexpr uint32_t kLseRows = 4096;  // lse staged in LDS at once
template <int FMT, int D, int NT>
__global__ void __launch_bounds__(64 * kWeighWaves, 2) weigh_chunk_kernel(WeighParams p, uint32_t tiles) {
    constexpr int KK = D / 16, RUN = D / 2, W = FMT == QUANT_Q8_0 ? D / 8 : D / 16;  // a lane: half a key
    constexpr uint32_t CB = 2 * W * 4, NB = D / 32;
    constexpr int KT = 32 * NT;
    __shared__ __attribute__((aligned(16))) float l2[kLseRows];
    __shared__ float part[kWeighWaves][KT];
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hk = blockIdx.x % p.geom.Hkv, G = p.G;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;
    const float c = p.scale * 1.4426950408889634f;
    for (uint32_t b = blockIdx.y; b < p.batch.B; b += gridDim.y) {
        const WeighSeq s = weigh_seq(p, b);
        const uint32_t rows = (uint32_t)s.n * G;
        for (int64_t k0 = s.lo / KT * (int64_t)KT + (int64_t)(blockIdx.x / p.geom.Hkv) * KT; k0 < s.keys; k0 += (int64_t)tiles * KT) {
            const int key0 = (int)k0;
            uint32_t page_id = 0xffffffffu;
            if (lane < 2 * NT && key0 + 16 * lane < s.keys)
                page_id = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)(key0 + 16 * lane) >> p.geom.log2_page)];
            h8_t kf[NT][KK];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t at = (uint32_t)__shfl((int)page_id, 2 * t + (j >> 4));
                const uint32_t slot = (uint32_t)(key0 + 32 * t + j) & pmask;
                const uint8_t* head = p.geom.pages + ((size_t)(at < p.geom.num_pages ? at : 0) * p.geom.Hkv + hk) * p.geom.head_bytes;
                uint32_t kw[W];
                load_words<W, false>(head + slot * CB + g * (W * 4), kw);
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    const uint32_t kd = *reinterpret_cast<const uint16_t*>(head + p.geom.ks_off + (slot * NB + g * NB / 2 + kk / 4) * 2);
                    kf[t][kk] = k_octet<FMT>(kw, kk, as_h2(kd | kd << 16));
                }
            }
            float sum[NT] = {};
            // rows that see some of these keys, and those that see them all
            const RowRange first_key = rows_of(p, s, key0), last_key = rows_of(p, s, key0 + KT - 1);
            const uint32_t f_lo = first_key.lo / 32 * 32, f_hi = last_key.hi;
            RowRange see[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) see[t] = rows_of(p, s, key0 + 32 * t + j);
            for (uint32_t f0 = f_lo; f0 < f_hi; f0 += kLseRows) {
                __syncthreads();
                for (uint32_t x = tid; x < min(kLseRows, (f_hi - f0 + 31) / 32 * 32); x += 64 * kWeighWaves) {
                    const uint32_t f = f0 + x;
                    l2[x] = f < rows ? p.lse.p[(int64_t)(s.q0 + (int)(f / G)) * p.lse.ts + (int64_t)(hk * G + f % G) * p.lse.hs] * 1.4426950408889634f
                                     : 0.0f;
                }
                __syncthreads();
                const uint32_t f1 = min(f0 + kLseRows, f_hi);
                for (uint32_t r0 = f0 + 32 * wave; r0 < f1; r0 += 32 * kWeighWaves) {
                    h8_t qf[KK];
                    {
                        const uint32_t f = min(r0 + j, rows - 1);
                        const _Float16* src = p.Q.p + (int64_t)(s.q0 + (int)(f / G)) * p.Q.ts + (int64_t)(hk * G + f % G) * p.Q.hs + g * RUN;
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) qf[kk] = *reinterpret_cast<const h8_t*>(src + 8 * kk);
                    }
                    float l[16];
#pragma unroll
                    for (int y = 0; y < 4; y++) *reinterpret_cast<f4_t*>(l + 4 * y) = *reinterpret_cast<const f4_t*>(&l2[r0 - f0 + 8 * y + 4 * g]);
                    const bool whole = r0 >= last_key.lo && r0 + 32 <= first_key.hi;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        f16v_t sc{};
#pragma unroll
                        for (int kk = 0; kk < KK; kk++) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf[kk], kf[t][kk], sc, 0, 0, 0);
                        if (whole) {
#pragma unroll
                            for (int e = 0; e < 16; e++) sum[t] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -l[e]));
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const uint32_t f = r0 + 4 * g + 8 * (e >> 2) + (e & 3);
                                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -l[e]));
                                sum[t] += f >= see[t].lo && f < see[t].hi ? w : 0.0f;
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                sum[t] += __shfl_xor(sum[t], 32);
                if (g == 0) part[wave][32 * t + j] = sum[t];
            }
            __syncthreads();
            for (int x = tid; x < KT; x += 64 * kWeighWaves) {
                const int key = key0 + x;
                float mine = 0.0f;
#pragma unroll
                for (int v = 0; v < kWeighWaves; v++) mine += part[v][x];
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

template <int FMT, int D>
static hipError_t launch_weigh(WeighParams p, hipStream_t st) {
    const uint64_t rows = (uint64_t)(p.max_new ? p.max_new : 1) * p.G;
    uint64_t keys = p.max_kv ? p.max_kv : 1;
    if (p.window && keys > (uint64_t)p.window + p.max_new) keys = (uint64_t)p.window + p.max_new;
    const bool chunks = rows >= kWeighChunk, both = chunks && p.batch.T < (uint64_t)p.batch.B * p.max_new && p.batch.B > 1;
    const uint32_t across = p.batch.B < 65535 ? p.batch.B : 65535;
    auto tiles_of = [&](uint32_t of) {  // of the longest sequence, no more workgroups than a launch may have
        const uint64_t t = (keys + of - 1) / of, most = (1u << 24) / p.geom.Hkv;
        return (uint32_t)(t < most ? t : most);
    };
    p.min_rows = 0;
    p.max_rows = both ? kWeighChunk : 0xffffffffu;
    if (!chunks || both) {
        const uint32_t tiles = tiles_of(4 * kWaveKeys);
        hipLaunchKernelGGL((weigh_rows_kernel<FMT, D>), dim3(tiles * p.geom.Hkv, across), dim3(256), 0, st, p, tiles);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !chunks) return e;
    }
    p.min_rows = both ? kWeighChunk : 0;
    p.max_rows = 0xffffffffu;
    constexpr int NT = 4;
    const uint32_t tiles = tiles_of(32 * NT);
    hipLaunchKernelGGL((weigh_chunk_kernel<FMT, D, NT>), dim3(tiles * p.geom.Hkv, across), dim3(64 * kWeighWaves), 0, st, p, tiles);
    return hipGetLastError();
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

// Weights as integers of the same order; 0 for a place that is not there, the top for one that
// is kept in any case, next to it NaN.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xfffffffeu;
    const uint32_t u = f32_bits(w == 0.0f ? 0.0f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A workgroup a sequence and KV head.  The budget-th largest is found digit by digit, eight bits
// at a time from the top, by counting; then the places at or above it are written in order.
// Keys stay in LDS where it holds them (as many as expected, up to kHeldKeys), else they are
// formed again from the sums.
constexpr int kPickThreads = 1024;
constexpr uint32_t kHeldKeys = 32768, kCopies = 16;
__global__ void __launch_bounds__(kPickThreads) evict_pick_kernel(EvictParams p, uint32_t held_keys) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    u4_t* held = reinterpret_cast<u4_t*>(smem);
    __shared__ uint32_t bins[256 * kCopies];
    __shared__ uint32_t wave_sum[kPickThreads / 64], found[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t pmask = (1u << p.geom.log2_page) - 1;
    for (uint64_t item = blockIdx.x; item < (uint64_t)p.batch.B * p.geom.Hkv; item += gridDim.x) {
        const uint32_t b = (uint32_t)(item / p.geom.Hkv), hk = (uint32_t)(item % p.geom.Hkv);
        const int len = max(p.batch.kv_len[b], 0);
        const uint32_t n = (uint32_t)min((uint64_t)len, (uint64_t)p.batch.table_pages << p.geom.log2_page);
        const int64_t last = (int64_t)len - (int64_t)p.recent;  // kept from there on
        const uint32_t quads = (n + 3) / 4;
        auto form = [&](uint32_t q) {
            u4_t k{};
            const uint32_t page = (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + (4 * q >> p.geom.log2_page)];
            if (page >= p.geom.num_pages) return k;
            const f4_t w = *reinterpret_cast<const f4_t*>(p.sums + (((size_t)page * p.geom.Hkv + hk) << p.geom.log2_page) + (4 * q & pmask));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t at = 4 * q + e;
                if (at < n) k[e] = at < p.sinks || (int64_t)at >= last ? 0xffffffffu : order_of(w[e]);
            }
            return k;
        };
        const bool hold = n <= held_keys;
        auto keys_of = [&](uint32_t q) { return hold ? held[q] : form(q); };
        // those that are there
        uint32_t mine = 0;
        for (uint32_t q = tid; q < quads; q += kPickThreads) {
            const u4_t k = form(q);
            if (hold) held[q] = k;
#pragma unroll
            for (int e = 0; e < 4; e++) mine += k[e] != 0;
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) mine += __shfl_xor((int)mine, x);
        if (lane == 0) wave_sum[wave] = mine;
        __syncthreads();
        uint32_t there = 0;
#pragma unroll
        for (int x = 0; x < kPickThreads / 64; x++) there += wave_sum[x];
        const uint32_t m = min(p.budget, there);
        uint32_t least = 0, equal = 0;  // kept: above `least`, and the first `equal` at it
        if (m < there) {
            uint32_t prefix = 0, want = m;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (uint32_t x = tid; x < 256 * kCopies; x += kPickThreads) bins[x] = 0;
                __syncthreads();
                for (uint32_t q = tid; q < quads; q += kPickThreads) {
                    const u4_t k = keys_of(q);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (k[e] && (shift == 24 || k[e] >> (shift + 8) == prefix)) atomicAdd(&bins[(k[e] >> shift & 255) * kCopies + lane % kCopies], 1u);
                }
                __syncthreads();
                if (tid < 256) {
                    uint32_t of = 0;
#pragma unroll
                    for (uint32_t x = 0; x < kCopies; x++) of += bins[tid * kCopies + (x + tid) % kCopies];
                    bins[tid * kCopies] = of;
                }
                __syncthreads();
                if (wave == 0) {  // a lane four digits; how many lie above them
                    uint32_t of[4], sum = 0;
#pragma unroll
                    for (int x = 0; x < 4; x++) sum += of[x] = bins[(4 * lane + x) * kCopies];
                    uint32_t above = sum;
#pragma unroll
                    for (int x = 1; x < 64; x <<= 1) {
                        const uint32_t y = (uint32_t)__shfl_down((int)above, x);
                        if (lane + x < 64) above += y;
                    }
                    above -= sum;
#pragma unroll
                    for (int x = 3; x >= 0; x--) {
                        if (above < want && want <= above + of[x]) {
                            found[0] = 4 * lane + x;
                            found[1] = want - above;
                        }
                        above += of[x];
                    }
                }
                __syncthreads();
                prefix = prefix << 8 | found[0];
                want = found[1];
            }
            least = prefix;
            equal = want;
        }
        int32_t* out = p.kept + ((size_t)b * p.geom.Hkv + hk) * p.budget;
        // counts of those above and at the threshold, 16 bits each
        uint32_t above0 = 0, equal0 = 0;
        for (uint32_t q0 = 0; q0 < quads; q0 += kPickThreads) {
            const uint32_t q = q0 + tid;
            const u4_t k = q < quads ? keys_of(q) : u4_t{};
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) c += (k[e] > least ? 1u : 0u) + (k[e] == least && k[e] ? 0x10000u : 0u);
            uint32_t incl = c;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                const uint32_t y = (uint32_t)__shfl_up((int)incl, x);
                if (lane >= (uint32_t)x) incl += y;
            }
            __syncthreads();
            if (lane == 63) wave_sum[wave] = incl;
            __syncthreads();
            uint32_t before = incl - c, all = 0;
#pragma unroll
            for (uint32_t x = 0; x < kPickThreads / 64; x++) {
                if (x < wave) before += wave_sum[x];
                all += wave_sum[x];
            }
            uint32_t na = above0 + (before & 0xffffu), ne = equal0 + (before >> 16);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool a = k[e] > least, at = k[e] == least && k[e];
                if (a || (at && ne < equal)) out[na + min(ne, equal)] = (int32_t)(4 * q + e);
                na += a;
                ne += at;
            }
            above0 += all & 0xffffu;
            equal0 += all >> 16;
        }
        for (uint32_t x = m + tid; x < p.budget; x += kPickThreads) out[x] = -1;
        if (hk == 0 && tid == 0) p.len_out[b] = (int32_t)m;
        __syncthreads();
    }
}

// Kept token i becomes token i of the other table's pages: 64 of them a workgroup, of one head.
// Codes of V lie in groups of four tokens, so four sources' bytes make a word; where the last
// group is not full, the others of its tokens keep their own.
constexpr uint32_t kCopyTokens = 64;
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
                const int from = i < p.budget ? kept[i] : -1;
                uint32_t dp = pi < p.out_pages ? (uint32_t)p.table_out[(size_t)b * p.out_stride + pi] : 0xffffffffu;
                if (dp >= p.geom.num_pages) dp = 0xffffffffu;
                dst_page[tid] = dp;
                live[tid] = from >= 0 && dp != 0xffffffffu;
                if (tid == 0) some = from >= 0;
                src_page[tid] = from >= 0 ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + ((uint32_t)from >> p.geom.log2_page)] : dp;
                src_slot[tid] = (uint32_t)(from >= 0 ? from : (int)i) & pmask;
            }
            __syncthreads();
            if (!some) break;  // the kept are the first
            for (uint32_t x = tid; x < kCopyTokens * KP; x += 256) {
                const uint32_t t = x / KP, u = x % KP;
                if (!live[t]) continue;
                *reinterpret_cast<u4_t*>(head_of(dst_page[t]) + ((t0 + t) & pmask) * CB + 16 * u) =
                    *reinterpret_cast<const u4_t*>(head_of(src_page[t]) + src_slot[t] * CB + 16 * u);
            }
            for (uint32_t x = tid; x < kCopyTokens / 4 * VP; x += 256) {
                const uint32_t t = x / VP * 4, u = x % VP;
                if (!live[t]) continue;
                u4_t w[4];
                uint32_t k[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t slot = src_slot[t + e];
                    k[e] = slot & 3;
                    w[e] = *reinterpret_cast<const u4_t*>(head_of(src_page[t + e]) + p.geom.v_off + (slot >> 2) * (4 * CB) + 16 * u);
                }
                const uint32_t lo = k[0] | (4 + k[1]) << 8 | 0x0c0c0000u, hi = 0x0c0cu | k[2] << 16 | (4 + k[3]) << 24;
                u4_t y;
#pragma unroll
                for (int d = 0; d < 4; d++) y[d] = perm(w[1][d], w[0][d], lo) | perm(w[3][d], w[2][d], hi);
                *reinterpret_cast<u4_t*>(head_of(dst_page[t]) + p.geom.v_off + ((t0 + t) & pmask) / 4 * (4 * CB) + 16 * u) = y;
            }
            // scales and sums: a token's of K and its sum, and of V block by block
            for (uint32_t x = tid; x < kCopyTokens * (1 + NB); x += 256) {
                const uint32_t t = x % kCopyTokens, y = x / kCopyTokens;
                if (!live[t]) continue;
                const uint8_t* src = head_of(src_page[t]);
                uint8_t* dst = head_of(dst_page[t]);
                const uint32_t ss = src_slot[t], ds = (t0 + t) & pmask;
                if (y == 0) {
                    p.sums[(((size_t)dst_page[t] * p.geom.Hkv + hk) << p.geom.log2_page) + ds] =
                        p.sums[(((size_t)src_page[t] * p.geom.Hkv + hk) << p.geom.log2_page) + ss];
                    if constexpr (NB == 4)
                        *reinterpret_cast<u2_t*>(dst + p.geom.ks_off + ds * 8) = *reinterpret_cast<const u2_t*>(src + p.geom.ks_off + ss * 8);
                    else
                        *reinterpret_cast<uint32_t*>(dst + p.geom.ks_off + ds * 4) = *reinterpret_cast<const uint32_t*>(src + p.geom.ks_off + ss * 4);
                } else {
                    *reinterpret_cast<uint16_t*>(dst + p.geom.vs_off + (((ds >> 2) * NB + y - 1) * 4 + (ds & 3)) * 2) =
                        *reinterpret_cast<const uint16_t*>(src + p.geom.vs_off + (((ss >> 2) * NB + y - 1) * 4 + (ss & 3)) * 2);
                }
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

hipError_t launch_kv_evict(const EvictParams& p, hipStream_t st) {
    if (p.batch.B == 0) return hipSuccess;
    const uint64_t items = (uint64_t)p.batch.B * p.geom.Hkv;
    static size_t attr[kMaxDevices] = {};
    const uint32_t held = p.max_kv < kHeldKeys ? (p.max_kv + 1023) / 1024 * 1024 : kHeldKeys;
    hipError_t e = lds_limit_once((const void*)evict_pick_kernel, kHeldKeys * 4, attr);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(evict_pick_kernel, dim3((uint32_t)(items < (1u << 20) ? items : 1u << 20)), dim3(kPickThreads), held * 4, st, p, held);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.format == QUANT_Q8_0) return p.D == 64 ? launch_copy<QUANT_Q8_0, 64>(p, st) : launch_copy<QUANT_Q8_0, 128>(p, st);
    return p.D == 64 ? launch_copy<QUANT_Q4_0, 64>(p, st) : launch_copy<QUANT_Q4_0, 128>(p, st);
}

}  // namespace qr
