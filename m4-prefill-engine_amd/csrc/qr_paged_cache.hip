// qr_paged_cache.hip -- rotary positions with several axes, quantizing a paged
// KV cache as it is written, and reading it back.
#include "qr_device.h"
#include "qr_paged.h"

namespace qr {

constexpr uint64_t kBlocks = 1024;  // that fill the chip
// Bytes from which rows that are read once are loaded past the caches (what the L2
// caches hold together), and results stored past them.
constexpr uint64_t kLoadPast = (uint64_t)32 << 20, kStorePast = (uint64_t)64 << 20;

// Where a token lies in the cache.
struct Place {
    uint32_t page, slot;
    int pos;
    bool ok;
};
// The places of rows t0 .. t0 + RPW - 1, lane's own in row t0 + sub: the lanes
// count the sequences that begin at or below each row, 64 at a time, and the
// rest is looked up for all rows at once.  Not ok: rows behind the last
// sequence, tokens before position 0 and tokens whose page is not there.
template <int RPW>
__device__ __forceinline__ Place place_of(const BatchView& bv, const PageGeom& g, uint32_t t0, int sub, int lane) {
    Place r{0, 0, 0, false};
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < bv.B; b0 += 64) {
        const uint32_t b = b0 + lane;
        const int start = b < bv.B ? bv.q_start[b] : 0x7fffffff;
        uint32_t n = 0;
#pragma unroll
        for (int s = 0; s < RPW; s++) {
            n = __popcll(__ballot(start <= (int)(t0 + s)));
            before += s == sub ? n : 0;
        }
        if (n < 64) break;
    }
    const uint32_t t = t0 + sub;
    if (before == 0 || t >= bv.T) return r;
    const uint32_t b = before - 1;
    const int end = bv.q_start[b + 1], len = max(bv.kv_len[b], 0);  // an end past T: rows that are not there
    if ((int)t >= end) return r;
    r.pos = len - (end - (int)t);
    if (r.pos < 0) return r;
    const uint32_t pi = (uint32_t)r.pos >> g.log2_page;
    if (pi >= bv.table_pages) return r;
    r.page = (uint32_t)bv.table[(size_t)b * bv.table_stride + pi];
    r.slot = (uint32_t)r.pos & ((1u << g.log2_page) - 1);
    r.ok = r.page < g.num_pages;
    return r;
}

// Sine and cosine of a fraction of a turn in 2^-32: the nearest quarter turn comes
// off as bits, what is left, at most pi / 4, goes through the Taylor series (left
// out: x^11 / 11! and x^12 / 12!, below 2^-28).  Within 2^-23.3, 2^-25.5 rms.  The
// hardware's own, within 2^-22.9, take 0.3 us less, but let more fp16 roundings and
// Q4_0 codes fall on the other side: K of three prompts, off by 2.1e-4 of its norm
// from the same in 64 bits, would be off by 2.5e-4.
__device__ __forceinline__ void sincos_turn(uint32_t turn, float& sn, float& cs) {
    const uint32_t quarter = turn + 0x20000000u;
    const float x = (float)(int32_t)((quarter & 0x3fffffffu) - 0x20000000u) * (6.283185307179586f * 0x1p-32f), x2 = x * x;
    float a = __builtin_fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
    a = __builtin_fmaf(x2, a, 8.3333333e-3f);
    a = __builtin_fmaf(x2, a, -1.6666667e-1f);
    a = __builtin_fmaf(x2 * x, a, x);
    float b = __builtin_fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
    b = __builtin_fmaf(x2, b, -1.3888889e-3f);
    b = __builtin_fmaf(x2, b, 4.1666667e-2f);
    b = __builtin_fmaf(x2, b, -0.5f);
    b = __builtin_fmaf(x2, b, 1.0f);
    const bool odd = quarter >> 30 & 1;
    const uint32_t flip_s = quarter & 0x80000000u, flip_c = (quarter + 0x40000000u) & 0x80000000u;
    sn = __builtin_bit_cast(float, f32_bits(odd ? b : a) ^ flip_s);
    cs = __builtin_bit_cast(float, f32_bits(odd ? a : b) ^ flip_c);
}

// Codes of 8 dims of a block of 32 that four neighbouring lanes hold (lane & 3
// the quarter), and the block's scale.  Q8_0 as quantize_block_q8_0: the code
// rounds x * (1 / d), d = amax / 127 in fp32, half away from zero, and is stored
// plus 128.  Q4_0: d = m / -8 of the value m of largest magnitude (the first of
// a tie), code = floor(x (1 / d) + 8.5), product and sum rounded apart.
template <int FMT>
__device__ __forceinline__ void quantize8(const float x[8], int lane, uint32_t code[8], uint32_t& d16) {
    if constexpr (FMT == QUANT_Q8_0) {
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const float d = amax / 127.0f;
        const float id = d > 0.0f ? 1.0f / d : 0.0f;
        d16 = f2h_bits(d);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            int q = (int)__builtin_roundf(x[e] * id);
            q = q < -128 ? -128 : (q > 127 ? 127 : q);
            code[e] = (uint32_t)(q + 128);
        }
    } else {
        // magnitude (15 bits of fp16), then the earliest index, then the sign
        uint32_t key = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t h = f2h_bits(x[e]);
            key = max(key, (h & 0x7fffu) << 6 | (uint32_t)(31 - (8 * (lane & 3) + e)) << 1 | h >> 15);
        }
        key = max(key, (uint32_t)__shfl_xor((int)key, 1));
        key = max(key, (uint32_t)__shfl_xor((int)key, 2));
        float d = h2f(key >> 6 | (key & 1u) << 15) / -8.0f;
        // apart from the rounding below: as one mixed-precision instruction the two lose a zero's sign
        asm volatile("" : "+v"(d));
        const float id = d != 0.0f ? 1.0f / d : 0.0f;
        d16 = f2h_bits(d);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float c = __builtin_floorf(__fadd_rn(__fmul_rn(x[e], id), 8.5f));
            code[e] = (uint32_t)(int)fminf(fmaxf(c, 0.0f), 15.0f);
        }
    }
}

// One row of T tokens per LPR lanes, 8 dims a lane; a wave takes 64 / LPR tokens
// and every so many of the heads, of Q (the first q_blocks of a row of blocks) or
// of K and V, so angles are formed once per wave and used for all its heads.  A
// rotated row is rounded to fp16 before it is quantized, as a rotation and a write
// apart would.  Bound by bytes once there are enough: 8100 tokens of 32 heads
// (133 MB) 27 us, 4.9 TB/s; 64 tokens 5 us, a chain of table and angle latencies.
// PAST: rows of Q, kLoadPast bytes and more, are loaded past the caches, which keep
// the turned ones: 30 us without; then attention over as many keys 710 us with both.
// Stored past them too it is 25, and the attention that reads them longer by more.
template <int LPR, int FMT, bool PAST>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendParams p, uint32_t q_blocks) {
    constexpr int RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = lane % LPR, sub = lane / LPR;
    const uint32_t t0 = (blockIdx.x * 4 + wave) * RPW, t = t0 + sub;
    const bool of_q = blockIdx.y < q_blocks;
    const uint32_t chunk = of_q ? blockIdx.y : blockIdx.y - q_blocks, chunks = of_q ? q_blocks : gridDim.y - q_blocks;
    const uint32_t heads = of_q ? p.H : p.geom.Hkv;
    if (t0 >= p.T) return;
    const bool live = t < p.T && 8u * l < p.D;

    // Heads chunk, chunk + chunks, ...: kAhead rows of Q, or kAhead / 2 of K and of V,
    // are loaded together, the next while these are turned and stored; the first are
    // under way while places and angles are found.
    constexpr int kAhead = 4;
    h8_t next[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) next[i] = h8_t{};
    const _Float16 *src = nullptr, *src2 = nullptr;  // the next row to load, of V too
    int64_t step, step2 = 0;
    if (of_q) {
        src = p.Q.p + (int64_t)t * p.Q.ts + (int64_t)chunk * p.Q.hs + 8 * l;
        step = (int64_t)chunks * p.Q.hs;
    } else {
        src = p.K.p + (int64_t)t * p.K.ts + (int64_t)chunk * p.K.hs + 8 * l;
        src2 = p.V.p + (int64_t)t * p.V.ts + (int64_t)chunk * p.V.hs + 8 * l;
        step = (int64_t)chunks * p.K.hs;
        step2 = (int64_t)chunks * p.V.hs;
    }
    uint32_t ahead = chunk;  // its head
    auto fetch = [&]() {
        if (of_q) {
#pragma unroll
            for (int i = 0; i < kAhead; i++, ahead += chunks, src += step)
                if (ahead < heads && live) {
                    if constexpr (PAST) next[i] = __builtin_nontemporal_load(reinterpret_cast<const h8_t*>(src));
                    else next[i] = *reinterpret_cast<const h8_t*>(src);
                }
        } else {
#pragma unroll
            for (int i = 0; i < kAhead; i += 2, ahead += chunks, src += step, src2 += step2)
                if (ahead < heads && live) {
                    next[i] = *reinterpret_cast<const h8_t*>(src);
                    next[i + 1] = *reinterpret_cast<const h8_t*>(src2);
                }
        }
    };
    fetch();

    Place at{0, 0, 0, false};
    bool row = live;
    if (p.batch.q_start) {
        at = place_of<RPW>(p.batch, p.geom, t0, sub, lane);
        // rows of Q with no place in the cache (behind the last sequence) stay
        row = live && at.ok;
    }

    // angles of this lane's pairs; `turned`: its dims take part, `other`: the
    // lane that holds the partners of its dims
    const uint32_t hp = p.rope.pairs / 8;  // lanes of the first halves
    bool turned;
    int other = lane;
    uint32_t pair0;
    if (p.rope.traditional) {
        turned = 4u * l < p.rope.pairs;
        pair0 = 4 * l;
    } else {
        turned = (uint32_t)l < 2 * hp;
        const bool second = (uint32_t)l >= hp;
        pair0 = 8 * (second ? l - hp : l);
        if (turned) other = second ? lane - (int)hp : lane + (int)hp;
    }
    float cs[8], sn[8];
    if (turned && row) {
        const int n = p.rope.traditional ? 4 : 8;
        const uint32_t* axis = reinterpret_cast<const uint32_t*>(p.rope.table + p.rope.pairs);
        // up to four axes' positions are loaded beside the table, more behind it
        int pos[4] = {at.pos, 0, 0, 0};
        if (p.rope.positions)
#pragma unroll
            for (int a = 0; a < 4; a++)
                if (a < (int)p.rope.axes) pos[a] = p.rope.positions[(size_t)a * p.rope.position_stride + t];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (e >= n) break;
            int at_axis = pos[0];
            if (p.rope.axes > 1) {
                const uint32_t a = min(axis[pair0 + e], p.rope.axes - 1);
                at_axis = a == 0 ? pos[0] : (a == 1 ? pos[1] : (a == 2 ? pos[2] : pos[3]));
                if (a > 3) at_axis = p.rope.positions[(size_t)a * p.rope.position_stride + t];
            }
            const uint64_t frac = (uint64_t)(int64_t)at_axis * p.rope.table[pair0 + e];
            sincos_turn((uint32_t)(frac >> 32), sn[e], cs[e]);
        }
        if (p.rope.traditional) {
#pragma unroll
            for (int e = 3; e >= 0; e--) {  // of dims 2 e and 2 e + 1
                cs[2 * e + 1] = cs[2 * e] = cs[e];
                sn[2 * e + 1] = sn[e];
                sn[2 * e] = -sn[e];
            }
        } else if ((uint32_t)l < hp) {
#pragma unroll
            for (int e = 0; e < 8; e++) sn[e] = -sn[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            cs[e] = 1.0f;
            sn[e] = 0.0f;
        }
        turned = false;
    }
    const bool any_turned = p.rope.pairs != 0;

    auto turn = [&](h8_t y) {
        u4_t mine = __builtin_bit_cast(u4_t, y), theirs;
        if (p.rope.traditional) {
            theirs = u4_t{mine.x >> 16 | mine.x << 16, mine.y >> 16 | mine.y << 16, mine.z >> 16 | mine.z << 16,
                          mine.w >> 16 | mine.w << 16};
        } else {
            theirs = u4_t{(uint32_t)__shfl((int)mine.x, other), (uint32_t)__shfl((int)mine.y, other),
                          (uint32_t)__shfl((int)mine.z, other), (uint32_t)__shfl((int)mine.w, other)};
        }
        const h8_t z = __builtin_bit_cast(h8_t, theirs);
        if (turned) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = (_Float16)((float)y[e] * cs[e] + (float)z[e] * sn[e]);
        }
        return y;
    };

    if (of_q) {
        _Float16* dst = p.Qo.p + (int64_t)t * p.Qo.ts + (int64_t)chunk * p.Qo.hs + 8 * l;
        for (uint32_t h = chunk; h < heads;) {
            h8_t now[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) now[i] = next[i];
            fetch();
#pragma unroll
            for (int i = 0; i < kAhead; i++, h += chunks, dst += (int64_t)chunks * p.Qo.hs) {
                if (h >= heads) break;
                const h8_t y = any_turned ? turn(now[i]) : now[i];
                if (row) *reinterpret_cast<h8_t*>(dst) = y;
            }
        }
        return;
    }
    if constexpr (FMT >= 0) {
        constexpr uint32_t D = LPR * 8, NB = D / 32, CB = FMT == QUANT_Q8_0 ? D : D / 2;
        const uint32_t g4 = at.slot >> 2, k4 = at.slot & 3;
        for (uint32_t h = chunk; h < heads;) {
            h8_t now[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) now[i] = next[i];
            fetch();
#pragma unroll
            for (int i = 0; i < kAhead; i += 2, h += chunks) {
                if (h >= heads) break;
                const h8_t k = any_turned ? turn(now[i]) : now[i], v = now[i + 1];
                float x[8];
                uint32_t c[8], d16;
                uint8_t* head = p.geom.pages + ((size_t)at.page * p.geom.Hkv + h) * p.geom.head_bytes;
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = (float)k[e];
                quantize8<FMT>(x, lane, c, d16);
                if (row) {
                    uint8_t* o = head + at.slot * CB;
                    if constexpr (FMT == QUANT_Q8_0) {
                        *reinterpret_cast<u2_t*>(o + 8 * l) = u2_t{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                                                                   c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
                    } else {
                        *reinterpret_cast<uint32_t*>(o + 4 * l) =
                            c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24 | c[4] << 4 | c[5] << 12 | c[6] << 20 | c[7] << 28;
                    }
                    if (l % 4 == 0)
                        *reinterpret_cast<uint16_t*>(head + p.geom.ks_off + (at.slot * NB + l / 4) * 2) = (uint16_t)d16;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = (float)v[e];
                quantize8<FMT>(x, lane, c, d16);
                if (row) {
                    uint8_t* o = head + p.geom.v_off + g4 * (4 * CB) + k4;
                    if constexpr (FMT == QUANT_Q8_0) {
#pragma unroll
                        for (int e = 0; e < 8; e++) o[(8 * l + e) * 4] = (uint8_t)c[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[(4 * l + e) * 4] = (uint8_t)(c[2 * e] | c[2 * e + 1] << 4);
                    }
                    if (l % 4 == 0)
                        *reinterpret_cast<uint16_t*>(head + p.geom.vs_off + ((g4 * NB + l / 4) * 4 + k4) * 2) = (uint16_t)d16;
                }
            }
        }
    }
}

hipError_t launch_kv_append(const AppendParams& p, hipStream_t st) {
    if (p.T == 0) return hipSuccess;
    const int lpr = p.D <= 64 ? 8 : (p.D <= 128 ? 16 : 32);
    if (p.D > 256 || p.D % 8 || p.rope.pairs > 128 || p.rope.pairs % 8 || 2 * p.rope.pairs > p.D)
        return hipErrorInvalidValue;
    if (p.geom.pages && p.D != 64 && p.D != 128) return hipErrorInvalidValue;
    // four waves of rows side by side; the heads of Q, and those of K and V, over as
    // many blocks as fill the chip (8100 x 32 heads: 1024 blocks 30.3 us, 4096 39.9)
    const uint32_t rows = 4 * 64 / lpr, groups = (p.T + rows - 1) / rows;
    uint32_t q_blocks = p.H, kv_blocks = p.geom.pages ? p.geom.Hkv : 0;
    if (q_blocks + kv_blocks == 0) return hipSuccess;
    // a head of K and V takes longer than eight of Q (three prompts of a 1B model, with
    // the read back: counted as 2 / 4 / 8 of Q 21.4 / 20.3 / 19.4 us)
    for (uint32_t each = 1; (uint64_t)groups * (q_blocks + kv_blocks) > kBlocks && each < 0x10000; each *= 2) {
        const uint32_t of_kv = each > 8 ? each / 8 : 1;
        q_blocks = (p.H + each - 1) / each;
        kv_blocks = p.geom.pages ? (p.geom.Hkv + of_kv - 1) / of_kv : 0;
    }
    const dim3 grid(groups, q_blocks + kv_blocks);
    const int fmt = p.geom.pages ? p.format : -1;
    const bool past = (uint64_t)p.T * p.H * p.D * 2 >= kLoadPast;
#define QR_APPEND(L, F)                                                                              \
    if (past) hipLaunchKernelGGL((kv_append_kernel<L, F, true>), grid, dim3(256), 0, st, p, q_blocks); \
    else hipLaunchKernelGGL((kv_append_kernel<L, F, false>), grid, dim3(256), 0, st, p, q_blocks)
    switch (fmt * 32 + lpr) {
        case -32 + 8: QR_APPEND(8, -1); break;
        case -32 + 16: QR_APPEND(16, -1); break;
        case -32 + 32: QR_APPEND(32, -1); break;
        case QUANT_Q8_0 * 32 + 8: QR_APPEND(8, QUANT_Q8_0); break;
        case QUANT_Q8_0 * 32 + 16: QR_APPEND(16, QUANT_Q8_0); break;
        case QUANT_Q4_0 * 32 + 8: QR_APPEND(8, QUANT_Q4_0); break;
        case QUANT_Q4_0 * 32 + 16: QR_APPEND(16, QUANT_Q4_0); break;
        default: return hipErrorInvalidValue;
    }
#undef QR_APPEND
    return hipGetLastError();
}

// The values of the batch's rows: half(q half(d)), or half((c - 8) half(d)).  A
// lane reads 8 dims of a token; of V the four tokens of its group, of which it
// keeps its own (the other three lanes' reads of the same bytes hit the cache).
// PAST: stores that do not stay in the caches, from kStorePast bytes of results
// on.  us without / with: 91 MB 36.7 / 25.0 (5.7 TB/s), and with a copy of the
// results behind it 85 MB 71 / 78, 195 MB 159 / 158; 39 MB 46.7 / 50.0.
template <int LPR, int FMT, bool PAST>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams p) {
    constexpr int RPW = 64 / LPR;
    constexpr uint32_t D = LPR * 8, NB = D / 32, CB = FMT == QUANT_Q8_0 ? D : D / 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = lane % LPR, sub = lane / LPR;
    const uint32_t t0 = (blockIdx.x * 4 + wave) * RPW, t = t0 + sub;
    const uint32_t chunk = blockIdx.y, chunks = gridDim.y, items = 2 * p.geom.Hkv;
    if (t0 >= p.batch.T) return;
    const Place at = place_of<RPW>(p.batch, p.geom, t0, sub, lane);
    if (!at.ok) return;
    for (uint32_t it = chunk; it < items; it += chunks) {
        const bool is_k = it < p.geom.Hkv;
        const uint32_t h = is_k ? it : it - p.geom.Hkv;
        const uint8_t* head = p.geom.pages + ((size_t)at.page * p.geom.Hkv + h) * p.geom.head_bytes;
        float q[8];
        uint32_t d16;
        if (is_k) {
            const uint8_t* c = head + at.slot * CB;
            d16 = *reinterpret_cast<const uint16_t*>(head + p.geom.ks_off + (at.slot * NB + l / 4) * 2);
            if constexpr (FMT == QUANT_Q8_0) {
                const u2_t w = *reinterpret_cast<const u2_t*>(c + 8 * l);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    q[e] = (float)(int)((w.x >> (8 * e) & 0xffu)) - 128.0f;
                    q[4 + e] = (float)(int)((w.y >> (8 * e) & 0xffu)) - 128.0f;
                }
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(c + 4 * l);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    q[e] = (float)(int)(w >> (8 * e) & 15u) - 8.0f;
                    q[4 + e] = (float)(int)(w >> (8 * e + 4) & 15u) - 8.0f;
                }
            }
        } else {
            const uint32_t g4 = at.slot >> 2, k4 = at.slot & 3;
            d16 = *reinterpret_cast<const uint16_t*>(head + p.geom.vs_off + ((g4 * NB + l / 4) * 4 + k4) * 2);
            const u4_t* c = reinterpret_cast<const u4_t*>(head + p.geom.v_off + g4 * (4 * CB) + l * (4 * CB / LPR));
            const u4_t a = c[0];
            if constexpr (FMT == QUANT_Q8_0) {
                const u4_t b = c[1];
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; e++) q[e] = (float)(int)(w[e] >> (8 * k4) & 0xffu) - 128.0f;
            } else {
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    q[2 * e] = (float)(int)(w[e] >> (8 * k4) & 15u) - 8.0f;
                    q[2 * e + 1] = (float)(int)(w[e] >> (8 * k4 + 4) & 15u) - 8.0f;
                }
            }
        }
        const float d = h2f(d16);
        h8_t y;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (_Float16)(q[e] * d);
        const RowsView& dst = is_k ? p.K : p.V;
        h8_t* to = reinterpret_cast<h8_t*>(dst.p + (int64_t)t * dst.ts + (int64_t)h * dst.hs + 8 * l);
        if constexpr (PAST) __builtin_nontemporal_store(y, to);
        else *to = y;
    }
}

hipError_t launch_kv_read(const ReadParams& p, hipStream_t st) {
    if (p.batch.T == 0 || p.geom.Hkv == 0) return hipSuccess;
    if (p.D != 64 && p.D != 128) return hipErrorInvalidValue;
    const uint32_t rows = p.D == 64 ? 32 : 16, groups = (p.batch.T + rows - 1) / rows;
    uint32_t blocks = 2 * p.geom.Hkv;
    while (blocks > 1 && (uint64_t)groups * blocks > kBlocks) blocks = (blocks + 1) / 2;
    const dim3 grid(groups, blocks);
    const bool past = (uint64_t)p.batch.T * p.geom.Hkv * p.D * 4 >= kStorePast;
#define QR_READ(L, F)                                                                        \
    if (past) hipLaunchKernelGGL((kv_read_kernel<L, F, true>), grid, dim3(256), 0, st, p);   \
    else hipLaunchKernelGGL((kv_read_kernel<L, F, false>), grid, dim3(256), 0, st, p);       \
    break
    switch ((p.D == 128 ? 1 : 0) + (p.format == QUANT_Q8_0 ? 2 : 0)) {
        case 0: QR_READ(8, QUANT_Q4_0);
        case 1: QR_READ(16, QUANT_Q4_0);
        case 2: QR_READ(8, QUANT_Q8_0);
        default: QR_READ(16, QUANT_Q8_0);
    }
#undef QR_READ
    return hipGetLastError();
}

}  // namespace qr
