// qr_paged_decode.h -- the paged cache's codes as fp16 values, for the kernels that multiply by
// them, and even shares of a line of work.
#pragma once
#include "qr_device.h"
#include "qr_paged.h"

namespace qr {

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

}  // namespace qr
