// qr_paged_tree.hip -- trees of drafted tokens: which nodes each one has before it, the walk
// that accepts a path of them, and the move of the path's tokens to their places.
#include "qr_device.h"
#include "qr_paged.h"

namespace qr {

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane) << 32 | (uint32_t)__shfl((int)(uint32_t)v, lane);
}

// A node's ancestors are itself and its parent's, anc(i) = {i} + anc(parent(i)), and a parent
// comes before its nodes.  64 nodes at a time, a lane each: pointers are doubled six times, so
// that every node has its ancestors among the 64 as one word; the lowest of them says where
// the path leaves the 64, to an earlier node or to none.
struct Near {
    uint64_t bits;
    int exit;
};
__device__ __forceinline__ Near near_of(int parent, int base, int lane) {
    int jump = parent >= base ? parent - base : -1;
    const int leave = parent >= 0 && parent < base ? parent : -1;
    uint64_t near = (uint64_t)1 << lane;
#pragma unroll
    for (int r = 0; r < 6; r++) {
        const int at = jump < 0 ? lane : jump;
        near |= shfl_u64(near, at);
        const int further = __shfl(jump, at);
        jump = jump < 0 ? -1 : further;
    }
    return Near{near, __shfl(leave, __ffsll((unsigned long long)near) - 1)};
}

// A block a sequence.  Up to kHeldNodes the words of all its 64s are formed side by side and kept
// in LDS; then a thread follows each node's path from 64 to 64 and writes its row.  Longer trees
// take one 64 after the other, whose rows copy the rest from those that are there already (300
// nodes of 64 requests so: 10.5 us, a round trip to memory for each 64; in LDS 4.5).
constexpr int kHeldNodes = 2048;
template <int THREADS>
__global__ void __launch_bounds__(THREADS) draft_tree_kernel(DraftParams p) {
    __shared__ uint64_t near[kHeldNodes];
    __shared__ int leave[kHeldNodes];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t W = p.words;
    for (uint32_t b = blockIdx.x; b < p.batch.B; b += gridDim.x) {
        const NewRows s = new_rows(p.batch, b);
        uint32_t* mask = p.mask + (size_t)s.q0 * W;
        auto parent_of = [&](int i) {
            const int parent = i < s.n ? p.parents[s.q0 + i] : -1;
            return parent < i ? parent : -1;
        };
        if (s.n <= kHeldNodes) {
            for (int base = 64 * wave; base < s.n; base += THREADS) {
                const Near at = near_of(parent_of(base + lane), base, lane);
                near[base + lane] = at.bits;
                leave[base + lane] = at.exit;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < s.n; i += THREADS) {
                uint32_t* row = mask + (size_t)i * W;
                int cur = i, depth = 0;
                for (uint32_t w = i / 64 * 2 + 2; w < W; w++) row[w] = 0;
                for (int x = i / 64; x >= 0; x--) {
                    uint64_t bits = 0;
                    if (cur >= 64 * x) {  // else the path passes these by
                        bits = near[cur];
                        cur = leave[cur];
                        depth += __popcll(bits);
                    }
                    if (2u * x < W) row[2 * x] = (uint32_t)bits;
                    if (2 * x + 1u < W) row[2 * x + 1] = (uint32_t)(bits >> 32);
                }
                p.places[s.q0 + i] = s.first + depth - 1;
            }
            __syncthreads();
            continue;
        }
        for (int base = 0; base < s.n; base += 64) {
            const int i = base + lane, parent = parent_of(i);
            if (wave == 0) {
                const Near at = near_of(parent, base, lane);
                near[lane] = at.bits;
                leave[lane] = at.exit;
                if (i < s.n) p.places[s.q0 + i] = (at.exit >= 0 ? p.places[s.q0 + at.exit] + 1 : s.first) + __popcll(at.bits) - 1;
            }
            __syncthreads();
            const uint32_t rows = min(s.n - base, 64), own = (uint32_t)base / 32;
            for (uint32_t x = threadIdx.x; x < rows * W; x += THREADS) {  // W is at most 2^21
                const uint32_t r = x / W, w = x % W;
                uint32_t bits = 0;
                if (w == own) bits = (uint32_t)near[r];
                else if (w == own + 1) bits = (uint32_t)(near[r] >> 32);
                else if (w < own && leave[r] >= 0) bits = mask[(size_t)leave[r] * W + w];
                mask[(size_t)base * W + x] = bits;
            }
            __syncthreads();  // rows of later nodes copy these
        }
    }
}

hipError_t launch_draft_tree(const DraftParams& p, hipStream_t st) {
    if (p.batch.B == 0 || p.batch.T == 0) return hipSuccess;
    hipLaunchKernelGGL(draft_tree_kernel<256>, dim3(min(p.batch.B, 1u << 20)), dim3(256), 0, st, p);
    return hipGetLastError();
}

// A call without rows has results for its sequences all the same, and needs nothing else: q_start may be null then.
__device__ __forceinline__ NewRows rows_if_any(const BatchView& v, uint32_t b) { return v.T ? new_rows(v, b) : NewRows{0, 0, 0}; }

// From node 0 on, the first node behind the present one that is its child and whose token is
// the model's choice there.  A wave a sequence, 64 nodes at a time: a child of the present node is
// one ballot, so what it takes is the loads (26 nodes 1.7 us, 64 requests of 64 nodes 3.8).
__global__ void __launch_bounds__(64) tree_accept_kernel(AcceptParams p) {
    const int lane = threadIdx.x;
    for (uint32_t b = blockIdx.x; b < p.batch.B; b += gridDim.x) {
        const NewRows s = rows_if_any(p.batch, b);
        const int32_t *parents = p.parents + s.q0, *tokens = p.tokens + s.q0, *targets = p.targets + s.q0;
        int count = 0, next = -1;
        if (s.n > 0) {
            int cur = 0, base = 0, parent = -1, token = 0, target = 0;
            auto load = [&](int from) {
                base = from;
                const int i = base + lane;
                parent = i < s.n ? parents[i] : -1;
                token = i < s.n ? tokens[i] : 0;
                target = i < s.n ? targets[i] : 0;
            };
            load(0);
            next = __builtin_amdgcn_readlane(target, 0);
            if (lane == 0) p.path[s.q0] = 0;
            count = 1;
            for (;;) {
                const uint64_t fits = __ballot(parent == cur && token == next && base + lane > cur && base + lane < s.n);
                if (fits) {
                    const int at = __ffsll((unsigned long long)fits) - 1;
                    cur = base + at;
                    next = __builtin_amdgcn_readlane(target, at);
                    if (lane == 0) p.path[s.q0 + count] = cur;
                    count++;
                    continue;  // its child may be among the same 64
                }
                if (base + 64 >= s.n) break;
                load(base + 64);
            }
        }
        for (int i = count + lane; i < s.n; i += 64) p.path[s.q0 + i] = -1;
        if (lane == 0) {  // null in a call without rows alone
            if (p.count) p.count[b] = count;
            if (p.next) p.next[b] = next;
        }
    }
}

hipError_t launch_tree_accept(const AcceptParams& p, hipStream_t st) {
    if (p.batch.B == 0) return hipSuccess;
    hipLaunchKernelGGL(tree_accept_kernel, dim3(min(p.batch.B, 1u << 20)), dim3(64), 0, st, p);
    return hipGetLastError();
}

// New token keep[i] of a sequence becomes its new token i.  Within a head, what a step writes
// is read by none of the later ones, since keep[i] >= i: a step's tokens are all loaded before
// any is stored.  A block a sequence, so that its length may be written where it was read.
// A token of a head is CB / 16 pieces of K codes, CB / 4 of V codes (of four tokens' words each
// the bytes of one) and one of its scales.  Few bytes, each behind its page number: 64 requests with
// some nodes kept of 64 (8 heads of 128, 8 bit) 9 us, one 2.3.
constexpr int kKeepThreads = 1024, kKeepList = 256;
template <int FMT, int D>
__global__ void __launch_bounds__(kKeepThreads) kv_keep_kernel(KeepParams p) {
    constexpr uint32_t CB = FMT == QUANT_Q8_0 ? D : D / 2, NB = D / 32;
    constexpr uint32_t KP = CB / 16, VP = CB / 4, PIECES = KP + VP + 1, PAIRS = kKeepThreads / PIECES;
    __shared__ uint32_t src_page[kKeepList], src_slot[kKeepList], dst_page[kKeepList], dst_slot[kKeepList];
    const uint32_t piece = threadIdx.x % PIECES, pair = threadIdx.x / PIECES;
    for (uint32_t b = blockIdx.x; b < p.batch.B; b += gridDim.x) {
        const NewRows s = rows_if_any(p.batch, b);
        const int len = max(p.batch.kv_len[b], 0), count = s.n ? min(max(p.count[b], 0), s.n) : 0;
        __syncthreads();  // the length is read
        if (threadIdx.x == 0 && p.len_out) p.len_out[b] = s.n ? max(s.first + count, 0) : len;
        for (int base = 0; base < count; base += kKeepList) {
            const uint32_t tokens = (uint32_t)min(count - base, kKeepList);
            __syncthreads();
            if (threadIdx.x < tokens) {
                const int i = base + (int)threadIdx.x, from = p.keep[s.q0 + i];
                const uint32_t none = 0xffffffffu;
                auto place = [&](int node, uint32_t& page, uint32_t& slot) {
                    const int at = s.first + node;
                    const uint32_t pi = (uint32_t)at >> p.geom.log2_page;
                    page = at >= 0 && pi < p.batch.table_pages ? (uint32_t)p.batch.table[(size_t)b * p.batch.table_stride + pi] : none;
                    if (page >= p.geom.num_pages) page = none;
                    slot = (uint32_t)at & ((1u << p.geom.log2_page) - 1);
                };
                uint32_t sp = none, ss = 0, dp = none, ds = 0;
                if (from >= 0 && from < s.n && from != i) {
                    place(from, sp, ss);
                    place(i, dp, ds);
                }
                if (sp == none) dp = none;
                src_page[threadIdx.x] = sp;
                src_slot[threadIdx.x] = ss;
                dst_page[threadIdx.x] = dp;
                dst_slot[threadIdx.x] = ds;
            }
            __syncthreads();
            const uint64_t pairs = (uint64_t)tokens * p.geom.Hkv;
            for (uint64_t x0 = 0; x0 < pairs; x0 += PAIRS) {
                const uint64_t x = x0 + pair;
                const uint32_t hk = (uint32_t)(x / tokens), t = (uint32_t)(x % tokens);
                const bool live = pair < PAIRS && x < pairs && dst_page[t] != 0xffffffffu;
                uint8_t *src = nullptr, *dst = nullptr;
                uint32_t ss = 0, ds = 0;
                u4_t v{};
                if (live) {
                    src = p.geom.pages + ((size_t)src_page[t] * p.geom.Hkv + hk) * p.geom.head_bytes;
                    dst = p.geom.pages + ((size_t)dst_page[t] * p.geom.Hkv + hk) * p.geom.head_bytes;
                    ss = src_slot[t];
                    ds = dst_slot[t];
                    if (piece < KP) {
                        v = *reinterpret_cast<const u4_t*>(src + ss * CB + 16 * piece);
                    } else if (piece < KP + VP) {
                        v = *reinterpret_cast<const u4_t*>(src + p.geom.v_off + (ss >> 2) * (4 * CB) + 16 * (piece - KP)) >> (8 * (ss & 3));
                    } else {
                        uint32_t h[8] = {};
#pragma unroll
                        for (uint32_t j = 0; j < NB; j++) {
                            h[j] = *reinterpret_cast<const uint16_t*>(src + p.geom.ks_off + (ss * NB + j) * 2);
                            h[4 + j] = *reinterpret_cast<const uint16_t*>(src + p.geom.vs_off + (((ss >> 2) * NB + j) * 4 + (ss & 3)) * 2);
                        }
                        v = u4_t{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
                    }
                }
                __syncthreads();
                if (!live) continue;
                if (piece < KP) {
                    *reinterpret_cast<u4_t*>(dst + ds * CB + 16 * piece) = v;
                } else if (piece < KP + VP) {
                    uint8_t* o = dst + p.geom.v_off + (ds >> 2) * (4 * CB) + 16 * (piece - KP) + (ds & 3);
                    o[0] = (uint8_t)v.x;
                    o[4] = (uint8_t)v.y;
                    o[8] = (uint8_t)v.z;
                    o[12] = (uint8_t)v.w;
                } else {
                    const uint32_t h[8] = {v.x, v.x >> 16, v.y, v.y >> 16, v.z, v.z >> 16, v.w, v.w >> 16};
#pragma unroll
                    for (uint32_t j = 0; j < NB; j++) {
                        *reinterpret_cast<uint16_t*>(dst + p.geom.ks_off + (ds * NB + j) * 2) = (uint16_t)h[j];
                        *reinterpret_cast<uint16_t*>(dst + p.geom.vs_off + (((ds >> 2) * NB + j) * 4 + (ds & 3)) * 2) = (uint16_t)h[4 + j];
                    }
                }
            }
        }
    }
}

hipError_t launch_kv_keep(const KeepParams& p, hipStream_t st) {
    if (p.batch.B == 0) return hipSuccess;
    const dim3 grid(min(p.batch.B, 1u << 20)), block(kKeepThreads);
    if (p.format == QUANT_Q8_0) {
        if (p.D == 64) hipLaunchKernelGGL((kv_keep_kernel<QUANT_Q8_0, 64>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((kv_keep_kernel<QUANT_Q8_0, 128>), grid, block, 0, st, p);
    } else {
        if (p.D == 64) hipLaunchKernelGGL((kv_keep_kernel<QUANT_Q4_0, 64>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((kv_keep_kernel<QUANT_Q4_0, 128>), grid, block, 0, st, p);
    }
    return hipGetLastError();
}

}  // namespace qr
