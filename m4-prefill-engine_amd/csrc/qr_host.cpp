// qr_host.cpp -- the bridge's host-only logic: argument validation and the
// host-range probe.  No HIP calls, so a sanitizer build of the host code can
// compile it alone (tests/c/sanitize_host.cpp).
#include "qr_host.h"

#include <sys/uio.h>
#include <unistd.h>

#include <cerrno>
#include <cmath>
#include <cstring>

namespace qr {

// Whether every page of the host range [p, p + bytes) can be read (and, for
// outputs, written) by this process.  The reference wraps host memory with
// newBufferWithBytesNoCopy and returns -5 when that fails for a range running
// into an unmapped or protected page (tests/redteam_bridge.py:178-221); here
// the staging copy would fault instead, so the range is probed first, one
// byte per page, by system calls that report EFAULT rather than raise a
// signal: process_vm_readv / process_vm_writev on this process, or where
// those are not permitted (seccomp), a pipe -- write(2) from the page reads
// it, read(2) of that byte back into the page writes it unchanged.  When no
// probe is possible the range counts as inaccessible (fail closed: -5).
static bool page_ok_pipe(int fds[2], const void* q, bool write) {
    char sink;
    if (::write(fds[1], q, 1) != 1) return false;  // EFAULT: not readable
    if (write) {
        if (::read(fds[0], const_cast<void*>(q), 1) == 1) return true;
        (void)::read(fds[0], &sink, 1);  // not writable: drain the byte
        return false;
    }
    return ::read(fds[0], &sink, 1) == 1;
}

bool host_range_ok(const void* p, size_t bytes, bool write) {
    if (bytes == 0) return true;
    const uintptr_t pg = (uintptr_t)sysconf(_SC_PAGESIZE);
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), e = a + bytes - 1;
    constexpr int kBatch = 512;
    char tmp[kBatch];
    struct iovec loc[kBatch], rem[kBatch];
    // probe addresses: a, then the first byte of every later page up to e
    uintptr_t q = a;
    bool more = true;
    while (more) {
        int n = 0;
        for (; n < kBatch && more; n++) {
            loc[n] = {tmp + n, 1};
            rem[n] = {reinterpret_cast<void*>(q), 1};
            const uintptr_t next = (q / pg + 1) * pg;
            more = next > q && next <= e;
            q = next;
        }
        errno = 0;
        ssize_t got = process_vm_readv(getpid(), loc, n, rem, n, 0);
        if (got >= 0 || errno == EFAULT) {
            if (got != n) return false;
            if (write) {
                got = process_vm_writev(getpid(), loc, n, rem, n, 0);  // the bytes just read, unchanged
                if (got != n) return false;
            }
            continue;
        }
        // process_vm_* not permitted: probe this batch's pages through a pipe
        int fds[2];
        if (pipe(fds) != 0) return false;
        bool ok = true;
        for (int i = 0; i < n && ok; i++) ok = page_ok_pipe(fds, rem[i].iov_base, write);
        close(fds[0]);
        close(fds[1]);
        if (!ok) return false;
    }
    return true;
}


// Formats m4_bridge_dispatch_gemm accepts (m4_mlx_bridge.mm:28-35, 211), and
// the wider set the kernel-name entry points accept: every format with a
// kernel here, i.e. also Q8_0 weights (6), PRISM_Q2_0 (7) and MLX g64 (8).
bool is_projection_format(int f) { return f >= 0 && f < 6; }
bool has_kernels(int f) { return f >= 0 && f <= qr::QUANT_MLX_4BIT_G64; }

// core/bridge/m4_mlx_bridge.mm:204-230, minus the init check.  `ext` widens
// the format range to every format with kernels (PRISM_Q2_0 needs K % 128).
int validate(const void* X, size_t Xb, const void* W, size_t Wb, const void* Y, size_t Yb, int format,
             uint32_t M, uint32_t K, uint32_t N, bool ext) {
    if (!X || !W || !Y) return -2;
    if ((reinterpret_cast<uintptr_t>(X) % 2) || (reinterpret_cast<uintptr_t>(Y) % 2)) return -2;
    if (!(ext ? has_kernels(format) : is_projection_format(format))) return -3;
    if (M == 0 || K == 0 || N == 0) return -4;
    if (K % 32) return -4;
    if ((format == 2 || format == 4 || format == 5) && (K % 256)) return -4;
    if (format == 7 && (K % 128)) return -4;
    if (format == qr::QUANT_MLX_4BIT_G64 && (K % 64)) return -4;
    if (Xb < (size_t)M * K * 2 || Yb < (size_t)M * N * 2 || Wb < qr::kernel_weight_bytes(format, K, N))
        return -2;
    return 0;
}

// ---- serving: paged cache, batches, rows, rotary tables ----

size_t kv_cache_bytes(int format, uint32_t num_pages, uint32_t P, uint32_t Hkv, uint32_t D) {
    if (format != QUANT_Q8_0 && format != QUANT_Q4_0) return 0;
    if (P < 16 || P > 256 || (P & (P - 1)) || (D != 64 && D != 128)) return 0;
    if (num_pages == 0 || num_pages > 0x7fffffffu || Hkv == 0 || Hkv > 0xffffu) return 0;
    const size_t row = (size_t)D / 32 * get_quant_info(static_cast<QuantFormat>(format)).block_bytes;
    return 2 * row * P * Hkv * num_pages;  // at most 2^9 * 2^8 * 2^16 * 2^31 bytes
}

namespace {

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int check_cache(const m4_kv_cache_t* c) {
    if (!c) return -2;
    if (c->format != QUANT_Q8_0 && c->format != QUANT_Q4_0) return -3;
    const size_t need = kv_cache_bytes(c->format, c->num_pages, c->page_size, c->Hkv, c->D);
    if (need == 0) return -4;
    if (!c->pages || misaligned(c->pages, 16) || c->bytes < need) return -2;
    return 0;
}

// Rows of a call: what a launch of one thread per eight dims of a row can number.
constexpr uint32_t kMaxRows = 1u << 26;

// B = 0 or T = 0: no rows, and no pointers needed.  Positions are 32-bit, with
// room for a stretch of pages on top.
int check_batch(const m4_kv_cache_t* c, const m4_kv_batch_t* b, uint32_t T, bool* empty) {
    if (!b) return -2;
    if (b->B > 0x7fffffffu || T > kMaxRows) return -4;
    *empty = b->B == 0 || T == 0;
    if (*empty) return 0;
    if (!b->q_start || !b->kv_len || !b->page_table) return -2;
    if (misaligned(b->q_start, 4) || misaligned(b->kv_len, 4) || misaligned(b->page_table, 4)) return -2;
    if (b->table_pages == 0 || (b->B > 1 && b->table_stride < b->table_pages)) return -4;
    if ((uint64_t)b->table_pages * c->page_size > 0x7fff0000u) return -4;
    return 0;
}

int check_rows(const m4_rows_t* r, uint32_t T, uint32_t heads, uint32_t D, bool out) {
    if (!r || !r->ptr || misaligned(r->ptr, 16)) return -2;
    const int64_t ts = r->token_stride, hs = r->head_stride;
    if (ts < 0 || hs < 0 || ts % 8 || hs % 8) return -4;
    if (out) {
        const bool t_inner = T > 1 && (heads <= 1 || ts < hs);
        const __int128 inner = t_inner ? ts : hs, outer = t_inner ? hs : ts;
        const uint32_t n_in = t_inner ? T : heads, n_out = t_inner ? heads : T;
        if (n_in > 1 && inner < D) return -4;
        if (n_out > 1 && outer < (n_in > 1 ? inner * (n_in - 1) : 0) + D) return -4;
    }
    const __int128 last = (__int128)(T - 1) * ts + (__int128)(heads - 1) * hs + D;
    if ((__int128)r->bytes < last * 2) return -2;
    return 0;
}

int check_rope(const m4_rope_axes_t* r, uint32_t D) {
    if (r->pairs == 0 || r->pairs > M4_ROPE_MAX_PAIRS || r->pairs % 8 || 2 * r->pairs > D) return -4;
    if (r->axes == 0 || r->axes > 256) return -4;
    if (!r->table || misaligned(r->table, 16) || r->table_bytes < (size_t)r->pairs * M4_ROPE_PAIR_BYTES) return -2;
    return 0;
}

// A stride of 0 is one row for all axes, as text has.
int check_positions(const int32_t* positions, uint32_t stride, uint32_t axes, uint32_t T) {
    if (misaligned(positions, 4)) return -2;
    return axes > 1 && stride != 0 && stride < T ? -4 : 0;
}

}  // namespace

// Frequencies in turns, as 64-bit fractions of one: whole turns per position
// drop out because positions are whole.  Double keeps a turn to 2^-23 at the
// farthest position.
int rope_axes_table(const double* inv_freq, const uint8_t* pair_axis, uint32_t pairs, uint32_t axes, void* table) {
    if (!inv_freq || !pair_axis || !table) return -2;
    if (pairs == 0 || pairs > M4_ROPE_MAX_PAIRS || pairs % 8 || axes == 0 || axes > 256) return -4;
    for (uint32_t i = 0; i < pairs; i++)
        if (pair_axis[i] >= axes || !std::isfinite(inv_freq[i])) return -4;
    uint8_t* out = static_cast<uint8_t*>(table);
    for (uint32_t i = 0; i < pairs; i++) {
        const double turns = inv_freq[i] * 0.15915494309189533576888376337251;
        const double part = turns - std::floor(turns);  // 1 for a tiny negative frequency: no turn
        const uint64_t turn = part < 1.0 ? (uint64_t)(part * 18446744073709551616.0) : 0;
        const uint32_t axis = pair_axis[i];
        std::memcpy(out + 8 * i, &turn, 8);
        std::memcpy(out + 8 * pairs + 4 * i, &axis, 4);
    }
    return 0;
}

int validate_rope_axes(const m4_rope_axes_t* rope, const int32_t* positions, uint32_t stride, const m4_rows_t* X,
                       const m4_rows_t* Y, uint32_t T, uint32_t H, uint32_t D, bool* empty) {
    *empty = false;
    if (!rope || !X || !Y) return -2;
    if (H == 0 || H > 0xffffu || D == 0 || D % 8 || D > 256 || T > kMaxRows) return -4;
    if (int rc = check_rope(rope, D)) return rc;
    if (T == 0) {
        *empty = true;
        return 0;
    }
    if (!positions) return -2;
    if (int rc = check_positions(positions, stride, rope->axes, T)) return rc;
    if (int rc = check_rows(X, T, H, D, false)) return rc;
    return check_rows(Y, T, H, D, true);
}

int validate_append(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* K, const m4_rows_t* V,
                    const m4_rope_axes_t* rope, const int32_t* positions, uint32_t stride, const m4_rows_t* Q,
                    const m4_rows_t* Q_out, uint32_t H, bool* empty) {
    *empty = false;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(cache, batch, T, empty)) return rc;
    if (Q && (!rope || !Q_out)) return -2;
    if (Q && (H == 0 || H > 0xffffu)) return -4;
    if (rope) {
        if (int rc = check_rope(rope, cache->D)) return rc;
        if (!positions && rope->axes > 1) return -2;
    }
    if (*empty) return 0;
    if (rope && positions)
        if (int rc = check_positions(positions, stride, rope->axes, T)) return rc;
    if (int rc = check_rows(K, T, cache->Hkv, cache->D, false)) return rc;
    if (int rc = check_rows(V, T, cache->Hkv, cache->D, false)) return rc;
    if (Q) {
        if (int rc = check_rows(Q, T, H, cache->D, false)) return rc;
        if (int rc = check_rows(Q_out, T, H, cache->D, true)) return rc;
    }
    return 0;
}

int validate_read(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* K, const m4_rows_t* V,
                  bool* empty) {
    *empty = false;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(cache, batch, T, empty)) return rc;
    if (*empty) return 0;
    if (int rc = check_rows(K, T, cache->Hkv, cache->D, true)) return rc;
    return check_rows(V, T, cache->Hkv, cache->D, true);
}

int validate_attn(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rows_t* Q, const m4_rows_t* O,
                  uint32_t H, float scale, const void* ws, bool* empty) {
    *empty = false;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(cache, batch, T, empty)) return rc;
    if (H == 0 || H > 0xffffu || H % cache->Hkv || !std::isfinite(scale)) return -4;
    if (*empty) return 0;
    if ((uint64_t)T * (H / cache->Hkv) > 0x7fffffffu) return -4;  // rows of a KV head are counted in 32 bits
    if (int rc = check_rows(Q, T, H, cache->D, false)) return rc;
    if (int rc = check_rows(O, T, H, cache->D, true)) return rc;
    if (!ws || misaligned(ws, 16)) return -2;
    return 0;
}

int validate_layer(const m4_kv_cache_t* cache, const m4_kv_batch_t* batch, uint32_t T, const m4_rope_axes_t* rope,
                   const int32_t* positions, uint32_t stride, int format, uint32_t dm, uint32_t Hq, uint32_t Nm,
                   float scale, bool norms, int norm_type, bool* empty) {
    *empty = false;
    if (!cache || !batch) return -2;
    if (!has_kernels(format) || (norms && norm_type != 1 && norm_type != 2)) return -3;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(cache, batch, T, empty)) return rc;
    if (dm == 0 || Nm == 0 || Hq == 0 || Hq > 0xffffu || Hq % cache->Hkv || !std::isfinite(scale)) return -4;
    const uint64_t HQ = (uint64_t)Hq * cache->D;
    const uint32_t bs = get_quant_info(static_cast<QuantFormat>(format)).block_size;
    if (dm % bs || HQ % bs || Nm % bs || dm % 32 || Nm % 32) return -4;
    if (rope) {
        if (int rc = check_rope(rope, cache->D)) return rc;
        if (!positions && rope->axes > 1) return -2;
    }
    if (*empty) return 0;
    if (rope && positions)
        if (int rc = check_positions(positions, stride, rope->axes, T)) return rc;
    if ((uint64_t)T * (Hq / cache->Hkv) > 0x7fffffffu) return -4;
    return 0;
}

}  // namespace qr
