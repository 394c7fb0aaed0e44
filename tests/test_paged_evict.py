"""Bounded caches -- the attention weight that each cached key has received, and eviction of the lightest -- against plain
implementations in 64 bits, and their refusals."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import m4_bridge
import paged_reference as ref
from paged_reference import Q8_0
from test_paged import FORMATS, Setup, close, dev, half, say
from test_paged_tree import attend, host, i32, launched, lib, rows_of, set_, token_bytes  # noqa: F401

gpu = pytest.mark.gpu
# what is expected of the lengths chooses the kernels; the results hold for any
EXPECTED = {"rows": {"max_new": 1, "max_kv": 1}, "chunks": {"max_new": 10 ** 6, "max_kv": 400}, "both": {"max_new": 2 ** 20, "max_kv": 10 ** 4},
            "wide": {"max_new": 10 ** 6, "max_kv": 2 * 10 ** 6},
            "alone": {"max_new": 200, "max_kv": 500}, "wide alone": {"max_new": 200, "max_kv": 10 ** 6}}


# ---- weights received -----------------------------------------------------------------------------------------------

def causal(first, n, L, window):
    p, j = first + np.arange(n)[:, None], np.arange(L)[None, :]
    return (j <= p) & (j > p - window) if window else j <= p


def weights(q, k, lse, seen, scale):
    """Sum over rows and query heads [Hkv, L] of exp(scale q . k - lse) in float64, and a bound on what a kernel may be off:
    scores by (D + 8) 2^-24 of the sum of |q k|, exponents by 2^-22 of them and of lse, exponentials 2^-21, the sum
    (rows + 8) 2^-24."""
    H, n, D = q.shape
    Hkv, L, _ = k.shape
    w, b = np.zeros((Hkv, L)), np.zeros((Hkv, L))
    for h in range(H):
        kk, qq = k[h // (H // Hkv)].astype(np.float64), q[h].astype(np.float64)
        z = np.where(np.isfinite(lse[h]), lse[h], 0).astype(np.float64)[:, None]
        s = qq @ kk.T * scale
        x = np.where(seen, np.exp(s - z), 0)
        e = np.abs(qq) @ np.abs(kk).T * abs(scale) * ((D + 8) * 2.0 ** -24 + 2.0 ** -22) + np.abs(z) * 2.0 ** -22 + 2.0 ** -21
        w[h // (H // Hkv)] += x.sum(0)
        b[h // (H // Hkv)] += (x * e).sum(0)
    return w, b + (n * H // Hkv + 8) * 2.0 ** -24 * w


def weighed(s, sums, q, lse, lens, starts, window, scale, table=None):
    """What sums [num_pages, Hkv, P] become (float64), and the bound; entries that are not touched have none."""
    want, bound = sums.astype(np.float64), np.zeros(sums.shape)
    table = s.table if table is None else table
    for b in range(len(lens)):
        a, n, first = rows_of(starts, lens, b, q.shape[1])
        L = min(max(first + n, 0), table.shape[1] * s.P)
        if n == 0 or L == 0:
            continue
        k = np.zeros((s.Hkv, L, s.D), np.float16)
        m = min(L, s.k[b].shape[1])
        k[:, :m] = s.k[b][:, :m]
        w, e = weights(q[:, a:a + n], k, lse[:, a:a + n], causal(first, n, L, window), scale)
        for p in range(L):
            page = table[b, p // s.P]
            if 0 <= page < s.num_pages:
                old = sums[page, :, p % s.P].astype(np.float64) if p < first else 0
                want[page, :, p % s.P] = old + w[:, p]
                bound[page, :, p % s.P] = e[:, p] + 2.0 ** -24 * want[page, :, p % s.P]
    return want, bound


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,H,Hkv,D,P,window,kernels", [
    ([1], [1], 1, 1, 64, 16, 0, "rows"),
    ([1000], [1], 32, 8, 128, 16, 0, "rows"),
    ([700, 3, 0, 65, 129], [1, 1, 0, 5, 3], 8, 2, 64, 32, 0, "rows"),
    ([700, 3, 0, 65, 129], [1, 1, 0, 5, 3], 8, 2, 64, 32, 7, "rows"),
    ([260, 131], [61, 100], 6, 2, 128, 64, 0, "rows"),
    ([260, 131], [61, 100], 6, 2, 128, 64, 0, "chunks"),
    ([260, 131, 700], [61, 100, 513], 6, 2, 128, 256, 50, "chunks"),
    ([64], [64], 4, 4, 64, 16, 0, "chunks"),
    ([1200, 40], [1100, 1], 5, 1, 128, 16, 0, "both"),                 # more rows than are held at once
    ([1200, 40, 90], [1100, 1, 90], 5, 1, 64, 16, 300, "both"),
])
def test_weigh(bridge, fmt, lens, new, H, Hkv, D, P, window, kernels):
    import torch

    s = Setup(fmt, lens, new, Hkv, D, P, seed=len(lens) * 7 + D)
    q, scale = half(s.rng, H, s.T, D), D ** -0.5
    lse = np.concatenate([attend(q[:, a:a + n], k, v, causal(L - n, n, L, window), scale)[2]
                          for a, n, L, k, v in zip(s.q_start, s.new, s.lens, s.k, s.v)], 1).astype(np.float32)
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32) * 3
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **EXPECTED[kernels])
    cache, got, again = s.cache(), dev(sums), dev(sums)
    say("weigh", fmt, lens, new, H, Hkv, D, P, window, kernels)
    bridge.kv_cache_weigh(cache, batch, dev(q), dev(lse), got, scale, window=window)
    # again: the same bits, from token-major rows and an lse of other strides
    bridge.kv_cache_weigh(cache, batch, dev(q.transpose(1, 0, 2)), dev(lse.T).T, again, scale, window=window, token_major=True)
    bridge.synchronize()
    assert torch.equal(got, again)
    close(got.cpu().numpy(), *weighed(s, sums, q, lse, lens, s.q_start, window, scale), "sums")
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,H,Hkv,D,P,window", [
    ([1], [1], 1, 1, 64, 16, 0),
    ([260, 131], [61, 100], 6, 2, 128, 64, 0),
    ([260, 131, 700], [61, 100, 513], 6, 2, 128, 256, 50),
    ([1200, 40], [1100, 1], 5, 1, 128, 16, 0),
    ([1200, 40, 90], [1100, 1, 90], 5, 1, 64, 16, 300),
    ([1500, 0, 513, 512], [3, 0, 513, 31], 8, 2, 64, 32, 0),
    ([1100, 1029], [200, 1029], 3, 1, 128, 16, 600),
])
def test_weigh_as_if_long(bridge, fmt, lens, new, H, Hkv, D, P, window):
    test_weigh(bridge, fmt, lens, new, H, Hkv, D, P, window, "wide")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kernels", ["alone", "wide alone"])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("lens,new,H,Hkv,D,P", [
    ([700, 40, 90, 300], [600, 1, 3, 300], 8, 2, 64, 16),    # more rows than three could have, so the fourth is held to be long
    ([900, 333, 0, 5], [700, 1, 0, 5], 5, 1, 128, 32),
])
def test_weigh_where_all_seem_long(bridge, fmt, kernels, window, lens, new, H, Hkv, D, P):
    test_weigh(bridge, fmt, lens, new, H, Hkv, D, P, window, kernels)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kernels", ["rows", "chunks", "both", "wide"])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 0.3])
def test_weigh_out_of_range(bridge, fmt, kernels, scale):
    """Starts outside the rows, lengths past the table, more rows than keys, pages that are not there, rows that see
    nothing (lse -infinity), garbage in unwritten places."""
    P, H, D = 16, 16, 64
    s = Setup(fmt, [100, 60, 64, 5], [40, 20, 30, 9], 2, D, P, seed=9)
    starts, lens = i32(-3, 40, 60, 90, 10 ** 9), i32(100, 60, 70, 5 + 10 ** 9 - s.T)
    table = s.table[:, :6].copy()  # 96 keys
    table[0, 2], table[1, 3] = 10 ** 9, -1
    q = half(s.rng, H, s.T, D)
    q[:, 95:] = 0
    sums = s.rng.random((s.num_pages, 2, P)).astype(np.float32)
    lse = s.rng.standard_normal((H, s.T)).astype(np.float32) + 4
    lse[:, 90:94] = -np.inf  # before position 0
    batch = m4_bridge.KVBatch(dev(starts), dev(lens), dev(table), **EXPECTED[kernels])
    got = dev(sums)
    say("weigh out of range", fmt, kernels, scale)
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), got, scale)
    bridge.synchronize()
    close(got.cpu().numpy(), *weighed(s, sums, q, lse, lens, starts, 0, scale, table), "sums")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("B,H,Hkv,P,pages,window", [
    (70, 6, 2, 16, 0, 0),               # more sequences than a wave has lanes
    (150, 7, 1, 32, 0, 33),
    (16, 16, 16, 256, 2 ** 21, 0),      # a table for so many keys that two tiles are counted as one
    (16, 16, 16, 256, 2 ** 21, 90),
])
def test_weigh_many_sequences(bridge, fmt, B, H, Hkv, P, pages, window):
    import torch

    D = 64
    lens = [(37 * b) % 401 + (b % 5 > 0) if b % 7 else 0 for b in range(B)]
    new = [min(n, b % 4) for b, n in enumerate(lens)]
    s = Setup(fmt, lens, new, Hkv, D, P, seed=B + P)
    table = dev(s.table)
    if pages:
        table = torch.full((B, pages), -1, dtype=torch.int32, device="cuda")
        table[:, :s.table.shape[1]] = dev(s.table)
    q = half(s.rng, H, s.T, D)
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32)
    lse = s.rng.standard_normal((H, s.T)).astype(np.float32) + 4
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), table, max_new=max(new), max_kv=max(lens))
    got = dev(sums)
    say("weigh many sequences", fmt, B, H, Hkv, P, pages, window)
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), got, 0.125, window=window)
    bridge.synchronize()
    close(got.cpu().numpy(), *weighed(s, sums, q, lse, lens, s.q_start, window, 0.125), "sums")


@gpu
@pytest.mark.parametrize("kernels", ["rows", "chunks", "wide"])
@pytest.mark.parametrize("G", [1, 2, 3, 7, 12, 16, 17, 31, 32, 33, 40, 64, 71])
@pytest.mark.parametrize("window", [0, 40])
def test_weigh_groups(bridge, kernels, G, window):
    """Query heads that share a KV head, any number: what belongs to no row weighs nothing, though its values are."""
    D, P, Hkv, lens, new = 128, 32, 2, [170, 33, 5, 64], [70, 20, 5, 1]
    s = Setup(Q8_0, lens, new, Hkv, D, P, seed=G)
    q = half(s.rng, G * Hkv, s.T, D)
    q[:, 60] = np.inf   # a row of the first sequence: NaN or infinity for the keys that it sees, and none else
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32)
    lse = s.rng.standard_normal((G * Hkv, s.T)).astype(np.float32) + 4
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **EXPECTED[kernels])
    got, clean = dev(sums), dev(sums)
    say("weigh groups", kernels, G, window)
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), got, 0.09, window=window)
    q[:, 60] = 0.5
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), clean, 0.09, window=window)
    bridge.synchronize()
    want, bound = weighed(s, sums, q, lse, lens, s.q_start, window, 0.09)
    close(clean.cpu().numpy(), want, bound, "sums")
    seen = np.zeros(sums.shape, bool)  # by that row: token 60 of positions 100 .. 169
    for k in range(max(0, 160 - window + 1) if window else 0, 161):
        seen[s.table[0, k // P], :, k % P] = True
    got = got.cpu().numpy()
    assert np.isfinite(got[~seen]).all() and (got[~seen] == clean.cpu().numpy()[~seen]).all()


@gpu
@pytest.mark.parametrize("kernels", ["rows", "chunks", "wide"])
@pytest.mark.parametrize("window", [0, 25])
def test_rows_without_a_sum_weigh_nothing(bridge, kernels, window):
    """lse -infinity, whether or not the row sees keys; +infinity too."""
    lens, new, H, Hkv, D, P = [200, 60], [70, 60], 8, 2, 64, 16
    s = Setup(Q8_0, lens, new, Hkv, D, P, seed=31)
    q = half(s.rng, H, s.T, D)
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32)
    lse = s.rng.standard_normal((H, s.T)).astype(np.float32) + 4
    none = s.rng.random((H, s.T)) < 0.4
    given = np.where(none, np.where(s.rng.random((H, s.T)) < 0.8, -np.inf, np.inf), lse).astype(np.float32)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **EXPECTED[kernels])
    got = dev(sums)
    say("weigh without a sum", kernels, window)
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(given), got, 0.1, window=window)
    bridge.synchronize()
    want, bound = weighed(s, sums, q, np.where(none, np.float32(1e5), lse), lens, s.q_start, window, 0.1)
    close(got.cpu().numpy(), want, bound, "sums")


@gpu
@pytest.mark.parametrize("kernels", ["rows", "chunks", "both", "wide", "wide alone"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 60, 2 ** 31, 2 ** 32 - 1])
def test_weigh_with_the_widest_windows(bridge, kernels, window):
    """Windows that reach past every key, with which tokens behind the first still see what is before them; and a length
    whose positions are as far as the window."""
    import torch

    lens, new, H, Hkv, D, P = [64, 200, 80, 160], [64, 70, 1, 130], 8, 2, 64, 16
    s = Setup(Q8_0, lens, new, Hkv, D, P, seed=7)
    q = half(s.rng, H, s.T, D)
    lse = s.rng.standard_normal((H, s.T)).astype(np.float32) + 4
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32)
    for far in (False, True):
        length = i32(64, 200, 2 ** 31 - 1 if far else 80, 160)  # keys past the table are not there
        batch = m4_bridge.KVBatch(dev(s.q_start), dev(length), dev(s.table), **EXPECTED[kernels])
        got, without = dev(sums), dev(sums)
        say("weigh with a window of", window, kernels, far)
        bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), got, 0.125, window=window)
        bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), without, 0.125)
        bridge.synchronize()
        close(got.cpu().numpy(), *weighed(s, sums, q, lse, length, s.q_start, window, 0.125), "sums")
        if not far or window >= 2 ** 31 - 1:
            assert torch.equal(got, without)  # the same terms in the same order


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kernels", ["rows", "chunks", "wide"])
@pytest.mark.parametrize("H", [8, 10, 66])
@pytest.mark.parametrize("window", [0, 25])
def test_rows_without_a_sum_weigh_nothing_whatever_they_hold(bridge, fmt, kernels, H, window):
    """Rows of a padded batch that nothing but their lse marks: NaN and infinities in them reach no key; nor do keys that
    are infinite (65504 in Q8_0) where no other row sees them."""
    import torch

    lens, new, Hkv, D, P = [200, 60, 300, 90, 33], [70, 60, 5, 1, 33], 2, 64, 16
    s = Setup(fmt, lens, new, Hkv, D, P, seed=32)
    k, v = half(s.rng, 2, 64), half(s.rng, 2, 64)
    k[:, 3] = 65504
    (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
    for p in (0, 17, 32):  # of the last sequence, none of whose rows has a sum
        s.pages.write(s.table[4, p // P], p % P, kq, kd, vq, vd)
    q = half(s.rng, H, s.T, D)
    sums = s.rng.random((s.num_pages, Hkv, P)).astype(np.float32)
    lse = s.rng.standard_normal((H, s.T)).astype(np.float32) + 4
    none = s.rng.random((H, s.T)) < 0.3
    none[:, 69:75] = True       # the last row of a sequence and the first of the next
    none[:, s.q_start[3]:] = True
    lse[none] = -np.inf
    odd = q.copy()
    odd[none] = np.array([np.nan, np.inf, -np.inf, 65504], np.float16)[s.rng.integers(0, 4, (int(none.sum()), D))]
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **EXPECTED[kernels])
    got, clean = dev(sums), dev(sums)
    say("weigh rows without a sum that hold anything", fmt, kernels, H, window)
    bridge.kv_cache_weigh(s.cache(), batch, dev(odd), dev(lse), got, 0.1, window=window)
    q[none] = 0
    bridge.kv_cache_weigh(s.cache(), batch, dev(q), dev(lse), clean, 0.1, window=window)
    bridge.synchronize()
    assert torch.equal(got, clean)
    s.k[4] = np.zeros_like(s.k[4])
    want, bound = weighed(s, sums, q, np.where(none, np.float32(1e5), lse), lens, s.q_start, window, 0.1)
    close(got.cpu().numpy(), want, bound, "sums")


@gpu
def test_pages_past_4_gib(bridge):
    """The same bits from pages that lie past 4 GiB of a cache as from its first ones."""
    import torch

    lens, new, H, Hkv, D, P, budget = [700, 90, 333], [40, 9, 64], 16, 8, 128, 256, 128
    s = Bounded(Q8_0, lens, new, Hkv, D, P, seed=77)
    s.grow(budget)
    few, pages = s.cache(), dev(s.pages.raw)
    far = (1 << 32) // (few.pages.numel() // s.num_pages) + 7
    many = m4_bridge.PagedKVCache(Q8_0, far + s.num_pages, P, Hkv, D)
    many.pages.view(far + s.num_pages, -1)[far:] = pages.view(s.num_pages, -1)
    q, parents = dev(half(s.rng, H, s.T, D)), dev(np.concatenate([np.arange(n, dtype=np.int32) - 1 for n in new]))
    keep = dev(np.concatenate([np.minimum(2 * np.arange(n), n).astype(np.int32) for n in new]))
    count, results = dev(np.array([n // 2 for n in new], np.int32)), []
    for cache, at in ((few, 0), (many, far)):
        batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table + at), max(new), max(lens))
        tree, O, lse = m4_bridge.DraftTree.empty(s.T, max(new)), torch.empty_like(q), torch.empty(H, s.T, device="cuda")
        sums = torch.zeros(cache.num_pages, Hkv, P, device="cuda")
        kept, length = i32(*[0] * (len(lens) * Hkv * budget)).reshape(len(lens), Hkv, budget), dev(i32(*[0] * len(lens)))
        kept = dev(kept)
        say("pages past 4 GiB", at)
        bridge.draft_tree(batch, parents, tree)
        bridge.dispatch_paged_attn(cache, batch, q, O, 0.09, tree=tree, lse=lse)
        bridge.kv_cache_keep(cache, batch, keep, count)
        bridge.kv_cache_weigh(cache, batch, q, lse, sums, 0.09)
        bridge.kv_cache_evict(cache, batch, sums, dev(s.table_out + at), length, budget, sinks=3, recent=20, kept=kept)
        bridge.synchronize()
        raw = cache.pages.view(cache.num_pages, -1)[at:at + s.num_pages]
        results.append([x.clone().view(torch.uint8) for x in (O, lse, sums[at:at + s.num_pages].contiguous(), kept, length, raw.contiguous())])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_of_a_row_add_up_to_one(bridge, fmt):
    """Attention hands its lse over: what the rows of a call give all keys is 1 for each row and query head."""
    import torch

    H, new = 16, [3, 200, 40]
    s = Setup(fmt, [900, 300, 40], new, 2, 128, 32, seed=12)
    q, cache, batch = dev(half(s.rng, H, s.T, 128)), s.cache(), s.batch()
    O, lse = torch.empty_like(q), torch.empty(H, s.T, device="cuda")
    sums = torch.zeros(s.num_pages, 2, 32, device="cuda")
    bridge.dispatch_paged_attn(cache, batch, q, O, 0.09, lse=lse)
    bridge.kv_cache_weigh(cache, batch, q, lse, sums, 0.09)
    bridge.synchronize()
    got = sums.cpu().numpy()
    for b, n in enumerate(new):
        pages = s.table[b][:-(-s.lens[b] // 32)]
        total = got[pages].astype(np.float64).sum((0, 2))
        assert np.abs(total / (n * H // 2) - 1).max() <= 2.0 ** -16  # each weight to some 2^-20, lse to 2^-18


# ---- eviction -------------------------------------------------------------------------------------------------------

def chosen(w, there, budget, sinks, recent, length):
    """The places [m] of one head that are kept: w [n] float32, there [n] bool."""
    n = w.size
    key = np.where(np.isnan(w), np.inf, w.astype(np.float64))
    rank = np.where(np.isnan(w), 1, 0)  # NaN above infinity
    j = np.arange(n)
    rank = np.where((j < sinks) | (j >= length - recent), 2, rank)
    key = np.where(rank == 2, 0, key)
    order = np.lexsort((j, -key, -rank))
    order = order[there[order]]
    return np.sort(order[:budget])


def evicted(s, raw, sums, lens, table, table_out, budget, sinks, recent):
    """(pages, sums, kept, lengths) after an eviction."""
    pages, out = raw.copy(), sums.copy()
    kept, length = np.full((len(lens), s.Hkv, budget), -1, np.int32), np.zeros(len(lens), np.int32)
    at_slot = np.array([token_bytes(s.pages, x) for x in range(s.P)])
    for b, L in enumerate(lens):
        n = min(max(int(L), 0), table.shape[1] * s.P)
        at = table[b, np.arange(n) // s.P]
        there = (at >= 0) & (at < s.num_pages)
        for h in range(s.Hkv):
            w = np.where(there, sums[np.where(there, at, 0), h, np.arange(n) % s.P], 0)
            places = chosen(w, there, budget, sinks, recent, int(L))
            kept[b, h, :places.size] = places
            length[b] = places.size
            i = np.arange(places.size)
            to = table_out[b, i // s.P]
            i, p, to = (x[(to >= 0) & (to < s.num_pages)] for x in (i, places, to))
            pages[to[:, None], h, at_slot[i % s.P]] = raw[at[p][:, None], h, at_slot[p % s.P]]
            out[to, h, i % s.P] = sums[at[p], h, p % s.P]
    return pages, out, kept, length


class Bounded(Setup):
    """Setup with pages for `budget` tokens of each sequence behind its own, and sums of many kinds."""

    def grow(self, budget):
        spare, self.num_pages = self.num_pages, self.num_pages + len(self.lens) * -(-budget // self.P)
        more = ref.Pages(self.fmt, self.num_pages, self.P, self.Hkv, self.D, 0xEE)
        more.raw[:spare] = self.pages.raw
        self.pages = more
        self.table_out = spare + self.rng.permutation(self.num_pages - spare).reshape(len(self.lens), -1).astype(np.int32)
        r = self.rng
        sums = np.exp(r.standard_normal((self.num_pages, self.Hkv, self.P))).astype(np.float32)
        kind = r.random(sums.shape)
        sums[kind < 0.2] = 0
        sums[(kind > 0.2) & (kind < 0.3)] = -0.0
        sums[(kind > 0.3) & (kind < 0.4)] = 1.5
        for i, x in enumerate((np.nan, np.inf, -np.inf, -3, 1e-42, 3e38)):
            sums[(kind > 0.9 + i / 1000) & (kind < 0.9 + (i + 1) / 1000)] = x
        self.sums = sums


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,Hkv,D,P,budget,sinks,recent,max_kv", [
    ([1], 1, 64, 16, 1, 0, 0, 1),
    ([300, 0, 17, 65, 64], 3, 128, 16, 64, 4, 16, 300),
    ([300, 0, 17, 65, 64], 2, 64, 32, 63, 0, 0, 1),          # expected shorter than they are
    ([2000, 1025], 2, 64, 64, 777, 700, 77, 5000),           # nothing left to choose
    ([5000, 4096, 4097], 1, 64, 256, 1000, 1, 999, 5000),
    ([5000], 2, 128, 16, 4999, 0, 3, 0),
    ([90] * 70, 1, 64, 16, 40, 2, 9, 90),
    ([40000, 100], 1, 64, 256, 3001, 5, 100, 10 ** 9),       # longer than what is held
    ([40000, 100, 16384, 16385], 2, 64, 256, 3001, 5, 100, 40000),   # by several workgroups a head, or one
    ([41000, 30000], 1, 128, 16, 29000, 0, 0, 41000),                # of the second all but a few
    ([60000, 40000], 1, 64, 64, 35000, 7, 9, 41000),                 # the first longer than expected
    ([50000], 1, 64, 32, 60000, 0, 0, 50000),                        # all of them
])
def test_evict(bridge, fmt, lens, Hkv, D, P, budget, sinks, recent, max_kv):
    """Every byte of the pages, the sums, the places and the lengths."""
    import torch

    s = Bounded(fmt, lens, [0] * len(lens), Hkv, D, P, seed=len(lens) * 3 + budget)
    s.grow(budget)
    cache, sums = s.cache(), dev(s.sums)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), 0, max_kv)
    kept = torch.full((len(lens), Hkv, budget), -5, dtype=torch.int32, device="cuda")
    length = torch.full((len(lens),), -5, dtype=torch.int32, device="cuda")
    say("evict", fmt, lens[:5], Hkv, D, P, budget, sinks, recent)
    bridge.kv_cache_evict(cache, batch, sums, dev(s.table_out), length, budget, sinks=sinks, recent=recent, kept=kept)
    bridge.synchronize()
    pages, out, places, n = evicted(s, s.pages.raw, s.sums, lens, s.table, s.table_out, budget, sinks, recent)
    np.testing.assert_array_equal(length.cpu().numpy(), n)
    np.testing.assert_array_equal(kept.cpu().numpy(), places)
    got = cache.pages.cpu().numpy()
    tail = np.zeros(got.shape, bool)  # the places behind the last kept token of a group of four may hold anything
    for b, m in enumerate(n):
        for i in range(m, -(-m // 4) * 4):
            tail[s.table_out[b, i // P]][:, token_bytes(s.pages, i % P)] = True
    np.testing.assert_array_equal(np.where(tail, 0, got), np.where(tail, 0, pages))
    np.testing.assert_array_equal(sums.cpu().numpy().view(np.uint32), out.view(np.uint32))


@gpu
@pytest.mark.parametrize("lens,Hkv,D,P,budget,sinks,recent,max_kv", [
    ([512, 511, 510, 257, 256, 255, 64, 1, 0], 3, 64, 16, 100, 3, 40, 512),
    ([512, 513, 90, 2000, 4], 2, 64, 32, 300, 0, 1, 512),                       # some longer than expected
    ([500, 20], 1, 128, 64, 512, 0, 0, 500),                                    # all of them
    ([80 + b % 9 for b in range(130)], 2, 64, 16, 1, 0, 1, 89),
    ([(911 * b) % 1025 for b in range(140)], 8, 64, 64, 33, 2, 5, 1024),        # many, and longer
    ([(911 * b) % 1025 for b in range(140)] + [3000], 8, 64, 64, 700, 0, 0, 600),
])
def test_evict_of_short_sequences(bridge, lens, Hkv, D, P, budget, sinks, recent, max_kv):
    test_evict(bridge, Q8_0, lens, Hkv, D, P, budget, sinks, recent, max_kv)


@gpu
@pytest.mark.parametrize("value", ["zero", "few", "near", "nan"])
@pytest.mark.parametrize("n,max_kv", [(512, 512), (300, 300), (1000, 300), (512, 513)])
def test_evict_where_many_of_few_are_alike(bridge, value, n, max_kv):
    test_evict_where_many_are_alike(bridge, value, n, max_kv)


@gpu
@pytest.mark.parametrize("value", ["zero", "few", "near", "nan"])
@pytest.mark.parametrize("n,max_kv", [(9000, 9000), (45000, 45000), (45000, 1)])
def test_evict_where_many_are_alike(bridge, value, n, max_kv):
    """Sums that share all their bits, or most: the lowest places of the equal ones stay."""
    import torch

    budget = n // 3
    s = Bounded(Q8_0, [n], [0], 1, 64, 256, seed=n)
    s.grow(budget)
    r = s.rng
    s.sums[:] = {"zero": lambda k: 0.0, "few": lambda k: r.integers(0, 3, k).astype(np.float32),
                 "near": lambda k: (np.float32(1) + r.integers(0, 4000, k) * np.float32(2.0 ** -23)).astype(np.float32),
                 "nan": lambda k: np.where(r.random(k) < 0.5, np.float32("nan"), np.float32(1))}[value](s.sums.shape)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(i32(n)), dev(s.table), 0, max_kv)
    kept, length = torch.empty(1, 1, budget, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    say("alike", value, n, max_kv)
    bridge.kv_cache_evict(s.cache(), batch, dev(s.sums), dev(s.table_out), length, budget, sinks=3, recent=50, kept=kept)
    bridge.synchronize()
    w = s.sums[s.table[0][np.arange(n) // 256], 0, np.arange(n) % 256]
    np.testing.assert_array_equal(kept.cpu().numpy()[0, 0], chosen(w, np.ones(n, bool), budget, 3, 50, n))
    assert int(length[0]) == budget


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_evict_out_of_range(bridge, fmt):
    """Pages that are not there, of the old and of the new table, lengths past the table and below zero; sequences that
    share pages; nothing is copied over the old ones."""
    import torch

    s = Bounded(fmt, [200, 150, 160, 90], [0] * 4, 2, 64, 16, seed=3)
    s.grow(48)
    table, lens = s.table.copy(), i32(200, 2 ** 31 - 1, -4, 90)
    table[0, 3], table[0, 12] = -1, s.num_pages  # keys 48 .. 63, and 192 .. 199, among the last
    table[3, :3] = table[0, :3]                  # a common beginning
    out = s.table_out.copy()
    out[1, 1] = -1
    cache, sums = s.cache(), dev(s.sums)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(lens), dev(table), 0, 200)
    kept = torch.empty(4, 2, 48, dtype=torch.int32, device="cuda")
    length = torch.empty(4, dtype=torch.int32, device="cuda")
    say("evict out of range", fmt)
    bridge.kv_cache_evict(cache, batch, sums, dev(out), length, 48, sinks=4, recent=20, kept=kept)
    bridge.synchronize()
    pages, want, places, n = evicted(s, s.pages.raw, s.sums, lens, table, out, 48, 4, 20)
    np.testing.assert_array_equal(length.cpu().numpy(), n)
    np.testing.assert_array_equal(kept.cpu().numpy(), places)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)
    np.testing.assert_array_equal(sums.cpu().numpy().view(np.uint32), want.view(np.uint32))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,budget,P,max_kv", [
    ([300, 1, 2, 3, 5, 66, 0, 203], 63, 16, 300), ([300, 127, 129, 130, 131, 90], 130, 16, 5000), ([700, 6, 257], 257, 256, 700),
    ([400, 21], 3, 32, 2 ** 31)])
def test_evict_leaves_what_lies_behind(bridge, fmt, D, lens, budget, P, max_kv):
    """Every byte, those of a last group of four that is not full among them; any length may be expected."""
    import torch

    s = Bounded(fmt, lens, [0] * len(lens), 2, D, P, seed=budget + D)
    s.grow(budget)
    cache, sums = s.cache(), dev(s.sums)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), 0, max_kv)
    length = torch.empty(len(lens), dtype=torch.int32, device="cuda")
    say("what lies behind", fmt, D, lens, budget, P, max_kv)
    bridge.kv_cache_evict(cache, batch, sums, dev(s.table_out), length, budget, sinks=1, recent=2)
    bridge.synchronize()
    pages, out, _, n = evicted(s, s.pages.raw, s.sums, lens, s.table, s.table_out, budget, 1, 2)
    np.testing.assert_array_equal(length.cpu().numpy(), n)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)
    np.testing.assert_array_equal(sums.cpu().numpy().view(np.uint32), out.view(np.uint32))


# ---- steps as they are used -----------------------------------------------------------------------------------------

class Steps:
    """Decoding two sequences step by step over a bounded cache, everything on the device."""

    def __init__(self, bridge, seed, fmt=Q8_0, H=8):
        import torch

        self.bridge, self.H = bridge, H
        self.s = s = Bounded(fmt, [60, 35], [0, 0], 2, 64, 16, seed=seed)
        s.grow(48)
        new = lambda *x, **kw: torch.zeros(*x, device="cuda", **kw)  # noqa: E731
        rest = s.rng.permutation(s.num_pages)
        self.tables = [dev(np.concatenate([s.table, s.table_out[:, :1]], 1)), dev(s.table_out)]
        self.cache = s.cache()
        self.sums = dev(np.where(np.isfinite(s.sums), np.abs(s.sums), 1).astype(np.float32))
        self.batch = m4_bridge.KVBatch(dev(i32(0, 1, 2)), dev(i32(61, 36)), self.tables[0], 1, 80)
        self.rope = m4_bridge.RotaryAxes(64, theta=1e4)
        self.positions = dev(i32(60, 35))
        self.q, self.k, self.v = (new(h, 2, 64, dtype=torch.float16) for h in (H, 2, 2))
        self.o, self.lse = new(H, 2, 64, dtype=torch.float16), new(H, 2)
        self.ws = new(bridge.paged_attn_workspace(self.cache, self.batch, H, 2), dtype=torch.uint8)
        self.len_out, self.kept = new(2, dtype=torch.int32), new(2, 2, 32, dtype=torch.int32)

    def step(self):
        b = self.bridge
        b.kv_cache_append(self.cache, self.batch, self.k, self.v, rope=self.rope, positions=self.positions, Q=self.q)
        b.dispatch_paged_attn(self.cache, self.batch, self.q, self.o, 0.125, workspace=self.ws, lse=self.lse)
        b.kv_cache_weigh(self.cache, self.batch, self.q, self.lse, self.sums, 0.125)

    def evict(self):
        self.bridge.kv_cache_evict(self.cache, self.batch, self.sums, self.tables[1], self.len_out, 32, sinks=2, recent=6, kept=self.kept)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_steps_over_a_bounded_cache(bridge, fmt):
    """Append, attend, weigh; evict; append at the token's own position and attend over the keys that each head kept."""
    x = Steps(bridge, 5, fmt)
    s, H = x.s, x.H
    rng = np.random.default_rng(6)
    q, k, v = half(rng, H, 2, 64), half(rng, 2, 2, 64), half(rng, 2, 2, 64)
    for t, a in ((x.q, q), (x.k, k), (x.v, v)):
        t.copy_(dev(a))
    x.step()
    bridge.synchronize()
    before, pages = x.sums.cpu().numpy(), x.cache.pages.cpu().numpy()
    x.evict()
    bridge.synchronize()
    _, _, places, n = evicted(s, pages, before, i32(61, 36), x.tables[0].cpu().numpy(), s.table_out, 32, 2, 6)
    np.testing.assert_array_equal(x.kept.cpu().numpy(), places)
    assert (n == 32).all()
    # the next token, behind the 32 that each head kept, at the position that it has in the text
    x.batch = m4_bridge.KVBatch(x.batch.q_start, x.len_out + 1, x.tables[1], 1, 48)
    x.positions.copy_(dev(i32(61, 36)))
    x.k.copy_(dev(k[:, ::-1]))
    x.step()
    bridge.synchronize()
    raw = ref.Pages(fmt, s.num_pages, 16, 2, 64)
    raw.raw = x.cache.pages.cpu().numpy().reshape(raw.raw.shape)
    old = ref.Pages(fmt, s.num_pages, 16, 2, 64)
    old.raw = pages.reshape(raw.raw.shape)
    qr = x.q.cpu().numpy()
    for b in range(2):
        now = [raw.read(s.table_out[b, p // 16], p % 16) for p in range(33)]
        was = [old.read(x.tables[0].cpu().numpy()[b, p // 16], p % 16) for p in range((61, 36)[b])]
        kk, vv = (np.stack([t[i] for t in now], 1) for i in range(2))
        for h in range(2):
            for i, p in enumerate(places[b, h]):
                assert (kk[h, i] == was[p][0][h]).all() and (vv[h, i] == was[p][1][h]).all()
        o, ob, z, zb = attend(qr[:, b:b + 1], kk, vv, np.ones((1, 33), bool), 0.125)
        close(x.o[:, b:b + 1].cpu().numpy(), o, ob, "o")
        close(x.lse[:, b:b + 1].cpu().numpy(), z, zb, "lse")


@gpu
def test_steps_in_a_graph(bridge):
    """A step and an eviction, captured and replayed with what is written to their tensors."""
    import torch

    eager, x = Steps(bridge, 7), Steps(bridge, 7)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            x.step()
            x.evict()
    for turn in range(4):
        rng = np.random.default_rng(turn)
        fresh = [half(rng, h, 2, 64) for h in (8, 2, 2)]
        for y in (eager, x):
            for t, a in zip((y.q, y.k, y.v), fresh):
                t.copy_(dev(a))
            y.batch.kv_len.copy_(dev(i32(61 + turn, 36 - 5 * turn)))
        eager.step()
        eager.evict()
        bridge.synchronize()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in ("o", "lse", "sums", "kept", "len_out"):
            assert torch.equal(getattr(x, n).view(torch.uint8), getattr(eager, n).view(torch.uint8)), (turn, n)
        assert torch.equal(x.cache.pages, eager.cache.pages)


# ---- refusals -------------------------------------------------------------------------------------------------------

class Args:
    """Valid arguments without a device, changed one at a time."""

    def __init__(self):
        self.cache = m4_bridge.KVCacheStruct(0x100000, 4 * 16 * 2 * 2 * 4 * 34, 6, 4, 16, 2, 128)
        self.batch = m4_bridge.KVBatchStruct(2, 0x1000, 0x2000, 0x3000, 4, 4, 5, 60)
        self.rows = m4_bridge.RowsStruct(0x300000, 10 * 8 * 128 * 2, 128, 10 * 128)
        self.lse = m4_bridge.RowsStruct(0x400000, 10 * 8 * 4, 1, 10)
        self.T, self.H, self.scale, self.sums, self.held = 10, 8, 0.1, 0x500000, 4 * 2 * 16 * 4
        self.table, self.pages, self.stride, self.budget, self.sinks, self.recent = 0x600000, 3, 3, 48, 4, 8
        self.kept, self.room, self.length = 0x700000, 2 * 2 * 48 * 4, 0x800000


@pytest.mark.parametrize("change,code", [
    (lambda a: None, 0), (set_("sums", 0), -2), (set_("sums", 0x500004), -2), (set_("held", 511), -2), (set_("lse.ptr", 0), -2),
    (set_("lse.bytes", 316), -2), (set_("lse.token_stride", 0), 0), (set_("lse.head_stride", -1), -4), (set_("rows.ptr", 0x300004), -2),
    (set_("rows.bytes", 100), -2), (set_("H", 9), -4), (set_("scale", float("inf")), -4), (set_("cache.format", 2), -3),
    (set_("batch.table_pages", 0), -4), (set_("T", 0), 0), (set_("batch.B", 0), 0), (set_("batch.B", 2 ** 30), -4)])
def test_refused_weights(lib, change, code):  # noqa: F811
    a, r = Args(), ctypes.addressof
    change(a)
    assert lib.m4_bridge_validate_kv_cache_weigh(r(a.cache), r(a.batch), a.T, r(a.rows), r(a.lse), a.H, a.scale, 0, a.sums, a.held) == code


@pytest.mark.parametrize("change,code", [
    (lambda a: None, 0), (set_("sums", 0), -2), (set_("sums", 0x500008), -2), (set_("held", 511), -2), (set_("table", 0), -2),
    (set_("table", 0x600002), -2), (set_("pages", 2), -4), (set_("pages", 0), -4), (set_("stride", 2), -4), (set_("budget", 0), -4),
    (set_("budget", 49), -4), (set_("budget", 11), -4), (set_("budget", 12), 0), (set_("sinks", 41), -4), (set_("sinks", 2 ** 32 - 1), -4),
    (set_("kept", 0), -2), (set_("room", 767), -2), (set_("length", 0), -2), (set_("table", 0x3000), -2), (set_("length", 0x2000), -2),
    (set_("cache.page_size", 8), -4), (set_("batch.kv_len", 0), -2), (set_("batch.B", 0), 0), (set_("batch.B", 2 ** 31), -4)])
def test_refused_evictions(lib, change, code):  # noqa: F811
    """Among them: the old table or its lengths in the place of the new."""
    a, r = Args(), ctypes.addressof
    change(a)
    call = lambda ws, size: lib.m4_bridge_validate_kv_cache_evict(  # noqa: E731
        r(a.cache), r(a.batch), a.sums, a.held, a.table, a.pages, a.stride, a.budget, a.sinks, a.recent, a.kept, a.room, a.length, ws, size)
    assert lib.m4_bridge_kv_evict_workspace(r(a.cache), r(a.batch)) == 0 and call(None, 0) == code
    if code == 0 and a.batch.B:  # long sequences
        a.batch.max_kv = 50000
        need = lib.m4_bridge_kv_evict_workspace(r(a.cache), r(a.batch))
        assert need > 0
        assert call(0x900000, need) == 0 and call(0x900000, need - 1) == -2 and call(None, need) == -2 and call(0x900008, need) == -2


@pytest.mark.parametrize("B,Hkv", [(1, 1), (2, 4), (31, 8)])
def test_workspace_of_evictions_goes_by_the_table(lib, B, Hkv):  # noqa: F811
    """Expectations may be any number: the workspace is for as many keys as the table holds, however many are expected."""
    a, r = Args(), ctypes.addressof
    a.batch.B, a.cache.Hkv, a.cache.page_size = B, Hkv, 256

    def need(pages, max_kv):
        a.batch.table_pages = a.batch.table_stride = pages
        a.batch.max_kv = max_kv
        return lib.m4_bridge_kv_evict_workspace(r(a.cache), r(a.batch))

    for pages in (157, 1024, 0x7fff00):  # 40192 keys, 2^18, all that positions reach
        keys = pages * 256
        for max_kv in (keys + 1, max(keys, 10 ** 9), 2 ** 32 - 1):
            assert need(pages, max_kv) == need(pages, keys) > 0
        assert need(pages, 16384) == 0 and need(pages, 16385) <= need(pages, keys)
    for max_kv in (16385, 10 ** 6, 10 ** 9, 2 ** 32 - 1):  # a table for fewer keys than are worth several workgroups
        assert need(4, max_kv) <= need(0x7fff00, 16385)


def test_what_a_call_holds_and_refuses(launched):  # noqa: F811
    import torch

    cache, batch, z = host()
    x, lse, sums = torch.zeros(2, 3, 64, dtype=torch.float16), torch.zeros(2, 3), torch.zeros(4, 2, 16)
    launched.kv_cache_weigh(cache, batch, x, lse, sums, 0.1)
    launched.kv_cache_evict(cache, batch, sums, z(2, 4), z(2), 32, sinks=4, recent=8)
    assert [c for c in launched.lib.calls if "stream" not in c] == ["m4_bridge_kv_cache_weigh", "m4_bridge_kv_cache_evict"]
    first, second = launched._in_flight_tensors
    assert any(t is sums for t in first) and any(t is sums for t in second)
    assert second[-2:] == (None, None)  # `kept` and a workspace of the call's own go back to its stream
    n = len(launched.lib.calls)
    for call in (lambda: launched.kv_cache_weigh(cache, batch, x, lse, sums.half(), 0.1),
                 lambda: launched.kv_cache_weigh(cache, batch, x, lse, sums[:3], 0.1),
                 lambda: launched.kv_cache_weigh(cache, batch, x, lse, sums.transpose(1, 2).contiguous().transpose(1, 2), 0.1),
                 lambda: launched.kv_cache_weigh(cache, batch, x, lse[:1], sums, 0.1),
                 lambda: launched.kv_cache_weigh(cache, batch, x, lse, sums, 0.1, window=-1),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(3, 4), z(2), 32),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(2, 4).long(), z(2), 32),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(2, 8)[:, ::2], z(2), 32),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(2, 4), z(3), 32),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(2, 4), z(2), -1),
                 lambda: launched.kv_cache_evict(cache, batch, sums, z(2, 4), z(2), 32, kept=z(2, 2, 31))):
        with pytest.raises(ValueError):
            call()
    assert len(launched.lib.calls) == n


@gpu
def test_host_memory_is_refused(bridge):
    import torch

    s = Setup(Q8_0, [40, 40], [2, 1], 2, 64, 16, seed=2)
    x, sums = torch.zeros(2, 3, 64, dtype=torch.float16, device="cuda"), torch.zeros(s.num_pages, 2, 16)
    with pytest.raises(RuntimeError, match="-2"):
        bridge.kv_cache_weigh(s.cache(), s.batch(), x, torch.zeros(2, 3, device="cuda"), sums, 0.1)
    with pytest.raises(RuntimeError, match="-2"):
        bridge.kv_cache_weigh(s.cache(), s.batch(), x, torch.zeros(2, 3), sums.cuda(), 0.1)
    z = lambda *a: torch.zeros(*a, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="-2"):
        bridge.kv_cache_evict(s.cache(), s.batch(), sums.cuda(), z(2, 2), z(2).cuda(), 32)
    assert "device" in bridge.last_error()
    bridge.synchronize()
