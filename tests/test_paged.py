"""The serving operators (rotary positions with several axes, the paged quantized KV cache, attention over it) against
plain implementations in 64 bits, and their refusals."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import m4_bridge
import paged_reference as ref
from paged_reference import Q4_0, Q8_0

gpu = pytest.mark.gpu
FORMATS = [pytest.param(Q8_0, id="q8_0"), pytest.param(Q4_0, id="q4_0")]


def say(*a):
    print(*a, flush=True)


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def half(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def table_of(rng, lens, P, spare=2):
    """A page table of pages in any order, entries past a sequence's end out of range."""
    need = [-(-max(n, 0) // P) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(need + [1])), -7, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


class Setup:
    """Sequences with a filled cache: numpy pages, their values per sequence, and the bridge's view of them."""

    def __init__(self, fmt, lens, new, Hkv, D, P, seed, fill=0xFF):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.new, self.fmt, self.P, self.Hkv, self.D = lens, new, fmt, P, Hkv, D
        self.table, self.num_pages = table_of(rng, lens, P)
        self.pages = ref.Pages(fmt, self.num_pages, P, Hkv, D, fill)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            k, v = half(rng, n, Hkv, D), half(rng, n, Hkv, D)
            (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
            for p in range(n):
                self.pages.write(self.table[b, p // P], p % P, kq[p], kd[p], vq[p], vd[p])
            self.k.append(ref.values(kq, kd).transpose(1, 0, 2))
            self.v.append(ref.values(vq, vd).transpose(1, 0, 2))
        self.q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.q_start[-1])

    def cache(self):
        return m4_bridge.PagedKVCache(self.fmt, self.num_pages, self.P, self.Hkv, self.D, pages=dev(self.pages.raw))

    def batch(self, **kw):
        return m4_bridge.KVBatch(dev(self.q_start), dev(np.array(self.lens, np.int32)), dev(self.table),
                                 **{"max_new": max(self.new), "max_kv": max(self.lens), **kw})

    def expected(self, q, window, scale):
        """q [H, T, D] -> (o, bound) [H, T, D]."""
        parts = [ref.attention(q[:, a:a + n], k, v, L - n, window, scale)
                 for a, n, L, k, v in zip(self.q_start, self.new, self.lens, self.k, self.v)]
        return [np.concatenate(x, 1) for x in zip(*parts)]


def close(got, want, bound, what=""):
    got = got.astype(np.float64)
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN in other places"
    if got.size == 0:
        return
    d = np.where(np.isnan(want), 0, np.abs(got - want))
    worst = np.unravel_index(np.argmax(d - bound), d.shape)
    assert (d <= bound).all(), f"{what}: {int((d > bound).sum())} of {d.size} off; at {worst} {d[worst]:.3g}, bound {bound[worst]:.3g}"


# ---- rotary positions ---------------------------------------------------------------------------------------------

def rope_bound(x, want):
    """fp16 result: 2^-11 of it or 2^-25; sine and cosine: angle to 2^-25 of half a turn, function and products to a
    few units of fp32, 2^-20 of the dims together."""
    return 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -20 * np.abs(x.astype(np.float64)).max(-1, keepdims=True) * 2


@gpu
@pytest.mark.parametrize("H,T,D,dims,sections,traditional,token_major", [
    (1, 1, 128, 128, None, False, False),
    (32, 64, 128, 128, (16, 24, 24), False, False),
    (3, 77, 64, 64, (8, 12, 12), True, True),
    (5, 33, 80, 80, (20, 20), False, True),     # a vision tower's head, rows and columns
    (2, 9, 72, 64, None, False, False),          # the last dims stay
    (7, 130, 256, 128, (0, 64), True, False),
    (40, 513, 128, 64, (10, 11, 11), False, True),
])
def test_rope_axes(bridge, H, T, D, dims, sections, traditional, token_major):
    rng = np.random.default_rng(H * 1000 + T)
    x = half(rng, H, T, D)
    axes = len(sections) if sections else 1
    positions = rng.integers(0, 100000, (axes, T)).astype(np.int32)
    positions[:, 0] = [2 ** 31 - 1, -(2 ** 31), 7][:axes]
    rope = m4_bridge.RotaryAxes(dims, theta=500000.0, sections=sections, traditional=traditional)
    pa = [a for a, n in enumerate(sections) for _ in range(n)] if sections else [0] * (dims // 2)
    want = ref.rotate(x, positions, pa, [500000.0 ** (-2 * i / dims) for i in range(dims // 2)], traditional)
    X = dev(x.transpose(1, 0, 2) if token_major else x)
    import torch

    Y = torch.full_like(X, float("nan"))
    bridge.rope_axes(X, Y, rope, dev(positions), token_major=token_major)
    bridge.synchronize()
    got = Y.cpu().numpy()
    got = got.transpose(1, 0, 2) if token_major else got
    # far positions: the double product pos * f is itself off by 2^-53 of the angle
    slack = 2.0 ** -52 * np.abs(positions.astype(np.float64)).max(0)[None, :, None] * np.abs(x.astype(np.float64)).max(-1, keepdims=True) * 2
    close(got, want, rope_bound(x, want) + slack, "rope")
    assert (got[..., dims:] == x[..., dims:]).all()
    bridge.rope_axes(X, X, rope, dev(positions), token_major=token_major)  # in place
    bridge.synchronize()
    assert torch.equal(X.view(torch.int16), Y.view(torch.int16))


@gpu
def test_rope_axes_matches_rope_and_takes_strides(bridge):
    """One axis with positions offset + m is the bridge's RoPE (both form angles far closer than fp16, so at most the
    last bit differs), on views of a fused projection's output."""
    import torch

    H, T, D, theta = 4, 50, 128, 10000.0
    rng = np.random.default_rng(3)
    x = half(rng, H, T, D)
    A = dev(x)
    bridge.rope(A, theta=theta, offset=17)
    fused = torch.full((T, 3 * H * D + 64), 9.0, dtype=torch.float16, device="cuda")
    X = fused[:, H * D:2 * H * D].view(T, H, D)
    X.copy_(dev(x).transpose(0, 1))
    bridge.rope_axes(X, X, m4_bridge.RotaryAxes(D, theta=theta), torch.arange(17, 17 + T, dtype=torch.int32, device="cuda"),
                     token_major=True)
    bridge.synchronize()
    a, b = A.cpu().numpy().astype(np.float64), X.cpu().numpy().transpose(1, 0, 2).astype(np.float64)
    assert (np.abs(a - b) <= 2.0 ** -10 * np.abs(a) + 2.0 ** -18).all()
    rest = torch.cat([fused[:, :H * D], fused[:, 2 * H * D:]], 1)
    assert bool((rest == 9.0).all())


@gpu
@pytest.mark.parametrize("D,fmt", [(64, None), (128, None), (256, None), (64, Q8_0), (128, Q8_0), (64, Q4_0), (128, Q4_0)])
def test_long_rows_turn_as_short_ones(bridge, D, fmt):
    """64 MB of rows and more, which are loaded another way, alone and beside an append, bit for bit those of parts."""
    import torch

    H, Hkv, T, P, parts = 64, 2, 4096 * 128 // D + 33, 256, 3
    x, kv = torch.randn(H, T, D, device="cuda").half(), torch.randn(Hkv, T, D, device="cuda").half()
    assert x.numel() * 2 > 64 << 20
    rope = m4_bridge.RotaryAxes(D, theta=1e6)
    long, short = torch.zeros_like(x), torch.zeros_like(x)
    places = torch.arange(T, dtype=torch.int32, device="cuda")
    pages = -(-T // P)
    cache = m4_bridge.PagedKVCache(fmt, pages, P, Hkv, D) if fmt is not None else None
    say("long rows", D, fmt)

    def turn(a, b, y):
        if fmt is None:
            return bridge.rope_axes(x[:, a:b], y[:, a:b], rope, places[a:b])
        batch = m4_bridge.KVBatch(dev(np.array([0, b - a], np.int32)), dev(np.array([b], np.int32)),
                                  torch.arange(pages, dtype=torch.int32, device="cuda")[None], b - a, b)
        bridge.kv_cache_append(cache, batch, kv[:, a:b], kv[:, a:b], rope=rope, Q=x[:, a:b], Q_out=y[:, a:b])

    turn(0, T, long)
    for i in range(parts):
        turn(T * i // parts, T * (i + 1) // parts, short)
    bridge.synchronize()
    assert torch.equal(long, short) and (long != x).any()
    turn(0, T, x)  # in place
    bridge.synchronize()
    assert torch.equal(long, x)


# ---- the cache ----------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,Hkv,D,P", [
    ([1], [1], 1, 64, 16),
    ([300, 0, 17, 65], [300, 0, 1, 33], 8, 128, 32),
    ([40, 41, 42, 43, 44], [1, 1, 1, 1, 1], 2, 64, 16),
    ([700], [513], 3, 128, 256),
    ([5, 3], [7, 3], 2, 64, 64),                      # more rows than keys: tokens before position 0 go nowhere
    (list(range(1, 131)), [1] * 130, 1, 64, 16),      # more sequences than a wave has lanes
])
def test_append_and_read(bridge, fmt, lens, new, Hkv, D, P):
    """Every byte of the pages, those of other tokens untouched; read gives the values, and the rest stays."""
    import torch

    s = Setup(fmt, lens, new, Hkv, D, P, seed=len(lens))
    T, pad = s.T, 5  # rows behind the last sequence
    k, v = half(s.rng, T + pad, Hkv, D), half(s.rng, T + pad, Hkv, D)
    k[0] = 0
    k[1 % T, :, :32] = np.float16(0.25)  # ties
    k[1 % T, :, 3] = np.float16(-0.25)
    v[T // 2, 0, 5] = np.float16(65504)
    cache, batch = s.cache(), s.batch()
    bridge.kv_cache_append(cache, batch, dev(k), dev(v), token_major=True)
    ko = torch.full((Hkv, T + pad, D), 3.0, dtype=torch.float16, device="cuda")
    vo = torch.full((Hkv, T + pad, D), 3.0, dtype=torch.float16, device="cuda")
    bridge.kv_cache_read(cache, batch, ko, vo)
    bridge.synchronize()
    (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
    ek, ev = np.full((Hkv, T + pad, D), 3, np.float16), np.full((Hkv, T + pad, D), 3, np.float16)
    for b, (L, n, a) in enumerate(zip(lens, new, s.q_start)):
        for i in range(n):
            p, t = L - n + i, a + i
            if p < 0:
                continue
            s.pages.write(s.table[b, p // P], p % P, kq[t], kd[t], vq[t], vd[t])
            ek[:, t], ev[:, t] = s.pages.read(s.table[b, p // P], p % P)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)
    np.testing.assert_array_equal(ko.cpu().numpy().view(np.uint16), ek.view(np.uint16))
    np.testing.assert_array_equal(vo.cpu().numpy().view(np.uint16), ev.view(np.uint16))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_long_reads_are_short_ones(bridge, fmt, D):
    """Results that pass the caches by, bit for bit those of parts that do not."""
    import torch

    T, Hkv, P, parts = 8192 * 128 // D + 77, 16, 256, 3
    pages = -(-T // P)
    cache = m4_bridge.PagedKVCache(fmt, pages, P, Hkv, D)
    x = torch.randn(2, Hkv, T, D, device="cuda").half()
    table = torch.randperm(pages, device="cuda").int()[None]
    batch = lambda a, b: m4_bridge.KVBatch(dev(np.array([0, b - a], np.int32)), dev(np.array([b], np.int32)),  # noqa: E731
                                           table, T, T)
    bridge.kv_cache_append(cache, batch(0, T), x[0], x[1])
    long, short = torch.zeros_like(x), torch.zeros_like(x)
    assert long.numel() * 2 > 64 << 20
    bridge.kv_cache_read(cache, batch(0, T), long[0], long[1])
    for i in range(parts):
        a, b = T * i // parts, T * (i + 1) // parts
        bridge.kv_cache_read(cache, batch(a, b), short[0, :, a:b], short[1, :, a:b])
    bridge.synchronize()
    assert torch.equal(long, short) and (long != 0).any()


@gpu
def test_append_matches_quantize_kv_q8_0(bridge):
    """The cache holds what m4_bridge_quantize_kv_q8_0 makes of the same rows, scale and code for code."""
    import torch

    Hkv, T, D = 2, 96, 128
    rng = np.random.default_rng(11)
    k = half(rng, Hkv, T, D)
    K = dev(k)
    blocks = torch.empty(Hkv * T * D // 32 * 34, dtype=torch.uint8, device="cuda")
    bridge.quantize_kv_q8_0(K, blocks)
    cache = m4_bridge.PagedKVCache(Q8_0, 6, 16, Hkv, D)
    batch = m4_bridge.KVBatch(dev(np.array([0, T], np.int32)), dev(np.array([T], np.int32)),
                              dev(np.arange(6, dtype=np.int32)[None]))
    bridge.kv_cache_append(cache, batch, K, K)
    ko, vo = torch.empty_like(K), torch.empty_like(K)
    bridge.kv_cache_read(cache, batch, ko, vo)
    bridge.synchronize()
    b = blocks.cpu().numpy().reshape(Hkv, T, D // 32, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0]
    want = ref.values(np.ascontiguousarray(b[..., 2:]).view(np.int8).reshape(Hkv, T, D).astype(np.int32), d)
    np.testing.assert_array_equal(ko.cpu().numpy().view(np.uint16), want.view(np.uint16))
    np.testing.assert_array_equal(vo.cpu().numpy().view(np.uint16), want.view(np.uint16))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,dims,axes,traditional", [(64, 64, 1, False), (128, 128, 3, False), (128, 64, 1, True)])
def test_fused_rope_append_is_rope_then_append(bridge, fmt, D, dims, axes, traditional):
    """Bit for bit, positions given or each token's place; rows without a place keep what Q_out held."""
    import torch

    H, Hkv, P = 6, 2, 16
    s = Setup(fmt, [70, 9, 33], [41, 9, 1], Hkv, D, P, seed=5)
    T, pad = s.T, 3
    rope = m4_bridge.RotaryAxes(dims, theta=1e6, sections=(8, 28, 28) if axes == 3 else None, traditional=traditional)
    q, k, v = (dev(half(s.rng, n, T + pad, D)) for n in (H, Hkv, Hkv))
    places = np.concatenate([np.arange(L - n, L) for L, n in zip(s.lens, s.new)] + [np.zeros(pad)]).astype(np.int32)
    positions = dev(np.stack([places * (a + 1) for a in range(axes)]))
    one, two = s.cache(), s.cache()
    qo = torch.full_like(q, 7.0)
    bridge.kv_cache_append(one, s.batch(), k, v, rope=rope, positions=positions if axes > 1 else None, Q=q, Q_out=qo)
    kr, qr = torch.empty_like(k), torch.empty_like(q)
    bridge.rope_axes(k, kr, rope, positions)
    bridge.rope_axes(q, qr, rope, positions)
    bridge.kv_cache_append(two, s.batch(), kr, v)
    bridge.synchronize()
    assert torch.equal(one.pages, two.pages)
    assert torch.equal(qo[:, :T].view(torch.int16), qr[:, :T].view(torch.int16))
    assert bool((qo[:, T:] == 7.0).all())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,max_new,max_kv", [(4, 20, 60), (32, 8, 10 ** 8), (32, 4096, 10 ** 8)],
                         ids=["rows", "chunks", "both"])
def test_bad_metadata_is_not_followed(bridge, fmt, H, max_new, max_kv):
    """Pages that are not there, more keys than the table holds, starts past the rows: such tokens are not written, not
    read and not seen, and nothing outside the buffers is touched."""
    import torch

    P, Hkv, D = 16, 2, 64
    s = Setup(fmt, [60, 40], [20, 6], Hkv, D, P, seed=9, fill=0)
    table = s.table.copy()
    table[0, 1] = 10 ** 9      # keys 16 .. 31 of sequence 0
    table[1, 2] = -1           # keys 32 .. 39 of sequence 1: its new tokens
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array([60, 40], np.int32)), dev(table), max_new, max_kv)
    cache = s.cache()
    q = half(s.rng, H, s.T, D)
    O = torch.full((H, s.T, D), 5.0, dtype=torch.float16, device="cuda")
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, 0.125)
    bridge.synchronize()
    for b in range(2):
        valid = np.ones(s.lens[b], bool)
        valid[16:32 if b == 0 else 16] = False
        valid[32 if b else 60:] = False
        a, n = s.q_start[b], s.new[b]
        want, bound = ref.attention(q[:, a:a + n], s.k[b], s.v[b], s.lens[b] - n, 0, 0.125, valid)
        close(O[:, a:a + n].cpu().numpy(), want, bound, f"sequence {b}")
    # writing: sequence 1's tokens have no page
    k = half(s.rng, s.T, Hkv, D)
    bridge.kv_cache_append(cache, batch, dev(k), dev(k), token_major=True)
    bridge.synchronize()
    kq, kd = ref.quantize(fmt, k)
    for i in range(20):
        p = 40 + i
        s.pages.write(s.table[0, p // P], p % P, kq[i], kd[i], kq[i], kd[i])
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)
    # lengths past the table and starts past the rows: no fault, rows in range still written
    wild = m4_bridge.KVBatch(dev(np.array([0, 10 ** 6, 5], np.int32)), dev(np.array([2 ** 31 - 1, -5], np.int32)),
                             dev(s.table), max_new, max_kv)
    bridge.dispatch_paged_attn(cache, wild, dev(q), O, 0.125)
    bridge.kv_cache_append(cache, wild, dev(k), dev(k), token_major=True)
    bridge.synchronize()
    assert bool(torch.isfinite(O).all())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_negative_lengths_hold_nothing(bridge, fmt):
    """However far below zero: positions are not formed from such a length past 32 bits."""
    import torch

    s = Setup(fmt, [40, 40], [3, 3], 2, 64, 16, seed=3)
    cache, x = s.cache(), dev(half(s.rng, 2, 6, 64))
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array([-2 ** 31, -1], np.int32)), dev(s.table), 3, 40)
    bridge.kv_cache_append(cache, batch, x, x)
    out, O = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    bridge.kv_cache_read(cache, batch, out, out.clone())
    bridge.dispatch_paged_attn(cache, batch, x, O, 0.125)
    bridge.synchronize()
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)
    assert (out == 7.0).all() and (O == 0.0).all()


# ---- attention ----------------------------------------------------------------------------------------------------

def check_attention(bridge, s, H, window=0, scale=None, token_major=False, infinite=False, **kw):
    import torch

    scale = s.D ** -0.5 if scale is None else scale
    pad = 3
    q = half(s.rng, H, s.T + pad, s.D)
    Q = dev(q.transpose(1, 0, 2) if token_major else q)
    O = torch.full((s.T + pad, H, s.D), 6.0, dtype=torch.float16, device="cuda")
    say("paged attention", s.fmt, s.lens[:6], s.new[:6], H, s.Hkv, s.D, s.P, window)
    bridge.dispatch_paged_attn(s.cache(), s.batch(**kw), Q, O, scale, token_major=token_major, o_token_major=True,
                               window=window)
    bridge.synchronize()
    got = O.cpu().numpy().transpose(1, 0, 2)
    assert (got[:, s.T:] == 6.0).all(), "rows behind the last sequence"
    want, bound = s.expected(q[:, :s.T], window, scale)
    got = got[:, :s.T]
    if infinite:
        got = np.where(np.isfinite(got), got, np.float16("nan"))
    close(got, want, bound, "attention")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,H,Hkv,D,P,window", [
    ([1], [1], 1, 1, 64, 16, 0),
    ([1000], [1], 32, 8, 128, 16, 0),
    ([1, 15, 16, 17, 127, 128, 129, 0, 500], [1, 1, 1, 1, 1, 1, 1, 0, 1], 8, 2, 64, 16, 0),
    ([200, 33, 64], [5, 5, 5], 32, 8, 64, 32, 0),             # drafted tokens
    ([700, 1, 90], [129, 1, 90], 8, 2, 128, 64, 0),           # a chunk among single tokens, a whole prompt
    ([300, 300], [1, 40], 4, 4, 64, 256, 0),                  # one head a KV head
    ([130], [7], 32, 1, 128, 16, 0),                          # one KV head
    ([257, 90], [3, 90], 10, 2, 64, 16, 0),                   # groups of 5
    ([400, 31], [70, 31], 6, 2, 128, 16, 1),                  # each row sees itself
    ([400, 900], [70, 2], 6, 2, 128, 16, 37),
    ([900, 500], [300, 1], 4, 1, 64, 64, 256),
    ([3, 2, 0], [9, 2, 4], 4, 2, 64, 16, 0),                  # rows that see nothing
    (list(range(1, 301)), [1] * 300, 2, 1, 64, 16, 0),        # more sequences than a workgroup has lanes
    ([1000], [1000], 4, 1, 128, 16, 0),                       # a whole prompt
    ([2100, 515], [260, 515], 16, 4, 64, 32, 0),
    ([700, 1], [333, 1], 10, 2, 128, 256, 100),               # groups of 5: row tiles that are not full
    ([300], [200], 160, 1, 64, 16, 0),                        # a group wider than a row tile
    ([5000], [70], 8, 8, 128, 64, 0),
    ([700, 90, 40, 33, 500], [300, 1, 2, 17, 128], 8, 2, 128, 16, 0),  # chunks and steps in any order
])
@pytest.mark.parametrize("kernels", ["as_planned", "rows", "chunks", "both"])
def test_paged_attention(bridge, fmt, lens, new, H, Hkv, D, P, window, kernels):
    # what is expected of the lengths chooses the kernels, as far as the batch allows: one of which most sequences have
    # few rows goes to the kernel for rows, or with its longer sequences to the other
    kw = {"as_planned": {}, "rows": {"max_new": 1, "max_kv": 1}, "both": {"max_new": 4096, "max_kv": 10 ** 8},
          "chunks": {"max_new": -(-128 // (H // Hkv)), "max_kv": 10 ** 8}}[kernels]
    check_attention(bridge, Setup(fmt, lens, new, Hkv, D, P, seed=sum(lens) + H), H, window, **kw)


@gpu
@pytest.mark.parametrize("max_new,max_kv", [(1, 1), (1, 100000), (5000, 1), (0, 0)])
def test_paged_attention_holds_for_any_expectation(bridge, max_new, max_kv):
    check_attention(bridge, Setup(Q8_0, [800, 5, 77], [60, 5, 1], 2, 64, 16, seed=4), 8, max_new=max_new, max_kv=max_kv,
                    token_major=True)


@gpu
@pytest.mark.parametrize("max_new,max_kv", [(2 ** 32 - 1, 2 ** 32 - 1), (2 ** 32 - 1, 1), (1, 2 ** 32 - 1)])
def test_expectations_past_any_length(bridge, max_new, max_kv):
    s = Setup(Q4_0, [70] * 5, [3] * 5, 2, 64, 16, seed=5)
    assert 0 < bridge.paged_attn_workspace(s.cache(), s.batch(max_new=max_new, max_kv=max_kv), 8, s.T) < 1 << 28
    check_attention(bridge, s, 8, max_new=max_new, max_kv=max_kv)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,kw", [(1, {"max_new": 1}), (8, {"max_new": 8}), (60, {"max_new": 4096, "max_kv": 10 ** 8})],
                         ids=["rows_of_16", "rows_of_32", "chunks"])
def test_many_light_keys_beside_a_heavy_one(bridge, D, n, kw):
    """Weights of 2^-24.4 beside one of 1: fp16 has two bits at most for them, and 40000 of them count."""
    import torch

    L, P = 40000, 256
    k, v = np.zeros((1, L, D), np.float16), np.ones((1, L, D), np.float16)
    k[0, 0], v[0, 0] = 24.4 * math.log(2) * 8 / D, 0.0
    q = np.ones((4, n, D), np.float16)
    pages = -(-L // P)
    cache = m4_bridge.PagedKVCache(Q8_0, pages, P, 1, D)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    kv_len = dev(np.array([L], np.int32))
    bridge.kv_cache_append(cache, m4_bridge.KVBatch(dev(np.array([0, L], np.int32)), kv_len, table, L, L), dev(k), dev(v))
    O = torch.zeros(4, n, D, dtype=torch.float16, device="cuda")
    batch = m4_bridge.KVBatch(dev(np.array([0, n], np.int32)), kv_len, table, **{"max_kv": L, **kw})
    say("light keys", D, n)
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, 0.125)
    bridge.synchronize()
    kx, vx = (ref.values(*ref.quantize(Q8_0, x[0])) for x in (k, v))
    want, bound = ref.attention(q, kx[None], vx[None], L - n, 0, 0.125)
    assert 0.001 < want.min() and want.max() < 0.01
    close(O.cpu().numpy(), want, bound, "light keys")


@gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_paged_attention_scales(bridge, scale):
    check_attention(bridge, Setup(Q8_0, [300, 40], [20, 1], 2, 64, 16, seed=6), 4, scale=scale)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,H,kw", [([60, 3], 16, {"max_new": 16, "max_kv": 10 ** 8}),
                                      ([60, 3], 16, {"max_new": 4096, "max_kv": 10 ** 8}), ([2, 3], 4, {}), ([15, 3], 4, {})],
                         ids=["chunks", "both", "rows_of_16", "rows_of_32"])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(bridge, fmt, D, new, H, kw):
    """A key whose V scale is infinite reaches the rows that see it, in its 32 dims, and no other; what was never written
    (all-ones bytes: NaN scales) reaches none.  Its values are its codes times infinity, so a row's result there is an
    infinity or NaN: `infinite` takes the two alike."""
    s = Setup(fmt, [100, 50], new, 2, D, 16, seed=8)
    for b, p in ((0, 70), (1, 48)):
        raw = s.pages.raw[s.table[b, p // 16]]
        avs = s.pages._places(p % 16)[3]
        raw[1, avs[1]], raw[1, avs[1] + 1] = 0x00, 0x7C  # +inf, dims 32 .. 63 of head 1
        s.v[b][1, p, 32:64] = np.nan
    check_attention(bridge, s, H, infinite=True, **kw)


@gpu
def test_two_gigabytes_and_more(bridge):
    """Pages whose byte offsets pass 2^32."""
    import torch

    Hkv, D, P = 8, 128, 64
    per = ref.page_bytes(Q8_0, P, D) * Hkv
    num = (5 << 30) // per
    s = Setup(Q8_0, [300, 65], [9, 1], Hkv, D, P, seed=12)
    mem = torch.empty(num * per, dtype=torch.uint8, device="cuda").view(num, Hkv, -1)
    where = torch.tensor(np.random.default_rng(1).permutation(np.arange(num - 60, num))[:s.num_pages].astype(np.int64))
    mem[where.cuda()] = dev(s.pages.raw)
    cache = m4_bridge.PagedKVCache(Q8_0, num, P, Hkv, D, pages=mem)
    table = np.where(s.table >= 0, where.numpy()[np.maximum(s.table, 0)], -1).astype(np.int32)
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(s.lens, np.int32)), dev(table), 9, 300)
    q = half(s.rng, 16, s.T, D)
    O = torch.empty(16, s.T, D, dtype=torch.float16, device="cuda")
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, D ** -0.5)
    bridge.synchronize()
    close(O.cpu().numpy(), *s.expected(q, 0, D ** -0.5), "attention")
    k = half(s.rng, s.T, Hkv, D)
    bridge.kv_cache_append(cache, batch, dev(k), dev(k), token_major=True)
    ko, vo = (torch.empty(s.T, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    bridge.kv_cache_read(cache, batch, ko, vo, token_major=True)
    bridge.synchronize()
    want = ref.values(*ref.quantize(Q8_0, k))
    assert (ko.cpu().numpy() == want).all() and (vo.cpu().numpy() == want).all()


# ---- together, as they are used -----------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_chunks_and_steps_of_a_growing_batch(bridge, fmt):
    """Prompts in chunks, then single tokens: rotate and write, attend, step after step, against 64 bits of the tokens
    that the cache holds."""
    import torch

    H, Hkv, D, P, theta = 8, 2, 64, 16, 10000.0
    rng = np.random.default_rng(2)
    plan = [[50, 3, 0], [20, 0, 70], [1, 1, 1], [5, 1, 1], [1, 1, 1]]
    total = np.sum(plan, 0)
    table, num = table_of(rng, list(total), P)
    cache = m4_bridge.PagedKVCache(fmt, num, P, Hkv, D)
    cache.pages.fill_(255)
    rope = m4_bridge.RotaryAxes(D, theta=theta)
    inv = [theta ** (-2 * i / D) for i in range(D // 2)]
    lens = np.zeros(3, np.int64)
    kv = [[np.zeros((Hkv, 0, D), np.float16)] * 2 for _ in range(3)]
    for new in plan:
        lens += new
        T = sum(new)
        q, k, v = half(rng, H, T, D), half(rng, Hkv, T, D), half(rng, Hkv, T, D)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        batch = m4_bridge.KVBatch(dev(starts), dev(lens.astype(np.int32)), dev(table))
        Q, O = dev(q), torch.empty(T, H * D, dtype=torch.float16, device="cuda")
        bridge.kv_cache_append(cache, batch, dev(k), dev(v), rope=rope, Q=Q)
        bridge.dispatch_paged_attn(cache, batch, Q, O.view(T, H, D), D ** -0.5, o_token_major=True)
        ko, vo = (torch.empty(Hkv, T, D, dtype=torch.float16, device="cuda") for _ in range(2))
        bridge.kv_cache_read(cache, batch, ko, vo)
        bridge.synchronize()
        qr = Q.cpu().numpy()
        for b, n in enumerate(new):
            a = starts[b]
            pos = np.arange(lens[b] - n, lens[b])[None]
            want = ref.rotate(q[:, a:a + n], pos, [0] * (D // 2), inv, False)
            close(qr[:, a:a + n], want, rope_bound(q[:, a:a + n], want), "rotated queries")
            # keys
            kw = ref.rotate(k[:, a:a + n], pos, [0] * (D // 2), inv, False)
            big = np.abs(kw).reshape(Hkv, n, D // 32, 32).max(-1).repeat(32, -1)
            step = big / (127 if fmt == Q8_0 else 8)
            got = ko[:, a:a + n].cpu().numpy()
            # half a step (Q4_0: a whole one for a value like the largest of the other sign), and three roundings to
            # fp16 of at most the largest value: the rotated key, the scale, the value (3 * 2^-11 < 2^-9)
            assert (np.abs(got - kw) <= step * (0.5 if fmt == Q8_0 else 1.0) + 2.0 ** -9 * big + 2.0 ** -24).all()
            kv[b] = [np.concatenate([old, x[:, a:a + n].cpu().numpy()], 1) for old, x in zip(kv[b], (ko, vo))]
            if n:
                o, bound = ref.attention(qr[:, a:a + n], *kv[b], lens[b] - n, 0, D ** -0.5)
                close(O.view(T, H, D)[a:a + n].cpu().numpy().transpose(1, 0, 2), o, bound, f"sequence {b}")


@gpu
@pytest.mark.parametrize("fmt,D", [(Q8_0, 64), (Q4_0, 128)])
def test_captured_chunks_among_steps(bridge, fmt, D):
    """A batch for both kernels, captured once: replays follow lengths, starts and pages that change on the device, so
    that a sequence goes from one kernel to the other, and equal the eager calls bit for bit."""
    import torch

    H, Hkv, P = 8, 2, 16
    s = Setup(fmt, [400, 300, 350], [90, 2, 7], Hkv, D, P, seed=31)
    cache, q = s.cache(), dev(half(s.rng, H, s.T, D))
    q_start, kv_len, table = dev(s.q_start), dev(np.array(s.lens, np.int32)), dev(s.table)
    batch = m4_bridge.KVBatch(q_start, kv_len, table, 4096, 10 ** 8)
    eager, graphed = torch.zeros_like(q), torch.zeros_like(q)
    ws = torch.empty(bridge.paged_attn_workspace(cache, batch, H, s.T), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        bridge.dispatch_paged_attn(cache, batch, q, graphed, 0.125, workspace=ws)
    for starts, lens in (([0, 90, 92, 99], [400, 300, 350]), ([0, 3, 80, 99], [50, 290, 19]), ([0, 0, 99, 99], [7, 200, 1]),
                         ([0, 90, 92, 95], [399, 300, 350])):
        q_start.copy_(dev(np.array(starts, np.int32)))
        kv_len.copy_(dev(np.array(lens, np.int32)))
        eager.fill_(3.0)
        graphed.fill_(3.0)
        ws.fill_(0x7F)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        bridge.dispatch_paged_attn(cache, batch, q, eager, 0.125)
        bridge.synchronize()
        assert torch.equal(eager.view(torch.int16), graphed.view(torch.int16)), f"{starts} {lens}"
        assert bool((graphed[:, starts[-1]:] == 3.0).all()) and not bool((graphed[:, :starts[-1]] == 3.0).all())
        s.q_start, s.new = np.array(starts, np.int32), [b - a for a, b in zip(starts, starts[1:])]
        n = starts[-1]
        want = [np.concatenate(x, 1) for x in zip(*[
            ref.attention(q.cpu().numpy()[:, a:a + m], k[:, :L], v[:, :L], L - m, 0, 0.125)
            for a, m, L, k, v in zip(starts, s.new, lens, s.k, s.v)])]
        close(graphed.cpu().numpy()[:, :n], want[0], want[1], f"replay of {starts} {lens}")


@gpu
@pytest.mark.parametrize("fmt,own_workspace", [(Q8_0, True), (Q4_0, False)])
def test_captured_decoding_steps(bridge, fmt, own_workspace):
    """A step captured once and replayed as the sequences grow, with the program's own work and waits in between,
    equals the eager calls bit for bit; two graphs with a workspace each replay side by side on their streams."""
    import torch

    H, Hkv, D, P, B, steps = 8, 2, 128, 16, 5, 4
    rng = np.random.default_rng(7)
    base = np.array([0, 15, 200, 31, 700])
    table, num = table_of(rng, list(base + steps), P)
    filled = rng.integers(0, 100, (num, Hkv, ref.page_bytes(fmt, P, D))).astype(np.uint8)
    rope = m4_bridge.RotaryAxes(D)
    xs = [[dev(half(rng, n, B, D)) for n in (H, Hkv, Hkv)] for _ in range(steps)]

    def lane(stream):
        cache = m4_bridge.PagedKVCache(fmt, num, P, Hkv, D, pages=dev(filled))
        kv_len = torch.zeros(B, dtype=torch.int32, device="cuda")
        batch = m4_bridge.KVBatch(torch.arange(B + 1, dtype=torch.int32, device="cuda"), kv_len, dev(table), 1, 704)
        q, k, v = (torch.zeros_like(t) for t in xs[0])
        o = torch.zeros(B, H, D, dtype=torch.float16, device="cuda")
        ws = torch.empty(bridge.paged_attn_workspace(cache, batch, H, B), dtype=torch.uint8, device="cuda") if own_workspace else None

        def step():
            bridge.kv_cache_append(cache, batch, k, v, rope=rope, Q=q)
            bridge.dispatch_paged_attn(cache, batch, q, o, D ** -0.5, o_token_major=True, workspace=ws)

        return cache, kv_len, (q, k, v), o, step

    def feed(lane_, i):
        lane_[1].copy_(dev((base + i + 1).astype(np.int32)))
        for dst, src in zip(lane_[2], xs[i]):
            dst.copy_(src)

    eager, one, two = (lane(None) for _ in range(3))
    graphs = []
    for l in (one, two):
        feed(l, 0)
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            l[4]()
        graphs.append((g, side))
    for i in range(steps):
        feed(eager, i)
        eager[4]()
        bridge.synchronize()
        torch.cuda.synchronize()
        for l in (one, two):
            feed(l, i)
        torch.cuda.synchronize()
        for g, side in graphs:
            with torch.cuda.stream(side):
                g.replay()
        torch.cuda.synchronize()
        for l in (one, two):
            assert torch.equal(l[3].view(torch.int16), eager[3].view(torch.int16)), f"step {i}"
            assert torch.equal(l[0].pages, eager[0].pages), f"step {i}"


@gpu
@pytest.mark.parametrize("norm_type,traditional,Hq,Hkv,D,wfmt", [(1, False, 4, 2, 64, 0), (2, True, 4, 1, 128, 3)])
def test_paged_layer_in_chunks_and_steps(bridge, oracle, norm_type, traditional, Hq, Hkv, D, wfmt):
    """The layer over two prompts that arrive in chunks beside each other, ending with single tokens, against the
    oracle's layer of each whole prompt: causal attention makes a row's result the same either way.  Tolerance as for
    the prefill layer: fp16 in between on both sides, a tie upstream moves a value by about one output step."""
    import synth
    import torch
    from tolerance import TOL

    dm, Nm, P = 256, 512, 16
    lens = [90, 41]
    rng = np.random.default_rng(72)
    Xs = [synth.activations(n, dm, 71 + n) for n in lens]
    na, nf = ((1 + 0.1 * rng.standard_normal(dm)).astype(np.float16) for _ in range(2))
    if norm_type == 2:
        na, nf = (na - 1).astype(np.float16), (nf - 1).astype(np.float16)
    shapes = [(Hq * D, dm), (Hkv * D, dm), (Hkv * D, dm), (dm, Hq * D), (Nm, dm), (Nm, dm), (dm, Nm)]
    Ws = [synth.quantized_weights(wfmt, n, k, 80 + i) for i, (n, k) in enumerate(shapes)]
    table, num = table_of(rng, lens, P)
    cache = m4_bridge.PagedKVCache(Q8_0, num, P, Hkv, D)
    rope = m4_bridge.RotaryAxes(D, traditional=traditional)
    scale = D ** -0.5
    W = [dev(w) for w in Ws]
    got = [np.zeros((0, dm), np.float16) for _ in lens]
    done = np.zeros(2, np.int64)
    for new in ([50, 7], [0, 33], [39, 0], [1, 1]):
        x = np.concatenate([Xs[b][done[b]:done[b] + n] for b, n in enumerate(new)])
        done += new
        batch = m4_bridge.KVBatch(dev(np.array([0, new[0], sum(new)], np.int32)), dev(done.astype(np.int32)), dev(table))
        out = torch.empty(len(x), dm, dtype=torch.float16, device="cuda")
        bridge.paged_layer(dev(x), dev(na), *W[:4], dev(nf), *W[4:], out, wfmt, dm, Hq, Nm, scale, cache, batch, rope,
                           norm_type=norm_type)
        bridge.synchronize()
        o = out.cpu().numpy()
        got = [np.concatenate([got[0], o[:new[0]]]), np.concatenate([got[1], o[new[0]:]])]
    for b, n in enumerate(lens):
        want = oracle.layer_ex(wfmt, Xs[b], na, *Ws[:4], nf, *Ws[4:], Hq, Hkv, D, Nm, scale, norm_type=norm_type, eps=1e-5,
                               rope=True, theta=10000.0, offset=0, traditional=traditional)
        d = np.abs(got[b].astype(np.float64) - want.astype(np.float64)).max()
        say(f"paged layer, sequence {b}: max|diff| {d:.3g}")
        assert d <= 2 * TOL
    with pytest.raises(RuntimeError, match="-2"):  # in place
        x = dev(Xs[0][:1])
        bridge.paged_layer(x, dev(na), *W[:4], dev(nf), *W[4:], x, wfmt, dm, Hq, Nm, scale, cache,
                           m4_bridge.KVBatch(dev(np.array([0, 1, 1], np.int32)), dev(np.array(lens, np.int32)), dev(table)))


@gpu
def test_paged_layer_captured(bridge):
    """A layer's decoding step, replayed as the sequence grows, against the eager calls."""
    import synth
    import torch

    dm, Nm, Hq, Hkv, D, P, steps = 256, 512, 4, 2, 64, 16, 4
    shapes = [(Hq * D, dm), (Hkv * D, dm), (Hkv * D, dm), (dm, Hq * D), (Nm, dm), (Nm, dm), (dm, Nm)]
    W = [dev(synth.quantized_weights(0, n, k, 80 + i)) for i, (n, k) in enumerate(shapes)]
    na = dev(np.ones(dm, np.float16))
    rope = m4_bridge.RotaryAxes(D)
    xs = [dev(synth.activations(2, dm, 90 + i)) for i in range(steps)]

    def lane():
        cache = m4_bridge.PagedKVCache(Q4_0, 4, P, Hkv, D)
        kv_len = torch.zeros(2, dtype=torch.int32, device="cuda")
        table = dev(np.array([[0, 1], [2, 3]], np.int32))
        batch = m4_bridge.KVBatch(dev(np.array([0, 1, 2], np.int32)), kv_len, table, 1, 32)
        x, out = torch.zeros(2, dm, dtype=torch.float16, device="cuda"), torch.zeros(2, dm, dtype=torch.float16, device="cuda")
        return cache, kv_len, x, out, lambda: bridge.paged_layer(x, na, *W[:4], na, *W[4:], out, 0, dm, Hq, Nm, 0.125, cache,
                                                                  batch, rope)

    eager, graphed, first = lane(), lane(), lane()
    first[4]()  # the bridge's scratch grows to this size before the capture (no keys yet: nothing is written)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        graphed[4]()
    for i in range(steps):
        for l in (eager, graphed):
            l[1].copy_(dev(np.array([i + 1, i + 14], np.int32)))
            l[2].copy_(xs[i])
        eager[4]()
        bridge.synchronize()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager[3].view(torch.int16), graphed[3].view(torch.int16)), f"step {i}"
        assert torch.equal(eager[0].pages, graphed[0].pages), f"step {i}"


@gpu
def test_on_another_stream(bridge):
    import torch

    s = Setup(Q8_0, [500, 80], [1, 30], 2, 64, 16, seed=21)
    q = half(s.rng, 8, s.T, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        O = torch.empty(8, s.T, 64, dtype=torch.float16, device="cuda")
        bridge.dispatch_paged_attn(s.cache(), s.batch(), dev(q), O, 0.125)
        done = O.clone()
    side.synchronize()
    bridge.synchronize()
    close(done.cpu().numpy(), *s.expected(q, 0, 0.125), "attention")


# ---- refusals -----------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib(libpath):
    return m4_bridge.load_library(libpath)


def test_cache_bytes(lib):
    f = lib.m4_bridge_kv_cache_bytes
    assert f(6, 10, 16, 8, 128) == 10 * 16 * 8 * 2 * 4 * 34
    assert f(0, 3, 256, 1, 64) == 3 * 256 * 2 * 2 * 18
    for bad in ((1, 10, 16, 8, 128), (6, 0, 16, 8, 128), (6, 10, 8, 8, 128), (6, 10, 24, 8, 128), (6, 10, 512, 8, 128),
                (6, 10, 16, 0, 128), (6, 10, 16, 8, 96)):
        assert f(*bad) == 0, bad


class Args:
    """Well-formed arguments at addresses that are never followed, to change one at a time."""

    def __init__(self):
        self.T, self.H = 10, 8
        self.cache = m4_bridge.KVCacheStruct(0x100000, 4 * 16 * 2 * 2 * 4 * 34, 6, 4, 16, 2, 128)
        self.batch = m4_bridge.KVBatchStruct(2, 0x1000, 0x2000, 0x3000, 4, 4, 5, 60)
        self.kv = m4_bridge.RowsStruct(0x200000, 2 * self.T * 128 * 2, 128, self.T * 128)
        self.q = m4_bridge.RowsStruct(0x300000, 8 * self.T * 128 * 2, 128, self.T * 128)
        self.rope = m4_bridge.RopeAxesStruct(64, 3, 0, 0x500000, 64 * 12)
        self.positions, self.stride, self.scale, self.ws, self.ws_bytes = 0x4000, self.T, 0.1, 0x400000, 1 << 30

    def codes(self, lib):
        r = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
        return (lib.m4_bridge_validate_kv_cache_append(r(self.cache), r(self.batch), self.T, r(self.kv), r(self.kv), r(self.rope),
                                                       self.positions, self.stride, r(self.q), r(self.q), self.H),
                lib.m4_bridge_validate_kv_cache_read(r(self.cache), r(self.batch), self.T, r(self.kv), r(self.kv)),
                lib.m4_bridge_validate_paged_attn(r(self.cache), r(self.batch), self.T, r(self.q), r(self.q), self.H, self.scale, 0,
                                                  self.ws, self.ws_bytes),
                lib.m4_bridge_validate_rope_axes(r(self.rope), self.positions, self.stride, r(self.q), r(self.q), self.T,
                                                 self.H, 128))


def _set(path, value):
    def change(a):
        *at, last = path.split(".")
        o = a
        for n in at:
            o = getattr(o, n)
        setattr(o, last, value)
    change.__name__ = f"{path}={value}"
    return change


@pytest.mark.parametrize("change,codes", [
    (lambda a: None, (0, 0, 0, 0)),
    (_set("cache", None), (-2, -2, -2, 0)),
    (_set("batch", None), (-2, -2, -2, 0)),
    (_set("cache.format", 2), (-3, -3, -3, 0)),
    (_set("cache.page_size", 24), (-4, -4, -4, 0)),
    (_set("cache.D", 96), (-4, -4, -4, 0)),
    (_set("cache.pages", None), (-2, -2, -2, 0)),
    (_set("cache.pages", 0x100008), (-2, -2, -2, 0)),
    (_set("cache.bytes", 4 * 16 * 2 * 2 * 4 * 34 - 1), (-2, -2, -2, 0)),
    (_set("batch.q_start", None), (-2, -2, -2, 0)),
    (_set("batch.kv_len", 0x2002), (-2, -2, -2, 0)),
    (_set("batch.table_pages", 0), (-4, -4, -4, 0)),
    (_set("batch.table_stride", 3), (-4, -4, -4, 0)),
    (_set("T", 0), (0, 0, 0, 0)),
    (_set("T", (1 << 26) + 1), (-4, -4, -4, -4)),
    (lambda a: (setattr(a.batch, "table_pages", 0x7fff0000 // 16 + 1), setattr(a.batch, "table_stride", 1 << 28)),
     (-4, -4, -4, 0)),
    (_set("batch.B", 0), (0, 0, 0, 0)),
    (_set("kv", None), (-2, -2, 0, 0)),
    (_set("kv.ptr", 0x200002), (-2, -2, 0, 0)),
    (_set("kv.bytes", 2 * 10 * 128 * 2 - 1), (-2, -2, 0, 0)),
    (_set("kv.token_stride", 4), (-4, -4, 0, 0)),
    (_set("kv.token_stride", -128), (-4, -4, 0, 0)),
    (_set("kv.token_stride", 0), (0, -4, 0, 0)),      # inputs may repeat a row, outputs not
    (_set("kv.head_stride", 1152), (0, -4, 0, 0)),    # heads that overlap
    (_set("q.head_stride", 64), (-4, 0, -4, -4)),
    (_set("q.ptr", None), (-2, 0, -2, -2)),
    (_set("H", 7), (0, 0, -4, 0)),
    (_set("H", 0), (-4, 0, -4, -4)),
    (_set("H", 9), (-2, 0, -4, -2)),                  # one head more than the buffers hold
    (_set("rope", None), (-2, 0, 0, -2)),
    (_set("rope.pairs", 12), (-4, 0, 0, -4)),
    (_set("rope.pairs", 72), (-4, 0, 0, -4)),
    (_set("rope.pairs", 0), (-4, 0, 0, -4)),
    (_set("rope.axes", 0), (-4, 0, 0, -4)),
    (_set("rope.axes", 257), (-4, 0, 0, -4)),
    (_set("rope.table", None), (-2, 0, 0, -2)),
    (_set("rope.table", 0x500008), (-2, 0, 0, -2)),
    (_set("rope.table_bytes", 64 * 12 - 1), (-2, 0, 0, -2)),
    (_set("positions", None), (-2, 0, 0, -2)),
    (_set("positions", 0x4002), (-2, 0, 0, -2)),
    (_set("stride", 9), (-4, 0, 0, -4)),
    (_set("scale", float("nan")), (0, 0, -4, 0)),
    (_set("scale", float("inf")), (0, 0, -4, 0)),
    (_set("ws", None), (0, 0, -2, 0)),
    (_set("ws", 0x400008), (0, 0, -2, 0)),
    (_set("ws_bytes", 100), (0, 0, -2, 0)),
], ids=lambda c: getattr(c, "__name__", "") if callable(c) else "")
def test_refusals(lib, change, codes):
    a = Args()
    change(a)
    assert a.codes(lib) == codes


def test_rotary_table(lib):
    """Turns as 64-bit fractions, whole turns dropped; frequencies and axes that are refused."""
    f = [1.0, -1.0, 2 * np.pi * 3.25, 0.0, 1e-30, -1e-30, 100.0, 2 * np.pi]
    axes = [0, 1, 2, 0, 1, 2, 0, 1]

    def table(f, axes, n=8, na=3):
        out = np.zeros(12, np.uint64)
        rc = lib.m4_bridge_rope_axes_table((ctypes.c_double * 8)(*f), (ctypes.c_uint8 * 8)(*axes), n, na, out.ctypes.data)
        return rc, out

    rc, out = table(f, axes)
    assert rc == 0 and list(out[8:].view(np.uint32)) == axes
    want = np.array(f) / (2 * np.pi)
    turns = out[:8].astype(np.float64) / 2.0 ** 64
    off = np.abs(turns - want)
    assert (np.abs(off - np.round(off)) <= 2.0 ** -51 * np.maximum(np.abs(want), 1)).all()  # double: product and floor
    assert table([float("inf")] + f[1:], axes)[0] == -4
    assert table(f, [3] + axes[1:])[0] == -4
    assert table(f, axes, n=4)[0] == -4 and table(f, axes, n=0)[0] == -4 and table(f, axes, na=0)[0] == -4
    assert lib.m4_bridge_rope_axes_table(None, None, 8, 3, None) == -2


def test_positions_default_to_the_place(lib):
    a = Args()
    a.rope.axes = 1
    a.positions = None
    assert a.codes(lib) == (0, 0, 0, -2)  # a rotation alone has no places to stand in


def test_uninitialized_bridge_refuses(lib):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    a, r = Args(), ctypes.addressof
    assert lib.m4_bridge_rope_axes(r(a.rope), 0x4000, 10, r(a.q), r(a.q), 10, 8, 128) == -1
    assert lib.m4_bridge_kv_cache_append(r(a.cache), r(a.batch), 10, r(a.kv), r(a.kv), None, None, 0, None, None, 0) == -1
    assert lib.m4_bridge_kv_cache_read(r(a.cache), r(a.batch), 10, r(a.kv), r(a.kv)) == -1
    assert lib.m4_bridge_paged_layer(*[0x600000] * 11, r(a.cache), r(a.batch), 10, None, None, 0, 0, 256, 8, 512, 0.1, 0, 1,
                                     1e-5) == -1
    assert lib.m4_bridge_dispatch_paged_attn(r(a.cache), r(a.batch), 10, r(a.q), r(a.q), 8, 0.1, 0, 0x400000, 1 << 30) == -1


@pytest.mark.parametrize("change", [_set("cache.page_size", 0xffffffff), _set("cache.page_size", 24), _set("cache.D", 32),
                                    _set("cache.Hkv", 3), _set("cache.format", 1), _set("H", 0), _set("H", 1 << 16)])
def test_no_workspace_for_what_is_refused(lib, change):
    a = Args()
    assert lib.m4_bridge_paged_attn_workspace(ctypes.addressof(a.cache), ctypes.addressof(a.batch), a.T, a.H, 0) > 0
    change(a)
    assert lib.m4_bridge_paged_attn_workspace(ctypes.addressof(a.cache), ctypes.addressof(a.batch), a.T, a.H, 0) == 0


def test_python_refusals(libpath):
    import torch

    b = m4_bridge.HIPBridge.get_instance(libpath)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        m4_bridge.PagedKVCache(3, 4, 16, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        m4_bridge.PagedKVCache(Q8_0, 4, 16, 2, 128, pages=torch.zeros(10, dtype=torch.uint8))
    cache = m4_bridge.PagedKVCache(Q8_0, 4, 16, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        m4_bridge.KVBatch(i32(2), i32(2), i32(2, 4), 1, 1)
    with pytest.raises(ValueError):
        m4_bridge.KVBatch(i32(3).long(), i32(2), i32(2, 4), 1, 1)
    batch = m4_bridge.KVBatch(i32(3), i32(2), i32(2, 4), 1, 1)
    for kw in ({"dims": 24}, {"dims": 320}, {"dims": 64, "sections": (8, 8)}, {"dims": 64, "inv_freq": [1.0]},
               {"dims": 64, "theta": 0.0}, {"dims": 64, "sections": (32,), "pair_axes": [0] * 32}):
        with pytest.raises(ValueError):
            m4_bridge.RotaryAxes(**kw)
    kv = torch.zeros(2, 3, 128, dtype=torch.float16)
    for K, V, kw in ((kv.float(), kv, {}), (kv, kv[:, :2], {}), (kv[:1], kv, {}), (kv, kv, {"Q": kv}), (kv, kv, {"Q_out": kv})):
        with pytest.raises(ValueError):
            b.kv_cache_append(cache, batch, K, V, **kw)
    with pytest.raises(ValueError):
        b.kv_cache_read(cache, batch, kv.transpose(1, 2).contiguous().transpose(1, 2), kv)
    with pytest.raises(ValueError):
        b.dispatch_paged_attn(cache, batch, kv, kv[:, :1], 0.1)
    with pytest.raises(ValueError):
        b.rope_axes(kv, kv, m4_bridge.RotaryAxes(128, sections=(16, 24, 24)), i32(3))
    x = torch.zeros(3, 256, dtype=torch.float16)
    with pytest.raises(ValueError):
        b.paged_layer(x, None, *[x] * 4, None, *[x] * 3, x.clone(), 0, 256, 2, 512, 0.1, cache, batch, window=-1)


@gpu
@pytest.mark.parametrize("change,code", [
    ({"fmt": 9}, -3), ({"norm_type": 3}, -3), ({"Hq": 3}, -4), ({"dm": 100}, -4), ({"Nm": 0}, -4), ({"cache_fmt": 1}, -3),
    ({"ptr": None}, -2), ({"ptr": 8}, -2), ({"B": 0}, 0),
])
def test_paged_layer_refusals(bridge, change, code):
    import torch

    v = {"fmt": 0, "norm_type": 1, "Hq": 4, "dm": 256, "Nm": 512, "cache_fmt": 6, "ptr": 0, "B": 2, **change}
    lib, a = bridge.lib, Args()
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    a.cache.pages, a.cache.format = buf.data_ptr(), v["cache_fmt"]
    a.batch.q_start = a.batch.kv_len = a.batch.page_table = buf.data_ptr()
    a.batch.B = v["B"]
    x = None if v["ptr"] is None else buf.data_ptr() + v["ptr"]
    r = ctypes.addressof
    # a well-formed call is not made here: B = 0 is the only one that passes
    assert lib.m4_bridge_paged_layer(x, *[buf.data_ptr() + 512] * 9, buf.data_ptr() + 1024, r(a.cache), r(a.batch), 10,
                                     None, None, 0, v["fmt"],
                                     v["dm"], v["Hq"], v["Nm"], 0.1, 0, v["norm_type"], 1e-5) == code
    bridge.synchronize()


@gpu
def test_host_memory_is_refused(bridge):
    """These entry points stage nothing: -2, nothing launched, and the next call works."""
    import torch

    s = Setup(Q8_0, [20], [2], 2, 64, 16, seed=31)
    cache, batch = s.cache(), s.batch()
    q = half(s.rng, 4, 2, 64)
    with pytest.raises(RuntimeError, match="-2"):
        bridge.dispatch_paged_attn(cache, batch, torch.from_numpy(q), torch.empty(4, 2, 64, dtype=torch.float16), 0.1,
                                   workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    assert "device" in bridge.last_error()
    host = m4_bridge.KVBatch(torch.from_numpy(s.q_start), torch.tensor([20], dtype=torch.int32), torch.from_numpy(s.table), 2, 20)
    with pytest.raises(RuntimeError, match="-2"):
        bridge.kv_cache_read(cache, host, dev(np.zeros((2, 2, 64), np.float16)), dev(np.zeros((2, 2, 64), np.float16)))
    check_attention(bridge, s, 4)
