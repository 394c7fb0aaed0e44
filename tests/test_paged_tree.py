"""Trees of drafted tokens over the paged cache -- masks and positions from parents, attention under any mask over the new
tokens with the logarithm of each row's sum, the walk that accepts a path, and the move of its tokens -- against plain
implementations in 64 bits, and their refusals."""
from __future__ import annotations

import ctypes
import weakref

import numpy as np
import pytest

import m4_bridge
import paged_reference as ref
from paged_reference import Q4_0, Q8_0
from test_paged import FORMATS, Setup, close, dev, half, say
from test_paged_limits import KERNELS, takes

gpu = pytest.mark.gpu


def i32(*a):
    return np.array(a, np.int32)


# ---- plain implementations ------------------------------------------------------------------------------------------

def rows_of(q_start, kv_len, b, T):
    """(first row, rows, position of the first) that a call has of sequence b."""
    q0 = min(max(int(q_start[b]), 0), T)
    n = max(min(max(int(q_start[b + 1]), 0), T) - q0, 0)
    return q0, n, max(int(kv_len[b]), 0) - (int(q_start[b + 1]) - q0) if n else 0


def ancestors(parents):
    """[n, n] bool: node j is i itself or before it."""
    n = len(parents)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            a[i] = a[p]
        a[i, i] = True
    return a


def words_of(a, words):
    """Bits [n, m] as int32 [n, words]; those past the words are lost."""
    bits = np.zeros((a.shape[0], 32 * words), bool)
    m = min(a.shape[1], 32 * words)
    bits[:, :m] = a[:, :m]
    return np.packbits(bits.reshape(a.shape[0], words, 32), axis=-1, bitorder="little").view(np.int32)[..., 0]


def walk(parents, tokens, targets):
    path = [0]
    while True:
        fits = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == targets[path[-1]]]
        if not fits:
            return path
        path.append(fits[0])


def attend(q, k, v, seen, scale):
    """q [H, n, D] over k, v [Hkv, L, D] where seen [n, L]: (o, bound of o, lse, bound of lse) in float64.  The bound of o is
    paged_reference.attention's, which allows a row's sum 2^-11 too.  lse: scores off by (D + 8) 2^-24 of the sum of
    |q k|, the exponent's factor and sum by 2^-22 of it, exponentials and rescalings 2^-20, their sum (L + 8) 2^-24, the
    logarithm and its parts 2^-22 of what they are."""
    H, n, D = q.shape
    Hkv, L, _ = k.shape
    o, bound, lse, lb = np.zeros((H, n, D)), np.zeros((H, n, D)), np.full((H, n), -np.inf), np.zeros((H, n))
    with np.errstate(all="ignore"):
        for h in range(H):
            kk, vv = k[h // (H // Hkv)].astype(np.float64), v[h // (H // Hkv)].astype(np.float64)
            qq = q[h].astype(np.float64)
            s = np.where(seen, qq @ kk.T * scale, -np.inf)
            a = np.where(seen, np.abs(qq) @ np.abs(kk).T * abs(scale), 0).max(-1, initial=0)
            m = s.max(-1, initial=-np.inf)
            some = np.isfinite(m)
            w = np.where(seen & some[:, None], np.exp(s - np.where(some, m, 0)[:, None]), 0)
            z = w.sum(-1)
            lse[h] = np.where(some, m + np.log(np.where(z > 0, z, 1)), -np.inf)
            w = w / np.where(z > 0, z, 1)[:, None]
            fin = np.where(np.isfinite(vv), vv, 0)
            o[h] = w @ fin
            es = a * ((D + 8) * 2.0 ** -24 + 2.0 ** -22)
            e = (2 * es + 2.0 ** -21)[:, None]
            big, top = w @ np.abs(fin), np.abs(fin).max(0, initial=0)[None, :]
            bound[h] = ((2.0 ** -11 + e) * (big + np.abs(o[h])) + seen.sum(-1, keepdims=True) * 2.0 ** -32 * (top + np.abs(o[h]))
                        + (L + 8) * 2.0 ** -24 * big + 2.0 ** -11 * np.abs(o[h]) + 2.0 ** -25)
            lb[h] = es + 2.0 ** -20 + (L + 8) * 2.0 ** -24 + 2.0 ** -22 * (np.abs(np.where(some, lse[h], 0)) + 8)
            for key in np.nonzero(~np.isfinite(vv).all(-1))[0]:  # a value that is not finite reaches the rows that see it
                o[h][np.ix_(seen[:, key], ~np.isfinite(vv[key]))] = np.nan
    return o, bound, lse, lb


def seen_of(first, n, L, bits, places, window):
    """Which of L keys the n rows see: the keys before `first` and, of the new ones, their bits; by position the last
    `window` of them."""
    new = np.zeros((n, max(L - first, 0)), bool)
    m = min(new.shape[1], bits.shape[1], n)
    new[:, :m] = bits[:, :m]
    seen = np.concatenate([np.ones((n, max(first, 0)), bool), new[:, max(-first, 0):]], 1)[:, :L]
    if window:
        at = np.clip(places.astype(np.int64), first, first + n - 1)
        key = np.arange(L, dtype=np.int64)
        inside = (key >= first) & (key < first + n)
        key[inside] = at[key[inside] - first]
        seen &= key[None, :] > at[:, None] - window
    return seen


class Trees(Setup):
    """Setup with masks over the new tokens: `kind` "tree" (random parents), "any" (random bits), "none" (no bits)."""

    def masks(self, kind, extra=0):
        self.words = -(-max(self.new) // 32) + extra
        self.bits, places = [], []
        for L, n in zip(self.lens, self.new):
            if kind == "tree":
                bits = ancestors([-1] + [int(self.rng.integers(max(0, i - 6), i)) for i in range(1, n)][:max(n - 1, 0)] if n else [])
            else:
                bits = self.rng.random((n, n)) < (0.4 if kind == "any" else 0)
            self.bits.append(bits)
            places.append(L - n + np.maximum(bits.sum(-1) - 1, 0))
        self.places = np.concatenate(places).astype(np.int32)
        self.mask = np.concatenate([words_of(b, self.words) for b in self.bits]) if self.T else np.zeros((0, self.words), np.int32)
        return m4_bridge.DraftTree(dev(self.mask), dev(self.places))

    def want(self, q, window, scale):
        parts = []
        for a, n, L, k, v, bits in zip(self.q_start, self.new, self.lens, self.k, self.v, self.bits):
            seen = seen_of(L - n, n, L, bits, self.places[a:a + n], window)
            parts.append(attend(q[:, a:a + n], k, v, seen, scale))
        return [np.concatenate(x, 1) for x in zip(*parts)]


# ---- masks and positions --------------------------------------------------------------------------------------------

def random_parents(rng, n, back):
    return [-1] + [int(rng.integers(max(0, i - back), i)) for i in range(1, n)] if n else []


@gpu
@pytest.mark.parametrize("sizes,back,words", [
    ([1], 1, 1), ([0, 1, 2, 0, 5], 3, 1), ([64, 63, 33, 32, 31], 8, 2), ([65, 128, 129, 1], 4, 5), ([300, 64], 1000, 10),
    ([700, 3], 1, 22),                       # a chain, and
    ([200, 130], 5, 2),                      # more nodes than a mask has bits
    ([40, 70], 9, 7),                        # more words than nodes
    ([3] * 130, 3, 1),
])
def test_draft_tree(bridge, sizes, back, words):
    import torch

    rng = np.random.default_rng(sum(sizes) + words)
    parents = [random_parents(rng, n, back) for n in sizes]
    for p in parents:  # parents that are none: the node itself, a later one, numbers that are no nodes
        for i, bad in zip(rng.integers(0, max(len(p), 1), 3), (10 ** 6, -9, None)):
            if len(p) > 20:
                p[i] = int(i) if bad is None else bad
    T, pad = sum(sizes), 3
    q_start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    kv_len = rng.integers(0, 5000, len(sizes)).astype(np.int32)
    tree = m4_bridge.DraftTree(torch.full((T + pad, words), 77, dtype=torch.int32, device="cuda"),
                               torch.full((T + pad,), 77, dtype=torch.int32, device="cuda"))
    batch = m4_bridge.KVBatch(dev(q_start), dev(kv_len), dev(np.zeros((len(sizes), 1), np.int32)), 1, 1)
    say("draft_tree", sizes[:4], back, words)
    bridge.draft_tree(batch, dev(np.array(sum(parents, []) + [0] * pad, np.int32)), tree)
    bridge.synchronize()
    a = [ancestors(p) for p in parents]
    mask = np.concatenate([words_of(x, words) for x in a] + [np.full((pad, words), 77, np.int32)])
    places = np.concatenate([L - n + x.sum(-1) - 1 for L, n, x in zip(kv_len, sizes, a)] + [np.full(pad, 77)])
    np.testing.assert_array_equal(tree.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(tree.positions.cpu().numpy(), places)


@gpu
@pytest.mark.parametrize("sizes,back,words", [
    ([2048, 70], 3, 64), ([2049, 70], 3, 65), ([2047, 2050], 5000, 65),  # about the most whose words are held together
    ([2048], 1, 3), ([3000], 1, 3), ([1000], 2, 0x41), ([2100], 2, 0x61),
])
def test_draft_tree_of_many_nodes(bridge, sizes, back, words):
    test_draft_tree(bridge, sizes, back, words)


@gpu
@pytest.mark.parametrize("starts", [(-3, 4, 9), (0, 2, 40), (-2 ** 31, 3, 2 ** 31 - 1), (5, 3, 7), (9, 9, 9)])
def test_rows_that_a_call_has_are_the_nodes(bridge, starts):
    """Starts below zero and past the rows: the nodes are the rows there are, from the first of them on; a sequence whose
    end comes before its start has none."""
    import torch

    T, rng = 9, np.random.default_rng(3)
    parents, kv_len = i32(-1, 0, 1, 0, 2, 0, 1, 3, 0), i32(20, -7)
    tree = m4_bridge.DraftTree(torch.full((T, 1), 5, dtype=torch.int32, device="cuda"), torch.full((T,), 5, dtype=torch.int32, device="cuda"))
    batch = m4_bridge.KVBatch(dev(i32(*starts)), dev(kv_len), dev(np.zeros((2, 1), np.int32)), 1, 1)
    tokens, targets = rng.integers(0, 2, T).astype(np.int32), rng.integers(0, 2, T).astype(np.int32)
    path, count, nxt = (torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (T, 2, 2))
    say("rows of", starts)
    bridge.draft_tree(batch, dev(parents), tree)
    bridge.tree_accept(batch, dev(parents), dev(tokens), dev(targets), path, count, nxt)
    bridge.synchronize()
    mask, places, want = np.full((T, 1), 5, np.int32), np.full(T, 5), np.full(T, 9)
    for b in range(2):
        q0, n, first = rows_of(starts, kv_len, b, T)
        a = ancestors(parents[q0:q0 + n])
        mask[q0:q0 + n] = words_of(a, 1)
        places[q0:q0 + n] = first + a.sum(-1) - 1
        p = walk(parents[q0:q0 + n], tokens[q0:q0 + n], targets[q0:q0 + n]) if n else []
        want[q0:q0 + n] = p + [-1] * (n - len(p))
        assert int(count[b]) == len(p) and int(nxt[b]) == (targets[q0 + p[-1]] if p else -1)
    np.testing.assert_array_equal(tree.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(tree.positions.cpu().numpy(), places)
    np.testing.assert_array_equal(path.cpu().numpy(), want)


# ---- attention ------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind,window", [("tree", 0), ("any", 0), ("none", 0), ("tree", 9), ("any", 40)])
@pytest.mark.parametrize("lens,new,H,Hkv,D,P,kernels", [
    ([1], [1], 1, 1, 64, 16, "rows"),
    ([1000], [16], 32, 8, 128, 16, "rows"),
    ([70, 3, 0, 700, 33], [5, 3, 0, 1, 33], 8, 2, 64, 16, "rows"),       # no keys before the tree, none at all
    ([260, 131], [61, 100], 6, 2, 128, 64, "rows"),                       # words and key tiles at odd places
    ([90, 200, 64], [40, 70, 64], 16, 2, 64, 32, "chunks"),
    ([500, 40], [130, 40], 16, 2, 128, 256, "chunks"),
    ([300, 65, 900], [40, 3, 90], 16, 2, 128, 16, "both"),
])
def test_tree_attention(bridge, fmt, kind, window, lens, new, H, Hkv, D, P, kernels):
    import torch

    if window and kernels == "chunks":
        kernels = "both"  # what chooses the chunk kernel alone leaves windows out
    s = Trees(fmt, lens, new, Hkv, D, P, seed=len(lens) * 100 + window)
    tree = s.masks(kind)
    q = half(s.rng, H, s.T, D)
    cache = s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **KERNELS[kernels])
    if kernels != "rows":
        assert takes(bridge, cache, batch, H, s.T, window) == kernels
    O = torch.full((H, s.T, D), 6.0, dtype=torch.float16, device="cuda")
    lse = torch.full((s.T, H + 1), 6.0, device="cuda")
    say("tree attention", fmt, kind, window, lens, new, H, Hkv, D, P, kernels)
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, D ** -0.5, window=window, tree=tree, lse=lse[:, :H].T)
    bridge.synchronize()
    o, ob, z, zb = s.want(q, window, D ** -0.5)
    close(O.cpu().numpy(), o, ob, "o")
    got = lse.cpu().numpy().astype(np.float64)
    assert (got[:, H] == 6).all()
    got = got[:, :H].T
    assert (np.isneginf(got) == np.isneginf(z)).all()
    close(np.where(np.isneginf(z), 0, got), np.where(np.isneginf(z), 0, z), zb, "lse")
    # again: the same bits, into other strides, from token-major rows, without lse
    again = torch.zeros((s.T, H, D), dtype=torch.float16, device="cuda")
    bridge.dispatch_paged_attn(cache, batch, dev(q.transpose(1, 0, 2)), again, D ** -0.5, window=window, token_major=True,
                               o_token_major=True, tree=tree)
    bridge.synchronize()
    assert torch.equal(again.transpose(0, 1).contiguous().view(torch.int16), O.view(torch.int16))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,kernels,new", [(0, "rows", [5, 1, 30]), (0, "chunks", [40, 20, 30]), (13, "both", [40, 3, 30])])
def test_lse_beside_causal_attention(bridge, fmt, window, kernels, new):
    """Without a tree rows see up to themselves, and the lower triangle as a mask is the same, bit for bit."""
    import torch

    s = Trees(fmt, [100, 60, 75], new, 2, 64, 16, seed=8)
    s.masks("tree")
    s.bits = [np.tril(np.ones((n, n), bool)) for n in new]
    s.places = np.concatenate([np.arange(L - n, L) for L, n in zip(s.lens, new)]).astype(np.int32)
    q, cache = half(s.rng, 16, s.T, 64), s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(s.lens, np.int32)), dev(s.table), **KERNELS[kernels])
    lower = m4_bridge.DraftTree(dev(np.concatenate([words_of(b, s.words) for b in s.bits])), dev(s.places))
    got = []
    say("lse", fmt, window, kernels, new)
    for tree in (None, lower):
        O, lse = torch.zeros(16, s.T, 64, dtype=torch.float16, device="cuda"), torch.zeros(16, s.T, device="cuda")
        bridge.dispatch_paged_attn(cache, batch, dev(q), O, -0.125, window=window, tree=tree, lse=lse)  # a negative scale too
        bridge.synchronize()
        got.append((O.cpu().numpy(), lse.cpu().numpy()))
    o, ob, z, zb = s.want(q, window, -0.125)
    close(got[0][0], o, ob, "o")
    close(got[0][1], z, zb, "lse")
    if kernels == "rows":  # chunks take the tree's keys as far as any row may see
        assert (got[0][0].view(np.uint16) == got[1][0].view(np.uint16)).all() and (got[0][1] == got[1][1]).all()
    else:
        close(got[1][0], o, ob, "o of a mask")
        close(got[1][1], z, zb, "lse of a mask")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kernels,new", [("rows", [2, 5, 1]), ("rows", [40, 20, 30]), ("chunks", [40, 20, 30]), ("both", [40, 20, 3])])
def test_largest_values_stay_with_the_rows_whose_bits_say_so(bridge, fmt, kernels, new):
    """V rows of +-65504 (infinite in Q8_0) among the nodes: rows without the node's bit do not notice."""
    import torch

    s = Trees(fmt, [100, 60, 75], new, 2, 64, 16, seed=40)
    tree = s.masks("any")
    for b, (L, n) in enumerate(zip(s.lens, new)):
        for p, h, dim, x in ((L - n, 1, 33, 65504), (L - 1, 0, 5, -65504), (L - n // 2 - 1, 1, 2, 65504), (L - n - 3, 0, 9, 65504)):
            v, k = half(s.rng, 2, 64), half(s.rng, 2, 64)
            v[h, dim] = x
            (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
            s.pages.write(s.table[b, p // 16], p % 16, kq, kd, vq, vd)
            s.k[b][:, p], s.v[b][:, p] = ref.values(kq, kd), ref.values(vq, vd)
    q, cache = half(s.rng, 16, s.T, 64), s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(s.lens, np.int32)), dev(s.table), **KERNELS[kernels])
    O = torch.full((16, s.T, 64), 6.0, dtype=torch.float16, device="cuda")
    say("largest values", fmt, kernels, new)
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, 0.125, tree=tree)
    bridge.synchronize()
    o, ob, _, _ = s.want(q, 0, 0.125)
    got = O.cpu().numpy()
    assert (fmt == Q4_0) or not np.isfinite(got).all()
    close(np.where(np.isfinite(got), got, np.float16("nan")), o, ob, "largest values")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kernels", ["rows", "both"])
def test_masks_and_positions_out_of_range(bridge, fmt, kernels):
    """Bits of nodes that are not there, words for more nodes than there are or fewer, positions that are anything, pages
    that are not there and rows without keys: nothing outside is read, and the rest holds."""
    import torch

    P, H, D = 16, 16, 64
    s = Trees(fmt, [100, 60, 4], [40, 20, 9], 2, D, P, seed=9)  # the last: more rows than keys
    s.masks("any")
    s.words = 1  # nodes 32 .. 39 of the first are seen by none
    mask = np.concatenate([words_of(b, 1) for b in s.bits])
    mask[s.q_start[1]:s.q_start[2]] |= np.int32(-1 << 20)  # nodes 20 .. 31 of the second
    s.bits = [b[:, :32] for b in s.bits]
    s.places = s.rng.integers(-2 ** 31, 2 ** 31, s.T).astype(np.int32)
    s.places[::3] = 77
    table = s.table.copy()
    table[0, 2] = 10 ** 9  # keys 32 .. 47
    table[0, 5] = -1       # keys 80 .. 95, nodes 20 .. 35
    q, cache = half(s.rng, H, s.T, D), s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(s.lens, np.int32)), dev(table), **KERNELS[kernels])
    for window in (0, 50):
        O = torch.full((H, s.T, D), 6.0, dtype=torch.float16, device="cuda")
        say("out of range", fmt, kernels, window)
        bridge.dispatch_paged_attn(cache, batch, dev(q), O, 0.125, window=window, tree=m4_bridge.DraftTree(dev(mask), dev(s.places)))
        bridge.synchronize()
        for b, (a, n, L) in enumerate(zip(s.q_start, s.new, s.lens)):
            seen = seen_of(L - n, n, L, s.bits[b], s.places[a:a + n], window)
            if b == 0:
                seen[:, 32:48] = seen[:, 80:96] = False
            o, ob, _, _ = attend(q[:, a:a + n], s.k[b], s.v[b], seen, 0.125)
            close(O[:, a:a + n].cpu().numpy(), o, ob, f"sequence {b}, window {window}")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,new,kernels", [
    ([40, 9, 33], [5, 9, 1], "rows"), ([900, 333, 2000], [40, 3, 16], "rows"), ([300, 65, 900], [40, 60, 90], "chunks"),
    ([2300, 65, 900], [40, 3, 90], "both")])
def test_weights_of_a_row_are_one_together(bridge, fmt, D, lens, new, kernels):
    """Where all keys of a sequence have one value, that is the result, to the last bit, whatever the weights: what O is
    divided by is the sum of the weights as the product with V took them.  fp32 sums are off by (keys + 8) 2^-24 at most,
    2^-12.8, which is less than half a step of any fp16 value, 2^-12 of it or more, so O's rounding takes it back."""
    import torch

    H, Hkv, P = 16, 2, 16
    s = Trees(fmt, lens, new, Hkv, D, P, seed=len(lens) + D + sum(new))
    tree = s.masks("any")
    value = np.zeros((H, s.T, D), np.float16)
    for b, (L, n, a) in enumerate(zip(lens, new, s.q_start)):
        v = (s.rng.integers(1, 8, (Hkv, D)) * 0.25).astype(np.float16)  # 0.25 .. 1.75
        k = half(s.rng, L, Hkv, D)
        (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
        held = ref.values(vq, vd)
        s.v[b] = np.repeat(held[:, None], L, 1)
        s.k[b] = ref.values(kq, kd).transpose(1, 0, 2)
        for p in range(L):
            s.pages.write(s.table[b, p // P], p % P, kq[p], kd[p], vq, vd)
        value[:, a:a + n] = np.repeat(held, H // Hkv, 0)[:, None]
    q = (3 * half(s.rng, H, s.T, D)).astype(np.float16)
    cache = s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(s.table), **KERNELS[kernels])
    for kw in ({}, {"lse": torch.empty(H, s.T, device="cuda")}, {"tree": tree}, {"tree": tree, "lse": torch.empty(H, s.T, device="cuda")}):
        O = torch.full((H, s.T, D), 6.0, dtype=torch.float16, device="cuda")
        say("one together", fmt, D, lens, new, kernels, sorted(kw))
        bridge.dispatch_paged_attn(cache, batch, dev(q), O, D ** -0.5, **kw)
        bridge.synchronize()
        want = value.copy()
        if "tree" in kw:  # rows that see nothing
            for b, (L, n, a) in enumerate(zip(lens, new, s.q_start)):
                if L == n:
                    want[:, a:a + n][:, s.bits[b].sum(-1) == 0] = 0
        np.testing.assert_array_equal(O.cpu().numpy(), want)


# ---- the accepted path ----------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("sizes,back,vocabulary", [([1], 1, 1), ([0, 1, 2, 26], 4, 2), ([64, 65, 300], 9, 2), ([700], 1, 1), ([5] * 140, 3, 2)])
def test_tree_accept(bridge, sizes, back, vocabulary):
    """Few tokens, so that siblings carry the same one: the lowest node counts.  Parents that are no earlier nodes lead
    nowhere; rows behind the last sequence stay."""
    import torch

    rng = np.random.default_rng(sum(sizes))
    T, pad, B = sum(sizes), 2, len(sizes)
    parents = [random_parents(rng, n, back) for n in sizes]
    for p in parents:
        if len(p) > 20:
            p[7], p[9] = 9, 10 ** 9
    tokens, targets = (rng.integers(0, vocabulary, T + pad).astype(np.int32) for _ in range(2))
    q_start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    batch = m4_bridge.KVBatch(dev(q_start), dev(np.full(B, 10, np.int32)), dev(np.zeros((B, 1), np.int32)), 1, 1)
    path, count, nxt = (torch.full((n,), 99, dtype=torch.int32, device="cuda") for n in (T + pad, B, B))
    bridge.tree_accept(batch, dev(np.array(sum(parents, []) + [0] * pad, np.int32)), dev(tokens), dev(targets), path, count, nxt)
    bridge.synchronize()
    want = np.full(T + pad, 99)
    for b, (a, n) in enumerate(zip(q_start, sizes)):
        p = walk(parents[b], tokens[a:a + n], targets[a:a + n]) if n else []
        want[a:a + n] = p + [-1] * (n - len(p))
        assert int(count[b]) == len(p) and int(nxt[b]) == (targets[a + p[-1]] if p else -1)
    np.testing.assert_array_equal(path.cpu().numpy(), want)


@gpu
def test_calls_without_rows_say_so(bridge):
    """T = 0: every sequence is one without rows, for each of which the header says what it gets."""
    import torch

    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    s = Setup(Q8_0, [40, 0, 60], [0, 0, 0], 2, 64, 16, seed=4)
    lens = dev(i32(40, 0, -3))
    batch = m4_bridge.KVBatch(dev(i32(0, 5, 9, 12)), lens, dev(s.table), 1, 1)
    count, nxt, out = z(3) + 9, z(3) + 9, z(3) + 9
    cache = s.cache()
    bridge.tree_accept(batch, z(0), z(0), z(0), z(0), count, nxt)
    bridge.kv_cache_keep(cache, batch, z(0), count, out)
    bridge.synchronize()
    assert count.tolist() == [0] * 3 and nxt.tolist() == [-1] * 3 and out.tolist() == [40, 0, 0]
    bridge.kv_cache_keep(cache, batch, z(0), count, batch.kv_len)
    bridge.kv_cache_keep(cache, batch, z(0), count)
    bridge.synchronize()
    assert batch.kv_len.tolist() == [40, 0, 0]
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)


def test_refused_without_rows(lib):
    """T = 0 needs nothing of the rows, and takes what it is given to write for the sequences."""
    a, r = Args(), ctypes.addressof
    accept = lambda *p: lib.m4_bridge_validate_tree_accept(r(a.batch), 0, None, None, None, None, *p)  # noqa: E731
    assert accept(0x700000, 0x710000) == 0 and accept(None, None) == 0 and accept(0x700000, None) == 0
    assert accept(0x700001, 0x710000) == -2 and accept(0x700000, 0x710002) == -2
    keep = lambda *p: lib.m4_bridge_validate_kv_cache_keep(r(a.cache), r(a.batch), 0, *p)  # noqa: E731
    assert keep(None, None, None) == 0 and keep(None, None, 0x700000) == 0 and keep(None, None, 0x700002) == -2
    a.batch.kv_len = 0
    assert keep(None, None, None) == 0 and keep(None, None, 0x700000) == -2 and accept(0x700000, 0x710000) == 0
    a.batch.kv_len = 0x2001
    assert keep(None, None, 0x700000) == -2
    a.batch.B = 0
    assert keep(None, None, 0x700000) == 0 and accept(0x700001, None) == 0


def token_bytes(pages, slot):
    """Where a token's bytes lie in a head's share of a page."""
    ak, av, aks, avs = pages._places(slot)
    return np.concatenate([ak, av, aks, aks + 1, avs, avs + 1])


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,Hkv,D,P", [
    ([1], [1], 1, 64, 16), ([300, 0, 17, 65], [33, 0, 1, 26], 8, 128, 16), ([700], [513], 3, 64, 32), ([5, 30], [9, 30], 2, 128, 256),
    ([40] * 66, [7] * 66, 1, 64, 16)])
def test_keep(bridge, fmt, lens, new, Hkv, D, P):
    """Every byte of the pages, and the lengths, written over the batch's own."""
    s = Setup(fmt, lens, new, Hkv, D, P, seed=len(lens) + D)
    keep, count = np.full(s.T, -1, np.int32), np.zeros(len(lens), np.int32)
    table = s.table.copy()
    if len(lens) == 4:
        table[3, 3] = 10 ** 8  # keys 48 .. 63
        table[0, 0] = -1
    raw, want = s.pages.raw.copy(), s.pages.raw.copy()
    for b, (L, n, a) in enumerate(zip(lens, new, s.q_start)):
        m = int(s.rng.integers(0, n + 1)) if n > 1 else n
        chosen = np.sort(s.rng.permutation(n)[:m])
        keep[a:a + m], count[b] = chosen, m
        for i, node in enumerate(chosen):
            src, dst = L - n + int(node), L - n + i
            if src < 0 or dst < 0:
                continue
            sp, dp = table[b, src // P], table[b, dst // P]
            if 0 <= sp < s.num_pages and 0 <= dp < s.num_pages:
                want[dp][:, token_bytes(s.pages, dst % P)] = raw[sp][:, token_bytes(s.pages, src % P)]
    cache = s.cache()
    batch = m4_bridge.KVBatch(dev(s.q_start), dev(np.array(lens, np.int32)), dev(table), 1, 1)
    say("keep", fmt, lens[:4], new[:4], Hkv, D, P)
    bridge.kv_cache_keep(cache, batch, dev(keep), dev(count), batch.kv_len)
    bridge.synchronize()
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), want)
    first = [L - n for L, n in zip(lens, new)]
    np.testing.assert_array_equal(batch.kv_len.cpu().numpy(), [max(f + int(m), 0) if n else L for f, m, n, L in zip(first, count, new, lens)])


@gpu
def test_keep_of_lists_that_are_none(bridge):
    """Counts past the rows or below zero, numbers that are no nodes, no lengths wanted; lists that fall move tokens
    among the sequence's own places only."""
    s = Setup(Q8_0, [40, 50, 60], [10, 10, 10], 2, 64, 16, seed=4)
    keep = np.concatenate([[0, 1, 10 ** 6, -4, 9] + [0] * 5, np.arange(10), np.arange(9, -1, -1)]).astype(np.int32)
    cache = s.cache()
    bridge.kv_cache_keep(cache, s.batch(), dev(keep), dev(i32(5, -3, 10 ** 9)))
    bridge.synchronize()
    got, want = cache.pages.cpu().numpy(), s.pages.raw.copy()
    at = lambda b, p: (s.table[b, p // 16], token_bytes(s.pages, p % 16))  # noqa: E731
    (sp, sb), (dp, db) = at(0, 39), at(0, 34)
    want[dp][:, db] = s.pages.raw[sp][:, sb]
    for p in range(50, 60):  # the falling list's own places
        page, b = at(2, p)
        got[page][:, b] = want[page][:, b]
    np.testing.assert_array_equal(got, want)


# ---- a step as it is used -------------------------------------------------------------------------------------------

class Step:
    """One step with a tree over two sequences, everything on the device."""

    def __init__(self, bridge, seed, fmt=Q8_0):
        import torch

        self.b, self.s = bridge, Setup(fmt, [70, 33], [0, 0], 2, 64, 16, seed=seed)
        self.n, T = [20, 37], 57
        r = self.s.rng
        self.parents = [random_parents(r, n, 5) for n in self.n]
        self.q, self.k, self.v = half(r, 8, T, 64), half(r, 2, T, 64), half(r, 2, T, 64)
        self.tokens, self.targets = r.integers(0, 3, T).astype(np.int32), r.integers(0, 3, T).astype(np.int32)
        self.table = np.arange(2 * 8, dtype=np.int32).reshape(2, 8)
        self.pages = ref.Pages(fmt, 16, 16, 2, 64)
        for b, L in enumerate(self.s.lens):
            for p in range(L):
                self.pages.write(self.table[b, p // 16], p % 16, *ref.quantize(fmt, half(r, 2, 64)), *ref.quantize(fmt, half(r, 2, 64)))
        self.rope = m4_bridge.RotaryAxes(64, theta=1e4)
        self.cache = m4_bridge.PagedKVCache(fmt, 16, 16, 2, 64, pages=dev(self.pages.raw))
        self.batch = m4_bridge.KVBatch(dev(i32(0, 20, 57)), dev(i32(90, 70)), dev(self.table), 37, 90)
        self.tree = m4_bridge.DraftTree.empty(T, 37)
        self.t = {n: dev(a) for n, a in (("q", self.q), ("k", self.k), ("v", self.v), ("tokens", self.tokens), ("targets", self.targets),
                                         ("parents", np.array(sum(self.parents, []), np.int32)))}
        new = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)  # noqa: E731
        self.o, self.lse, self.qo = new(8, T, 64, dtype=torch.float16), new(8, T), new(8, T, 64, dtype=torch.float16)
        self.path, self.count, self.next = (new(x, dtype=torch.int32) for x in (T, 2, 2))
        self.ws = new(bridge.paged_attn_workspace(self.cache, self.batch, 8, T), dtype=torch.uint8)

    def run(self):
        b, t = self.b, self.t
        b.draft_tree(self.batch, t["parents"], self.tree)
        b.kv_cache_append(self.cache, self.batch, t["k"], t["v"], rope=self.rope, positions=self.tree.positions, Q=t["q"], Q_out=self.qo)
        b.dispatch_paged_attn(self.cache, self.batch, self.qo, self.o, 0.125, workspace=self.ws, tree=self.tree, lse=self.lse)
        b.tree_accept(self.batch, t["parents"], t["tokens"], t["targets"], self.path, self.count, self.next)
        b.kv_cache_keep(self.cache, self.batch, self.path, self.count, self.batch.kv_len)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_step_with_a_tree_is_one_with_its_path(bridge, fmt):
    """Along the accepted path, the tree's rows and the cache that it leaves are those of the same tokens as a chain."""
    import torch

    x = Step(bridge, 21, fmt)
    x.run()
    bridge.synchronize()
    path, count = x.path.cpu().numpy(), x.count.cpu().numpy()
    assert (count >= 2).any()
    np.testing.assert_array_equal(x.batch.kv_len.cpu().numpy(), [70 + count[0], 33 + count[1]])
    rows = np.concatenate([path[:count[0]], 20 + path[20:20 + count[1]]])
    chain = m4_bridge.PagedKVCache(fmt, 16, 16, 2, 64, pages=dev(x.pages.raw))
    batch = m4_bridge.KVBatch(dev(i32(0, count[0], count.sum())), x.batch.kv_len, x.batch.page_table, 37, 90)
    q = dev(x.q[:, rows])
    bridge.kv_cache_append(chain, batch, dev(x.k[:, rows]), dev(x.v[:, rows]), rope=x.rope, Q=q)
    O, lse = torch.zeros_like(q), torch.zeros(8, len(rows), device="cuda")
    bridge.dispatch_paged_attn(chain, batch, q, O, 0.125, lse=lse)
    both = []
    for cache in (x.cache, chain):  # the rows that each cache now holds
        k, v = torch.zeros(2, int(count.sum()), 64, dtype=torch.float16, device="cuda"), torch.zeros(2, int(count.sum()), 64, dtype=torch.float16, device="cuda")
        bridge.kv_cache_read(cache, batch, k, v)
        both.append((k, v))
    bridge.synchronize()
    assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[1][1])
    # both calls are off a row's result by at most 2^-11 of sum w |v|, |o| and their rounding each; |v| is at most 5
    assert float((x.o[:, rows].float() - O.float()).abs().max()) <= 2 * (3 * 2.0 ** -11 * 5)
    assert float((x.lse[:, rows] - lse).abs().max()) <= 2.0 ** -15


@gpu
def test_a_step_in_a_graph(bridge):
    """Captured once and replayed with what is written to its tensors, between eager work."""
    import torch

    eager, x = Step(bridge, 30), Step(bridge, 30)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            x.run()
    for turn in range(4):
        rng = np.random.default_rng(turn)
        lens = i32(90 + turn, 70 - 7 * turn)
        parents = np.array(sum([random_parents(rng, n, 2 + turn) for n in x.n], []), np.int32)
        tokens, q = rng.integers(0, 2, 57).astype(np.int32), half(rng, 8, 57, 64)
        for y in (eager, x):
            y.batch.kv_len.copy_(dev(lens))
            y.t["parents"].copy_(dev(parents))
            y.t["tokens"].copy_(dev(tokens))
            y.t["q"].copy_(dev(q))
            y.cache.pages.copy_(dev(x.pages.raw))
        eager.run()
        bridge.synchronize()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in ("o", "lse", "path", "count", "next"):  # bit for bit: a row may see keys that nobody wrote
            assert torch.equal(getattr(x, n).view(torch.uint8), getattr(eager, n).view(torch.uint8)), (turn, n)
        assert torch.equal(x.batch.kv_len, eager.batch.kv_len) and torch.equal(x.cache.pages, eager.cache.pages)
        assert torch.equal(x.tree.mask, eager.tree.mask) and torch.equal(x.tree.positions, eager.tree.positions)


# ---- refusals -------------------------------------------------------------------------------------------------------

class Args:
    """Valid arguments without a device, changed one at a time."""

    def __init__(self):
        self.cache = m4_bridge.KVCacheStruct(0x100000, 4 * 16 * 2 * 2 * 4 * 34, 6, 4, 16, 2, 128)
        self.batch = m4_bridge.KVBatchStruct(2, 0x1000, 0x2000, 0x3000, 4, 4, 5, 60)
        self.rows = m4_bridge.RowsStruct(0x300000, 10 * 8 * 128 * 2, 128, 10 * 128)
        self.lse = m4_bridge.RowsStruct(0x400000, 10 * 8 * 4, 1, 10)
        self.tree = m4_bridge.DraftTreeStruct(0x500000, 10 * 4, 0x600000, 10 * 4, 1)
        self.T, self.H, self.window, self.scale = 10, 8, 0, 0.1


@pytest.fixture
def lib(libpath):
    return m4_bridge.load_library(libpath)


def set_(path, value):
    def change(a):
        o = a
        for n in path.split(".")[:-1]:
            o = getattr(o, n)
        setattr(o, path.split(".")[-1], value)
    return change


@pytest.mark.parametrize("change,code", [
    (lambda a: None, 0), (set_("tree.mask", 0), -2), (set_("tree.mask", 0x500002), -2), (set_("tree.mask_bytes", 39), -2),
    (set_("tree.words", 0), -4), (set_("tree.words", 2 ** 21 + 1), -4), (set_("tree.words", 2), -2), (set_("tree.positions", 0x600001), -2),
    (set_("T", 2 ** 26 + 1), -4), (set_("batch.B", 2 ** 31), -4), (set_("batch.q_start", 0), -2), (set_("batch.kv_len", 0x2001), -2),
    (set_("batch.B", 0), 0), (set_("T", 0), 0)])
def test_refused_trees(lib, change, code):
    a, r = Args(), ctypes.addressof
    change(a)
    assert lib.m4_bridge_validate_draft_tree(r(a.batch), a.T, 0x700000, r(a.tree)) == code
    if code == 0:
        assert lib.m4_bridge_validate_draft_tree(r(a.batch), a.T, None, r(a.tree)) == (0 if a.T == 0 or a.batch.B == 0 else -2)
    assert lib.m4_bridge_validate_draft_tree(None, a.T, 0x700000, r(a.tree)) == -2
    assert lib.m4_bridge_validate_draft_tree(r(a.batch), 10, 0x700000, None) == (-4 if a.batch.B > 2 else 0 if a.batch.B == 0 else -2)


def test_refused_positions(lib):
    """Filled, they have to be there; attended, with a window."""
    a, r = Args(), ctypes.addressof
    for at, size in ((0, 0), (0x600000, 39)):
        a.tree.positions, a.tree.positions_bytes = at, size
        assert lib.m4_bridge_validate_draft_tree(r(a.batch), 10, 0x700000, r(a.tree)) == -2
        for window, code in ((0, 0), (5, -2)):
            assert lib.m4_bridge_validate_paged_attn_tree(r(a.cache), r(a.batch), 10, r(a.rows), r(a.rows), 8, 0.1, window, r(a.tree), None,
                                                          0x800000, 1 << 40) == code


@pytest.mark.parametrize("change,code", [
    (lambda a: None, 0), (set_("tree.mask", 0), -2), (set_("tree.mask_bytes", 39), -2), (set_("tree.words", 0), -4), (set_("lse.ptr", 0), -2),
    (set_("lse.ptr", 0x400002), -2), (set_("lse.bytes", 319), -2), (set_("lse.token_stride", -1), -4), (set_("lse.token_stride", 0), -4),
    (set_("lse.head_stride", 9), -4), (set_("lse.head_stride", 2 ** 62), -2), (set_("cache.format", 1), -3), (set_("cache.D", 96), -4),
    (set_("rows.token_stride", 4), -4), (set_("H", 7), -4), (set_("H", 0), -4), (set_("scale", float("nan")), -4), (set_("T", 0), 0)])
def test_refused_attention(lib, change, code):
    a, r = Args(), ctypes.addressof
    change(a)
    call = lambda ws, size: lib.m4_bridge_validate_paged_attn_tree(  # noqa: E731
        r(a.cache), r(a.batch), a.T, r(a.rows), r(a.rows), a.H, a.scale, a.window, r(a.tree), r(a.lse), ws, size)
    assert call(0x800000, 1 << 40) == code
    if code == 0 and a.T:
        need = lib.m4_bridge_paged_attn_workspace(r(a.cache), r(a.batch), a.T, a.H, 0)
        assert call(0x800000, need) == 0 and call(0x800000, need - 1) == -2 and call(None, need) == -2
        assert lib.m4_bridge_validate_paged_attn_tree(r(a.cache), r(a.batch), a.T, r(a.rows), r(a.rows), a.H, a.scale, 7, None, None, 0x800000,
                                                      1 << 40) == 0


def test_refused_paths_and_moves(lib):
    a, r = Args(), ctypes.addressof
    ok = [0x700000, 0x710000, 0x720000, 0x730000, 0x740000, 0x750000]
    assert lib.m4_bridge_validate_tree_accept(r(a.batch), 10, *ok) == 0
    for i in range(6):
        for bad in (None, 0x700001):
            assert lib.m4_bridge_validate_tree_accept(r(a.batch), 10, *ok[:i], bad, *ok[i + 1:]) == -2
    assert lib.m4_bridge_validate_tree_accept(r(a.batch), 0, *[None] * 6) == 0
    keep = lambda *p: lib.m4_bridge_validate_kv_cache_keep(r(a.cache), r(a.batch), 10, *p)  # noqa: E731
    assert keep(0x700000, 0x710000, 0x2000) == 0 and keep(0x700000, 0x710000, None) == 0
    assert keep(None, 0x710000, None) == -2 and keep(0x700000, None, None) == -2 and keep(0x700000, 0x710000, 0x2002) == -2
    a.batch.table_stride = 3
    assert keep(0x700000, 0x710000, None) == -4
    a.cache.page_size = 24
    assert keep(0x700000, 0x710000, None) == -4
    for name in ("draft_tree", "tree_accept", "kv_cache_keep", "dispatch_paged_attn_tree"):
        assert hasattr(lib, "m4_bridge_" + name)


class Launched:
    """The library, but for the calls that need a device, which launch nothing and succeed."""

    def __init__(self, lib):
        self._lib, self.calls = lib, []

    def __getattr__(self, name):
        if name.startswith("m4_bridge_") and "validate" not in name and not name.endswith(("_workspace", "_bytes", "_table")):
            self.calls.append(name)
            return lambda *a: 0
        return getattr(self._lib, name)


@pytest.fixture
def launched(libpath, monkeypatch):
    b = m4_bridge.HIPBridge.get_instance(libpath)
    monkeypatch.setattr(b, "_lib", Launched(b.lib))
    monkeypatch.setattr(b, "_in_flight_tensors", [])
    yield b


def host():
    import torch

    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return m4_bridge.PagedKVCache(Q8_0, 4, 16, 2, 64, device="cpu"), m4_bridge.KVBatch(z(3), z(2), z(2, 4), 1, 64), z


def test_what_a_call_holds_and_refuses(launched):
    """Tensors are held until synchronize(); shapes, types and strides that a call does not take raise."""
    import torch

    cache, batch, z = host()
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    tree = m4_bridge.DraftTree.empty(3, 5, device="cpu")
    lse = torch.zeros(2, 3)
    held = weakref.ref(tree)
    launched.draft_tree(batch, z(3), tree)
    launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.125, tree=tree, lse=lse)
    launched.tree_accept(batch, z(3), z(3), z(3), z(3), z(2), z(2))
    launched.kv_cache_keep(cache, batch, z(3), z(2), batch.kv_len)
    assert [c for c in launched.lib.calls if "stream" not in c] == ["m4_bridge_draft_tree", "m4_bridge_dispatch_paged_attn_tree",
                                                                    "m4_bridge_tree_accept", "m4_bridge_kv_cache_keep"]
    del tree
    assert held() is not None
    launched.synchronize()
    assert held() is None
    n = len(launched.lib.calls)
    tree = m4_bridge.DraftTree.empty(3, 5, device="cpu")
    blind = m4_bridge.DraftTree(z(3, 1))
    for call in (lambda: launched.draft_tree(batch, z(2), tree), lambda: launched.draft_tree(batch, z(3).long(), tree),
                 lambda: launched.draft_tree(batch, z(6)[::2], tree), lambda: launched.draft_tree(batch, z(3), blind),
                 lambda: launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.1, tree=m4_bridge.DraftTree.empty(4, 5, device="cpu")),
                 lambda: launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.1, tree=blind, window=4),
                 lambda: launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.1, lse=lse.half()),
                 lambda: launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.1, lse=lse.T),
                 lambda: launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.1, lse=lse[:, :1].expand(2, 3)),
                 lambda: launched.tree_accept(batch, z(3), z(3), z(3), z(3), z(3), z(2)),
                 lambda: launched.kv_cache_keep(cache, batch, z(3), z(3)), lambda: launched.kv_cache_keep(cache, batch, z(3), z(2), z(1)),
                 lambda: m4_bridge.DraftTree(z(3)), lambda: m4_bridge.DraftTree(z(3, 0)), lambda: m4_bridge.DraftTree(z(3, 2).float()),
                 lambda: m4_bridge.DraftTree(z(3, 4)[:, :2]), lambda: m4_bridge.DraftTree(z(3, 2), z(4))):
        with pytest.raises(ValueError):
            call()
    assert len(launched.lib.calls) == n


@gpu
def test_host_memory_is_refused(bridge):
    """Nothing is staged: a buffer that is not the device's is named and refused."""
    import torch

    cache, batch, z = host()
    s = Setup(Q8_0, [40, 40], [2, 1], 2, 64, 16, seed=2)
    tree = m4_bridge.DraftTree.empty(3, 5)
    with pytest.raises(RuntimeError, match="-2"):
        bridge.draft_tree(s.batch(), z(3), tree)
    assert "device" in bridge.last_error()
    with pytest.raises(RuntimeError, match="-2"):
        bridge.tree_accept(s.batch(), *[z(3).cuda()] * 3, z(3), z(2).cuda(), z(2).cuda())
    with pytest.raises(RuntimeError, match="-2"):
        bridge.kv_cache_keep(s.cache(), s.batch(), z(3).cuda(), z(2))
    x = torch.zeros(2, 3, 64, dtype=torch.float16, device="cuda")
    for kw in ({"lse": torch.zeros(2, 3)}, {"tree": m4_bridge.DraftTree(z(3, 1))}):
        with pytest.raises(RuntimeError, match="-2"):
            bridge.dispatch_paged_attn(s.cache(), s.batch(), x, x.clone(), 0.1, **kw)
    bridge.synchronize()


@gpu
def test_calls_on_two_streams(bridge):
    """Two steps at once, on streams of their own, are as each alone."""
    import torch

    steps = [Step(bridge, 50 + i) for i in range(2)]
    alone = [Step(bridge, 50 + i) for i in range(2)]
    for x in alone:
        x.run()
    bridge.synchronize()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for x, st in zip(steps, streams):
        with torch.cuda.stream(st):
            x.run()
    torch.cuda.synchronize()
    bridge.synchronize()
    for x, y in zip(steps, alone):
        assert torch.equal(x.o, y.o) and torch.equal(x.cache.pages, y.cache.pages) and torch.equal(x.path, y.path)
