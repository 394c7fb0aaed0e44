"""The serving operators at the limits of what a batch and its cache may hold.  References and their bounds are those of
paged_reference.py."""
from __future__ import annotations

import numpy as np
import pytest

import m4_bridge
import paged_reference as ref
from paged_reference import Q8_0
from test_paged import FORMATS, Setup, close, dev, half, say

gpu = pytest.mark.gpu

# what is expected of the lengths chooses the kernels: for 8 query heads a KV head, rows alone, chunks alone (no window,
# and rows enough for 16 tokens of each sequence) and sequences of 16 tokens and more on the one, the others on the other
KERNELS = {"rows": {"max_new": 1, "max_kv": 1}, "chunks": {"max_new": 16, "max_kv": 10 ** 8},
           "both": {"max_new": 2 ** 31 - 1, "max_kv": 10 ** 8}}


def takes(bridge, cache, batch, H, T, window):
    """The kernels of a call, by the workspace that they need: of a group of workgroups two row tiles and 32 bytes."""
    D = cache.D
    ws = bridge.paged_attn_workspace(cache, batch, H, T, window)
    tile = lambda rows: 32 + 2 * rows * (D + 2) * 4  # noqa: E731
    few = [a for a in (16, 32) if ws % tile(a) == 0 and ws // tile(a) <= 512]
    if ws % tile(256) == 0 and ws // tile(256) <= 256:
        return "chunks"
    return "rows" if few else "both"


def attend(bridge, s, q, starts, lens, window, kernels):
    """The call's results [H, T, D] over s's cache, for starts and lengths given apart."""
    import torch

    H, T, D = q.shape
    cache = s.cache()
    batch = m4_bridge.KVBatch(dev(np.array(starts, np.int32)), dev(np.array(lens, np.int32)), dev(s.table), **KERNELS[kernels])
    assert takes(bridge, cache, batch, H, T, window) == kernels
    O = torch.full((H, T, D), 6.0, dtype=torch.float16, device="cuda")
    say("paged limits", s.fmt, starts, lens, H, s.Hkv, D, s.P, window, kernels)
    bridge.dispatch_paged_attn(cache, batch, dev(q), O, D ** -0.5, window=window)
    bridge.synchronize()
    return O.cpu().numpy()


# ---- values that are not finite -----------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,kernels,new", [
    (0, "rows", [2, 5, 1]), (0, "rows", [40, 20, 30]), (0, "chunks", [40, 20, 30]), (0, "both", [40, 20, 3]),
    (20, "rows", [2, 5, 1]), (20, "rows", [40, 20, 30]), (20, "both", [40, 20, 3])])
def test_largest_values_stay_with_the_rows_that_see_them(bridge, fmt, D, window, kernels, new):
    """V rows of +-65504, finite in fp16, whose Q8_0 value half(127 half(65504 / 127)) is infinite: rows that see the key
    get what that gives in its dim and finite results in the 31 that share its scale; the others do not notice."""
    s = Setup(fmt, [100, 60, 75], new, 2, D, 16, seed=40)
    big = {0: [(70, 1, 33, 65504), (99, 0, 5, -65504), (83, 1, 2, 65504), (84, 1, 2, -65504)], 1: [(58, 0, D - 1, -65504), (30, 1, 0, 65504)],
           2: [(74, 0, 40, 65504)]}
    for b, places in big.items():
        for p, h, dim, x in places:
            v = half(s.rng, s.Hkv, D)
            v[h, dim] = x
            k = half(s.rng, s.Hkv, D)
            (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
            s.pages.write(s.table[b, p // 16], p % 16, kq, kd, vq, vd)
            s.k[b][:, p], s.v[b][:, p] = ref.values(kq, kd), ref.values(vq, vd)
            assert np.isinf(s.v[b][h, p, dim]) == (fmt == Q8_0)
    q = half(s.rng, 16, s.T, D)
    got = attend(bridge, s, q, s.q_start, s.lens, window, kernels)
    if fmt == Q8_0:  # the last rows of two sequences
        assert (got[:8, s.q_start[3] - 1, 40] == np.inf).all() and (got[:8, s.q_start[2] - 1, D - 1] == -np.inf).all()
    got = np.where(np.isfinite(got), got, np.float16("nan"))  # an infinity or, of two, NaN: taken alike
    close(got, *s.expected(q, window, D ** -0.5), "largest values")


# ---- lengths past the table and starts past the rows ---------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,kernels,new", [
    (0, "rows", [5, 3, 2]), (0, "rows", [40, 3, 30]), (0, "chunks", [40, 3, 30]), (0, "both", [40, 3, 30]),
    (9, "rows", [5, 3, 2]), (37, "rows", [40, 3, 30]), (9, "both", [40, 3, 30]), (37, "both", [40, 3, 30])])
@pytest.mark.parametrize("past", [1, 2, 30, 2 ** 31 - 1 - 160])
def test_lengths_past_the_table(bridge, fmt, D, window, kernels, new, past):
    """A sequence that is longer than its row of the table: its tokens keep their positions, and see those keys of theirs
    that the table holds."""
    s = Setup(fmt, [160, 40, 160], new, 2, D, 16, seed=41)
    assert s.table.shape[1] * 16 == 160
    lens = [160 + past, 40, 160 + min(past, 5)]
    q = half(s.rng, 16, s.T, D)
    got = attend(bridge, s, q, s.q_start, lens, window, kernels)
    for b, (a, n, L) in enumerate(zip(s.q_start, new, lens)):
        want, bound = ref.attention(q[:, a:a + n], s.k[b], s.v[b], L - n, window, D ** -0.5)
        close(got[:, a:a + n], want, bound, f"sequence {b} of {L}")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,kernels", [(0, "rows"), (0, "chunks"), (0, "both"), (9, "rows"), (9, "both")])
@pytest.mark.parametrize("before,past", [(0, 1), (3, 7), (40, 200), (2 ** 31, 2 ** 31 - 1 - 72)])
def test_starts_past_the_rows(bridge, fmt, window, kernels, before, past):
    """Starts below zero and past T stand for rows that a call does not have.  Those that it has keep their positions,
    kv_len less the rows from them to the sequence's end, wherever they are written, read and attended."""
    import torch

    D, P = 64, 16
    s = Setup(fmt, [90, 130, 300], [30, 12, 30], 2, D, P, seed=42)
    starts = [-before, 30, 42, 72 + past]
    first = [60, 118, 300 - 30 - past]  # positions of the first rows that are there
    q = half(s.rng, 16, s.T, D)
    got = attend(bridge, s, q, starts, s.lens, window, kernels)
    for b, (a, n, p0) in enumerate(zip(s.q_start, s.new, first)):
        want, bound = ref.attention(q[:, a:a + n], s.k[b], s.v[b], p0, window, D ** -0.5)
        close(got[:, a:a + n], want, bound, f"sequence {b}")
    cache = s.cache()
    batch = m4_bridge.KVBatch(dev(np.array(starts, np.int32)), dev(np.array(s.lens, np.int32)), dev(s.table), **KERNELS[kernels])
    k, v = half(s.rng, s.T, 2, D), half(s.rng, s.T, 2, D)
    bridge.kv_cache_append(cache, batch, dev(k), dev(v), token_major=True)
    ko, vo = (torch.full((s.T, 2, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    bridge.kv_cache_read(cache, batch, ko, vo, token_major=True)
    bridge.synchronize()
    (kq, kd), (vq, vd) = ref.quantize(fmt, k), ref.quantize(fmt, v)
    ek, ev = np.full((s.T, 2, D), 3, np.float16), np.full((s.T, 2, D), 3, np.float16)
    for b, (a, n, p0) in enumerate(zip(s.q_start, s.new, first)):
        for i in range(n):
            if p0 + i >= 0:
                s.pages.write(s.table[b, (p0 + i) // P], (p0 + i) % P, kq[a + i], kd[a + i], vq[a + i], vd[a + i])
                ek[a + i], ev[a + i] = s.pages.read(s.table[b, (p0 + i) // P], (p0 + i) % P)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), s.pages.raw)
    np.testing.assert_array_equal(ko.cpu().numpy().view(np.uint16), ek.view(np.uint16))
    np.testing.assert_array_equal(vo.cpu().numpy().view(np.uint16), ev.view(np.uint16))


# ---- positions that repeat ------------------------------------------------------------------------------------------

def test_positions_of_all_axes_may_be_one_row(libpath):
    """A stride of 0: every axis reads the same positions.  Other strides below the number of tokens stay refused."""
    import ctypes

    lib, T = m4_bridge.load_library(libpath), 10
    rows = m4_bridge.RowsStruct(0x300000, 8 * T * 128 * 2, 128, T * 128)
    rope = m4_bridge.RopeAxesStruct(64, 3, 0, 0x500000, 64 * 12)
    cache = m4_bridge.KVCacheStruct(0x100000, 4 * 16 * 2 * 2 * 4 * 34, 6, 4, 16, 2, 128)
    batch = m4_bridge.KVBatchStruct(2, 0x1000, 0x2000, 0x3000, 4, 4, 5, 60)
    r = ctypes.addressof
    for stride, code in ((0, 0), (1, -4), (T - 1, -4), (T, 0)):
        assert lib.m4_bridge_validate_rope_axes(r(rope), 0x4000, stride, r(rows), r(rows), T, 8, 128) == code
        assert lib.m4_bridge_validate_kv_cache_append(r(cache), r(batch), T, r(rows), r(rows), r(rope), 0x4000, stride, r(rows),
                                                      r(rows), 8) == code


@gpu
def test_expanded_positions_are_repeated_ones(bridge):
    """Text positions expanded over the axes, as they stand, alone and beside an append."""
    import torch

    s = Setup(Q8_0, [70, 9], [41, 9], 2, 64, 16, seed=43)
    rope = m4_bridge.RotaryAxes(64, sections=(8, 12, 12))
    text = torch.arange(1000, 1000 + s.T, dtype=torch.int32, device="cuda")
    q, k = dev(half(s.rng, 4, s.T, 64)), dev(half(s.rng, 2, s.T, 64))
    results = []
    for positions in (text.expand(3, s.T), text.repeat(3, 1)):
        y, qo, cache = torch.empty_like(q), torch.empty_like(q), s.cache()
        bridge.rope_axes(q, y, rope, positions)
        bridge.kv_cache_append(cache, s.batch(), k, k, rope=rope, positions=positions, Q=q, Q_out=qo)
        bridge.synchronize()
        results.append((y, qo, cache.pages))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*results))
    assert not torch.equal(results[0][0], q)


# ---- what a call holds, and the workspace that it takes ---------------------------------------------------------------

class Launched:
    """The library, but for the calls that need a device, which launch nothing and succeed."""

    def __init__(self, lib):
        self._lib, self.calls = lib, []

    def __getattr__(self, name):
        if name in ("m4_bridge_rope_axes", "m4_bridge_kv_cache_append", "m4_bridge_dispatch_paged_attn", "m4_bridge_paged_layer",
                    "m4_bridge_synchronize"):
            self.calls.append(name)
            return lambda *a: 0
        return getattr(self._lib, name)


@pytest.fixture
def launched(libpath, monkeypatch):
    b = m4_bridge.HIPBridge.get_instance(libpath)
    lib = Launched(b.lib)
    monkeypatch.setattr(b, "_lib", lib)
    monkeypatch.setattr(b, "_in_flight_tensors", [])
    yield b


def host_batch():
    import torch

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return (m4_bridge.PagedKVCache(Q8_0, 4, 16, 2, 64, device="cpu"), m4_bridge.KVBatch(i32(3), i32(2), i32(2, 4), 1, 64))


@pytest.mark.parametrize("call", ["rope_axes", "append", "layer", "attention"])
def test_rotary_tables_and_workspaces_are_held(launched, call):
    """Until synchronize(), as the tensors of a call are: a table or workspace that the caller lets go of while the kernel
    waits would go back to its stream's memory."""
    import weakref

    import torch

    cache, batch = host_batch()
    rope, ws = m4_bridge.RotaryAxes(64), torch.zeros(1 << 20, dtype=torch.uint8)
    x, positions = torch.zeros(2, 3, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    held = weakref.ref(ws if call == "attention" else rope)
    if call == "rope_axes":
        launched.rope_axes(x, x, rope, positions)
    elif call == "append":
        launched.kv_cache_append(cache, batch, x, x, rope=rope)
    elif call == "layer":
        X, W = torch.zeros(3, 256, dtype=torch.float16), torch.zeros(64, dtype=torch.uint8)
        launched.paged_layer(X, None, *[W] * 4, None, *[W] * 3, X.clone(), 0, 256, 2, 512, 0.1, cache, batch, rope)
    else:
        launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.125, workspace=ws)
    assert len(launched.lib.calls) == 1
    del rope, ws
    assert held() is not None
    launched.synchronize()
    assert held() is None


def test_a_workspace_of_the_calls_own_is_not_held(launched):
    """It is torch's memory of the stream that the kernels run on: held, a loop of eager steps would take one a step."""
    import torch

    cache, batch = host_batch()
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.125)
    assert launched.lib.calls == ["m4_bridge_dispatch_paged_attn"]
    (held,) = launched._in_flight_tensors
    assert not any(isinstance(t, torch.Tensor) and t.dtype == torch.uint8 for t in held)


def test_workspaces_that_are_refused(launched):
    """One whose elements share their bytes, or have others' between them: the kernels would write past it or there."""
    import torch

    cache, batch = host_batch()
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    n = launched.paged_attn_workspace(cache, batch, 2, 3)
    assert n > 0
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(2 * n), torch.zeros(4 * n, dtype=torch.uint8)[::2], bytearray(2 * n)):
        with pytest.raises(ValueError, match="workspace"):
            launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.125, workspace=ws)
    assert launched.lib.calls == []
    launched.dispatch_paged_attn(cache, batch, x, x.clone(), 0.125, workspace=torch.zeros(n, dtype=torch.uint8))


# ---- another device -------------------------------------------------------------------------------------------------

@gpu
def test_layers_of_another_device_are_refused(bridge):
    """The layer's scratch is on the device that the bridge was initialized on; the other calls have none of the bridge's."""
    import torch

    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    with torch.cuda.device(1), torch.cuda.stream(torch.cuda.Stream(1)):
        s = Setup(Q8_0, [40], [2], 2, 64, 16, seed=44)
        one = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to("cuda:1")  # noqa: E731
        cache = m4_bridge.PagedKVCache(Q8_0, s.num_pages, 16, 2, 64, pages=one(s.pages.raw))
        batch = m4_bridge.KVBatch(one(s.q_start), one(np.array(s.lens, np.int32)), one(s.table), 2, 40)
        q = half(s.rng, 4, s.T, 64)
        O = torch.empty(4, s.T, 64, dtype=torch.float16, device="cuda:1")
        bridge.dispatch_paged_attn(cache, batch, one(q), O, 0.125)
        bridge.synchronize()
        close(O.cpu().numpy(), *s.expected(q, 0, 0.125), "attention")
        X, W = torch.zeros(2, 256, dtype=torch.float16, device="cuda:1"), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda:1")
        with pytest.raises(RuntimeError, match="-2"):
            bridge.paged_layer(X, None, *[W] * 4, None, *[W] * 3, X.clone(), 0, 256, 4, 512, 0.125, cache, batch)
        assert "initialized" in bridge.last_error()


# ---- batches that the kernel for chunks takes alone ------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,new,H,Hkv,D,P,window,kernels", [
    ([40 + 3 * (i % 50) for i in range(100)], [20 + i % 21 for i in range(100)], 8, 1, 64, 16, 0, "chunks"),  # more than one a lane
    ([40 + 3 * (i % 50) for i in range(100)], [20 + i % 21 for i in range(100)], 8, 1, 64, 16, 25, "both"),
    ([30] * 70, [30 if i % 3 else 0 for i in range(70)], 16, 2, 64, 32, 0, "chunks"),                      # some without rows
    ([3, 200, 10], [40, 30, 20], 16, 2, 64, 16, 0, "chunks"),                                             # rows that see nothing
    ([0, 17, 0], [30, 30, 30], 16, 2, 128, 16, 0, "chunks"),
    ([0, 17, 0], [30, 30, 30], 16, 2, 128, 16, 5, "both"),
    ([100, 0, 300, 8, 25], [40, 0, 60, 0, 25], 8, 1, 128, 64, 0, "chunks"),                                # and none at all
    ([700, 1, 0, 0, 90], [64, 1, 0, 0, 40], 32, 4, 64, 256, 0, "chunks"),
    ([300, 4, 90], [64, 24, 40], 32, 4, 64, 256, 100, "both"),
])
def test_batches_of_chunks(bridge, fmt, lens, new, H, Hkv, D, P, window, kernels):
    """No sequence of these is the rows kernel's: with both, each has the 128 rows a KV head that make a chunk."""
    assert kernels == "chunks" or min(n * H // Hkv for n in new) >= 128
    s = Setup(fmt, lens, new, Hkv, D, P, seed=len(lens) + H)
    q = half(s.rng, H, s.T, D)
    got = attend(bridge, s, q, s.q_start, lens, window, kernels)
    close(got, *s.expected(q, window, D ** -0.5), "chunks")
