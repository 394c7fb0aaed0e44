"""The operators of serving over a paged, quantized KV cache, as data: rotary positions with several axes, quantizing
a cache as it is written and reading it back, and attention of new tokens over it.  From one decoded token to prompts
of thousands, one sequence or many of different lengths.

  own                  False: `run` computes the plain forms (elementary torch operations in 32 bits or more);
                       True: it makes the calls of the bridge
  listed()             the named cases;  draw(rng) one more of the same ranges
  prepare(case, seed)  inputs and cache on the GPU
  run(state)           one pass
  exact(case, seed)    the same results in 64 bits
  work(case)           bytes and operations that a pass cannot do without

A cache page holds, for each KV head, P tokens of D dims as
  K codes [P][D] | V codes [P/4][D][4 tokens] | K scales [P][D/32] fp16 | V scales [P/4][D/32][4 tokens] fp16;
Q8_0 codes are stored plus 128; of Q4_0 codes a byte holds two dims: of K, byte 4m + i dims 8m + i (low) and 8m + 4 + i,
of V dims 2x (low) and 2x + 1.  The new tokens of sequence b are rows q_start[b] .. q_start[b + 1] and the last of its
kv_len[b] keys.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

Q4_0, Q8_0 = 0, 6
THETA = 500000.0


# ---- cases ------------------------------------------------------------------------------------------------------

def _rope(name, T, H, D, axes, rot, traditional=False, token_major=False):
    return {"name": name, "op": "rope", "T": T, "H": H, "D": D, "axes": axes, "rot": rot, "traditional": traditional,
            "token_major": token_major}


def _cached(name, op, fmt, B, new, lo, hi, H, Hkv, D, page, **more):
    """B sequences of lo .. hi keys, spread over the logarithm; `new` of them are the rows of a pass."""
    return {"name": name, "op": op, "fmt": fmt, "B": B, "new": new, "lo": lo, "hi": hi, "H": H, "Hkv": Hkv, "D": D,
            "page": page, "spread": 1, "window": 0, "mixed": False, "axes": 1, **more}


def listed():
    return [
        # one decoded token each of 64 requests, an 8B model's query heads: launch latency counts
        _rope("rope_step_b64", 64, 32, 128, 1, 128),
        # a long prompt of image and text, positions in time, height and width
        _rope("rope_image_t8100", 8100, 32, 128, 3, 128),
        # the cache update of a decoding step: rotate, quantize, write one token of 64 requests of any length
        _cached("append_step_q8_b64", "append", Q8_0, 64, 1, 1, 8192, 32, 8, 128, 16),
        # prompts of three requests of a 1B model arriving together, lengths not whole pages, 4-bit cache
        _cached("append_prompts_q4_b3", "append", Q4_0, 3, 2048, 700, 2048, 32, 8, 64, 16),
        # eight requests' whole caches handed to another program
        _cached("read_q8_b8", "read", Q8_0, 8, 0, 500, 8192, 32, 8, 128, 64),
        # one short request's 4-bit cache
        _cached("read_q4_1000", "read", Q4_0, 1, 0, 1000, 1000, 32, 8, 64, 16),
        # one decoded token of one request: launches, the split over the keys and its join
        _cached("attn_step_q8_1000", "attn", Q8_0, 1, 1, 1000, 1000, 32, 8, 128, 16),
        # a decoding step of 64 requests of any length
        _cached("attn_step_q8_b64", "attn", Q8_0, 64, 1, 1, 8192, 32, 8, 128, 16),
        # a decoding step of four very long requests in a 4-bit cache
        _cached("attn_step_q4_131072", "attn", Q4_0, 4, 1, 131072, 131072, 32, 8, 128, 64),
        # five drafted tokens of 16 requests checked at once, a 1B model's heads
        _cached("attn_draft_q8_b16", "attn", Q8_0, 16, 5, 200, 8192, 32, 8, 64, 32),
        # a prompt's chunk among decoding requests, a sliding window
        _cached("attn_mixed_q4_b16", "attn", Q4_0, 16, 300, 400, 4096, 32, 8, 128, 16, mixed=True, window=1024),
        # the largest: a chunk of 2048 tokens of a long prompt
        _cached("attn_chunk_q8_30000", "attn", Q8_0, 1, 2048, 30000, 30000, 32, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attn", "attn", "attn"])
    D = rng.choice([64, 128])
    if op == "rope":
        axes = rng.choice([1, 2, 3])
        c = _rope("", _log(rng, 1, 8192), _log(rng, 1, 48), D, axes, rng.choice([D, D, D // 2]), rng.random() < 0.3,
                  rng.random() < 0.5)
    else:
        Hkv = rng.choice([1, 2, 4, 8, 8, 32])
        H = Hkv * (1 if Hkv == 32 else rng.choice([1, 2, 4, 5, 8]))
        B = _log(rng, 1, 128)
        hi = _log(rng, 16, min(65536, 4 * 131072 * 8 * 128 // (B * Hkv * D)))  # no more cache than the largest listed
        lo = max(1, int(hi * rng.choice([0.02, 0.3, 1.0])))
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 2048)])
        # no more rows times keys than the largest listed case, nor more rows of plain scores
        while new > 1 and (B * new * hi * H > 2048 * 30000 * 32 or B * new > 8192):
            new //= 2
        mixed = op == "attn" and B > 1 and new > 8 and rng.random() < 0.5
        lo, hi = max(lo, min(new, 4096)), max(hi, new)
        c = _cached("", op, rng.choice([Q8_0, Q4_0]), B, 0 if op == "read" else new, lo, hi, H, Hkv, D,
                    rng.choice([16, 32, 64, 128, 256]), spread=rng.randint(1, 10 ** 6),
                    window=_log(rng, 1, 8192) if op == "attn" and rng.random() < 0.25 else 0, mixed=mixed,
                    axes=rng.choice([1, 3]) if op == "append" else 1)
    del c["name"]
    return c


def _lengths(case):
    """(kv_len, new rows) of each sequence; new = 0 stands for all keys, mixed for one chunk among single tokens."""
    r = random.Random(case["spread"])
    lens = [_log(r, case["lo"], case["hi"]) for _ in range(case["B"])]
    new = [n if case["new"] == 0 else min(n, 1 if case["mixed"] and b else case["new"]) for b, n in enumerate(lens)]
    return lens, new


# ---- inputs -----------------------------------------------------------------------------------------------------

def _half(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen).to(torch.float16)


def _sections(pairs, axes):
    """The axis of each pair, in one run per axis: a quarter for time, the rest shared by height and width."""
    first = pairs // 4 if axes == 3 else pairs // axes
    rest = [(pairs - first) // (axes - 1)] * (axes - 1) if axes > 1 else []
    sizes = [pairs - sum(rest)] + rest
    return [a for a, n in enumerate(sizes) for _ in range(n)]


def _positions(gen, axes, T):
    """Text has one position on all axes; of several, some run in rows and columns as an image's do."""
    t = torch.arange(T, device="cuda") + int(torch.randint(0, 100000, (1,), device="cuda", generator=gen))
    return torch.stack([t if a == 0 else (t // 30 if a == 1 else t % 30) for a in range(axes)]).to(torch.int32)


def _codes(fmt, n, gen):
    """Codes (int16, 0 the middle) and fp16 scales of n blocks of 32 as the quantizer makes them of N(0, 1)."""
    x = torch.randn(n, 32, device="cuda", generator=gen).to(torch.float16).float()
    if fmt == Q8_0:
        d = x.abs().amax(-1, keepdim=True) / 127.0
        q = torch.round(x / d).clamp(-128, 127)
    else:
        d = x.gather(-1, x.abs().argmax(-1, keepdim=True)) / -8.0
        q = torch.floor(x / d + 8.5).clamp(0, 15) - 8
    return q.to(torch.int16), d[:, 0].to(torch.float16)


def _pack(fmt, k, ks, v, vs):
    """Pages [N, Hkv, bytes] of codes [N, Hkv, P, D] and scales [N, Hkv, P, D / 32] of K and V."""
    N, Hkv, P, D = k.shape
    v = v.reshape(N, Hkv, P // 4, 4, D).transpose(-1, -2)
    if fmt == Q8_0:
        kb, vb = (k + 128).to(torch.uint8), (v + 128).to(torch.uint8)
    else:
        k, v = (k + 8).to(torch.uint8).reshape(N, Hkv, P, D // 8, 2, 4), (v + 8).to(torch.uint8).reshape(N, Hkv, P // 4, D // 2, 2, 4)
        kb, vb = k[..., 0, :] | (k[..., 1, :] << 4), v[..., 0, :] | (v[..., 1, :] << 4)
    vs = vs.reshape(N, Hkv, P // 4, 4, D // 32).transpose(-1, -2)
    return torch.cat([x.reshape(N, Hkv, -1).contiguous().view(torch.uint8) for x in (kb, vb, ks, vs)], -1)


def _cache(case, gen):
    """Codes, scales and the page table of a filled cache whose pages lie in any order."""
    lens, _ = _lengths(case)
    Hkv, P, D = case["Hkv"], case["page"], case["D"]
    need = [-(-n // P) for n in lens]
    N = sum(need) + 3
    order = torch.randperm(N, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    parts = [_codes(case["fmt"], N * Hkv * P * D // 32, gen) for _ in range(2)]
    k, v = (q.reshape(N, Hkv, P, D) for q, _ in parts)
    ks, vs = (d.reshape(N, Hkv, P, D // 32) for _, d in parts)
    return k, ks, v, vs, table


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = {}
    if case["op"] == "rope":
        T, H, D = case["T"], case["H"], case["D"]
        t["x"] = _half(gen, *((T, H, D) if case["token_major"] else (H, T, D)))
        t["positions"] = _positions(gen, case["axes"], T)
        return t, None
    lens, new = _lengths(case)
    T, H, Hkv, D = sum(new), case["H"], case["Hkv"], case["D"]
    t["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    t["q_start"] = torch.tensor([0] + [sum(new[:b + 1]) for b in range(len(new))], dtype=torch.int32, device="cuda")
    cache = _cache(case, gen)
    t["table"] = cache[-1]
    if case["op"] == "append":
        t["q"], t["k"], t["v"] = _half(gen, H, T, D), _half(gen, Hkv, T, D), _half(gen, Hkv, T, D)
        t["positions"] = _positions(gen, case["axes"], T)
    elif case["op"] == "attn":
        t["q"] = _half(gen, H, T, D)
    return t, cache


def _package():
    at = str(Path(__file__).resolve().parents[1] / "m4-prefill-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import m4_bridge

    b = m4_bridge.HIPBridge.get_instance()
    if not b.is_initialized() and not b.init():
        raise RuntimeError(b.last_error())
    return m4_bridge, b


def prepare(case, seed):
    t, cache = _inputs(case, seed)
    state = {"case": case, "t": t}
    op = case["op"]
    if cache is not None:
        t["pages"] = _pack(case["fmt"], *cache[:-1])
    if op in ("rope", "append"):
        pairs = (case["rot"] if op == "rope" else case["D"]) // 2
        state["axis"] = _sections(pairs, case["axes"])
        t["axis"] = torch.tensor(state["axis"], device="cuda")
    if op == "rope":
        t["y"] = torch.empty_like(t["x"])
    elif op == "attn":
        t["o"] = torch.empty(t["q"].shape[1], case["H"], case["D"], dtype=torch.float16, device="cuda")
    else:
        T = int(t["q_start"][-1])
        t["k_out"], t["v_out"] = (torch.empty(case["Hkv"], T, case["D"], dtype=torch.float16, device="cuda") for _ in range(2))
        if op == "append":
            t["q_out"] = torch.empty_like(t["q"])
    if own:  # what a program keeps beside its tensors: the bridge, the cache and the batch it is about to run
        m, b = _package()
        b.synchronize()
        state["b"] = b
        if cache is not None:
            lens, new = _lengths(case)
            state["cache"] = m.PagedKVCache(case["fmt"], t["pages"].shape[0], case["page"], case["Hkv"], case["D"],
                                            pages=t["pages"])
            state["batch"] = m.KVBatch(t["q_start"], t["kv_len"], t["table"], max_new=max(new), max_kv=max(lens))
        if op in ("rope", "append"):
            state["rope"] = m.RotaryAxes(2 * len(state["axis"]), theta=THETA, pair_axes=state["axis"],
                                         traditional=case.get("traditional", False))
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _rotate(x, positions, axis, traditional):
    """x [..., T, D] by the angles of its rows, in fp32, rounded to fp16."""
    pairs = axis.numel()
    f = THETA ** (-torch.arange(pairs, device=x.device, dtype=torch.float64) / pairs)
    ang = positions.double().T[:, axis] * f
    cs, sn = torch.cos(ang).float(), torch.sin(ang).float()
    r, tail = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    if traditional:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2)
    else:
        a, b = r[..., :pairs], r[..., pairs:]
        y = torch.cat([a * cs - b * sn, a * sn + b * cs], -1)
    return torch.cat([y.to(torch.float16), tail], -1)


def _quantize(fmt, x):
    """Codes (0 the middle, fp32) and fp16 scales of fp16 x [..., D], in blocks of 32."""
    b = x.float().unflatten(-1, (-1, 32))
    if fmt == Q8_0:
        d = b.abs().amax(-1) / 127.0
        p = b * torch.where(d > 0, 1.0 / d, 0.0)[..., None]
        q = (torch.sign(p) * torch.floor(p.abs() + 0.5)).clamp(-128, 127)
    else:
        d = b.gather(-1, b.abs().argmax(-1, keepdim=True))[..., 0] / -8.0
        q = torch.floor(b * torch.where(d != 0, 1.0 / d, 0.0)[..., None] + 8.5).clamp(0, 15) - 8
    return q, d.to(torch.float16)


def _values(q, d):
    return (q * d.float()[..., None]).to(torch.float16).flatten(-2)


def _places(t, P, T):
    """Page, slot of every row."""
    rows = torch.arange(T, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(t["q_start"], rows, right=True) - 1
    p = t["kv_len"][b] - t["q_start"][b + 1] + rows
    return t["table"][b, p // P].long(), (p % P).long()


def _append_plain(state):
    c, t = state["case"], state["t"]
    fmt, P, D, T = c["fmt"], c["page"], c["D"], t["q"].shape[1]
    q = _rotate(t["q"], t["positions"], t["axis"], False)
    k = _rotate(t["k"], t["positions"], t["axis"], False)
    (kq, kd), (vq, vd) = _quantize(fmt, k), _quantize(fmt, t["v"])
    page, slot = _places(t, P, T)
    page, slot = page[:, None], slot[:, None]
    pages = t["pages"].transpose(0, 1)  # [Hkv, N, bytes]
    width = D if fmt == Q8_0 else D // 2
    i = torch.arange(width, device="cuda")
    if fmt == Q8_0:
        kb, vb = (kq.flatten(-2) + 128).to(torch.uint8), (vq.flatten(-2) + 128).to(torch.uint8)
    else:
        kn = (kq.flatten(-2) + 8).to(torch.uint8).unflatten(-1, (-1, 2, 4))
        vn = (vq.flatten(-2) + 8).to(torch.uint8).unflatten(-1, (-1, 2))
        kb, vb = (kn[..., 0, :] | (kn[..., 1, :] << 4)).flatten(-2), vn[..., 0] | (vn[..., 1] << 4)
    pages[:, page, slot * width + i] = kb
    pages[:, page, P * width + (slot // 4 * width + i) * 4 + slot % 4] = vb
    blocks = D // 32
    j = torch.arange(2 * blocks, device="cuda")
    pages[:, page, 2 * P * width + slot * 2 * blocks + j] = kd.view(torch.uint8)
    pages[:, page, 2 * P * width + 2 * P * blocks + (slot // 4 * blocks + j // 2) * 8 + slot % 4 * 2 + j % 2] = vd.view(torch.uint8)
    return {"q": q, "k": _values(kq, kd), "v": _values(vq, vd)}


def _decode(raw, fmt, P, D):
    """K and V [..., P, D] in fp32 of pages [..., bytes]."""
    width, blocks = (D if fmt == Q8_0 else D // 2), D // 32
    k, v, ks, vs = raw.split([P * width, P * width, 2 * P * blocks, 2 * P * blocks], -1)
    if fmt == Q8_0:
        k = k.unflatten(-1, (P, D)).float() - 128
        v = v.unflatten(-1, (P // 4, D, 4)).transpose(-1, -2).flatten(-3, -2).float() - 128
    else:
        k = k.unflatten(-1, (P, D // 8, 1, 4))
        k = torch.cat([k & 15, k >> 4], -2).flatten(-3).float() - 8
        v = v.unflatten(-1, (P // 4, D // 2, 1, 4))
        v = torch.cat([v & 15, v >> 4], -2).flatten(-3, -2).transpose(-1, -2).flatten(-3, -2).float() - 8
    ks = ks.contiguous().view(torch.float16).unflatten(-1, (P, blocks)).float()
    vs = vs.contiguous().view(torch.float16).unflatten(-1, (P // 4, blocks, 4)).transpose(-1, -2).flatten(-3, -2).float()
    return ((x.unflatten(-1, (blocks, 32)) * s[..., None]).flatten(-2) for x, s in ((k, ks), (v, vs)))


def _gathered(state):
    """K and V [B, Hkv, keys, D] in fp32, the keys padded to the longest sequence's pages."""
    c, t = state["case"], state["t"]
    raw = t["pages"][t["table"].clamp(min=0).long()].transpose(1, 2)  # [B, Hkv, pages, bytes]
    return [x.flatten(2, 3) for x in _decode(raw, c["fmt"], c["page"], c["D"])]


def _read_plain(state):
    k, v = (x.to(torch.float16) for x in _gathered(state))
    kept = torch.arange(k.shape[2], device="cuda") < state["t"]["kv_len"][:, None]
    return {n: x.transpose(1, 2)[kept].transpose(0, 1).contiguous() for n, x in (("k", k), ("v", v))}


def _attn_plain(state):
    c, t = state["case"], state["t"]
    k, v = _gathered(state)
    H, T, D = t["q"].shape
    B, Hkv, L, _ = k.shape
    new = t["q_start"].diff()
    most = max(_lengths(c)[1])
    i = torch.arange(most, device="cuda")
    live = i < new[:, None]  # [B, most]
    q = torch.zeros(B, most, H, D, device="cuda")
    q[live] = t["q"].transpose(0, 1).float()
    q = q.transpose(1, 2).reshape(B, Hkv, H // Hkv * most, D)
    s = torch.matmul(q, k.transpose(-1, -2)).reshape(B, H, most, L) * D ** -0.5
    p = (t["kv_len"] - new)[:, None, None] + i[None, :, None]
    j = torch.arange(L, device="cuda")
    hidden = j > p
    if c["window"]:
        hidden = hidden | (j <= p - c["window"])
    hidden = hidden | (j >= t["kv_len"][:, None, None])
    s.masked_fill_(hidden[:, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    z = s.sum(-1, keepdim=True)
    v = torch.where((j < t["kv_len"][:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(s.reshape(B, Hkv, H // Hkv * most, L), v).reshape(B, H, most, D) / z
    return o.transpose(1, 2)[live].to(torch.float16)


def run(state):
    c, t, op = state["case"], state["t"], state["case"]["op"]
    if own:
        b = state["b"]
        if op == "rope":
            b.rope_axes(t["x"], t["y"], state["rope"], t["positions"], token_major=c["token_major"])
            return t["y"]
        if op == "attn":
            b.dispatch_paged_attn(state["cache"], state["batch"], t["q"], t["o"], c["D"] ** -0.5, o_token_major=True,
                                  window=c["window"])
            return t["o"]
        if op == "append":
            b.kv_cache_append(state["cache"], state["batch"], t["k"], t["v"], rope=state["rope"],
                              positions=t["positions"], Q=t["q"], Q_out=t["q_out"])
        b.kv_cache_read(state["cache"], state["batch"], t["k_out"], t["v_out"])
        out = {"k": t["k_out"], "v": t["v_out"]}
        return {"q": t["q_out"], **out} if op == "append" else out
    if op == "rope":
        x = t["x"].transpose(0, 1) if c["token_major"] else t["x"]
        y = _rotate(x, t["positions"], t["axis"], c["traditional"])
        return y.transpose(0, 1) if c["token_major"] else y
    return {"append": _append_plain, "read": _read_plain, "attn": _attn_plain}[op](state)


# ---- the same in 64 bits ----------------------------------------------------------------------------------------

def _turned(x, positions, axis, traditional):
    """Rotation of x [H, T, D] as a product of complex numbers in float64."""
    n = len(axis)
    out = x.double().clone()
    at = positions.double()[torch.tensor(axis, device=x.device)]  # [pairs, T]
    w = torch.polar(torch.ones_like(at), at * torch.pow(torch.tensor(THETA, dtype=torch.float64, device=x.device),
                                                        -torch.arange(n, device=x.device).double() / n)[:, None]).T
    re, im = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if traditional else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(out[..., re], out[..., im]) * w
    out[..., re], out[..., im] = z.real.clone(), z.imag.clone()
    return out


def _cached_values(fmt, x):
    """The values that a cache holds of fp16 x: codes from the definition's steps, each rounded where it rounds (fp32
    scale, its inverse and the product), evaluated in float64."""
    f32 = lambda v: v.float().double()  # noqa: E731
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    big, first = b.abs().max(-1)
    d = f32(big / 127) if fmt == Q8_0 else f32(torch.take_along_dim(b, first[..., None], -1)[..., 0] / -8)
    inverse = torch.where(d != 0, f32(1 / torch.where(d != 0, d, 1.0)), 0.0)
    p = f32(b * inverse[..., None])
    if fmt == Q8_0:
        q = torch.clamp(torch.where(p < 0, -1.0, 1.0) * torch.floor(p.abs() + 0.5), -128, 127)
    else:
        q = torch.clamp(torch.floor(f32(p + 8.5)), 0, 15) - 8
    return (q * d.half().double()[..., None]).reshape(x.shape)


def exact(case, seed):
    t, cache = _inputs(case, seed)
    op = case["op"]
    if op == "rope":
        axis = _sections(case["rot"] // 2, case["axes"])
        x = t["x"].transpose(0, 1) if case["token_major"] else t["x"]
        y = _turned(x, t["positions"], axis, case["traditional"])
        return y.transpose(0, 1) if case["token_major"] else y
    if op == "append":
        axis = _sections(case["D"] // 2, case["axes"])
        return {"q": _turned(t["q"], t["positions"], axis, False),
                "k": _cached_values(case["fmt"], _turned(t["k"], t["positions"], axis, False).half()),
                "v": _cached_values(case["fmt"], t["v"])}
    kq, ks, vq, vs, table = cache
    lens, new = _lengths(case)
    P = case["page"]

    def sequence(b, q, s):
        """The values [Hkv, keys, D] of sequence b."""
        at = table[b, :-(-lens[b] // P)].long()
        x = q[at].double() * s[at].double().repeat_interleave(32, -1)
        return x.transpose(0, 1).flatten(1, 2)[:, :lens[b]]

    if op == "read":
        return {n: torch.cat([sequence(b, q, s) for b in range(len(lens))], 1) for n, q, s in (("k", kq, ks), ("v", vq, vs))}
    out, at = [], 0
    for b, (L, n) in enumerate(zip(lens, new)):
        k, v = sequence(b, kq, ks), sequence(b, vq, vs)
        G = case["H"] // case["Hkv"]
        p = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None, :]
        seen = (j <= p) & (j > p - case["window"]) if case["window"] else j <= p
        heads = []
        for h in range(case["H"]):
            s = t["q"][h, at:at + n].double() @ k[h // G].T * case["D"] ** -0.5
            heads.append(torch.softmax(torch.where(seen, s, -math.inf), -1) @ v[h // G])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    op, D = case["op"], case["D"]
    if op == "rope":
        T, H = case["T"], case["H"]
        return {"bytes": 4 * T * H * D + 4 * case["axes"] * T, "flops": 3 * T * H * case["rot"]}
    lens, new = _lengths(case)
    T, H, Hkv = sum(new), case["H"], case["Hkv"]
    row = 2 * Hkv * (34 if case["fmt"] == Q8_0 else 18) * D // 32  # a token's K and V in the cache
    if op == "read":
        return {"bytes": T * (row + 4 * Hkv * D), "flops": 2 * T * Hkv * D}
    if op == "append":  # the read back of the new rows is part of the pass
        return {"bytes": T * (4 * H * D + 4 * Hkv * D + row + 4 * Hkv * D + 4 * case["axes"]),
                "flops": T * D * (3 * H + 3 * Hkv + 8 * Hkv)}
    keys = seen = 0
    for L, n in zip(lens, new):
        w = case["window"] or L
        keys += L - max(0, L - n + 1 - w)
        seen += sum(min(p + 1, w) for p in range(L - n, L))
    return {"bytes": keys * row + 4 * T * H * D, "flops": 4 * H * D * seen}
