"""The operators of serving with trees of drafted tokens and with bounded caches, as data.  A step with a tree: the
ancestors and positions of its nodes, attention of the nodes over the cache and their ancestors, the walk that accepts a
path, and the move of the path's tokens to their places.  A bounded cache: the attention weight that each cached key
has received, and eviction of the lightest.  The cache is the paged, quantized one.

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
of V dims 2x (low) and 2x + 1.  Its values are half(q half(d)).  The new tokens of sequence b are rows
q_start[b] .. q_start[b + 1] and the last of its kv_len[b] keys; of a tree they are its nodes, each behind its parent,
and node 0, the sequence's newest token, is the root.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

Q4_0, Q8_0 = 0, 6


# ---- cases ------------------------------------------------------------------------------------------------------

def _tree(name, B, nodes, bushy=8):
    """B sequences with a tree of `nodes` nodes each, a node's parent about `bushy` nodes before it."""
    return {"name": name, "op": "tree", "B": B, "new": nodes, "bushy": bushy, "spread": 1}


def _cached(name, op, fmt, B, new, lo, hi, H, Hkv, D, page, **more):
    """B sequences of lo .. hi keys, spread over the logarithm; `new` of them are the rows of a pass."""
    return {"name": name, "op": op, "fmt": fmt, "B": B, "new": new, "lo": lo, "hi": hi, "H": H, "Hkv": Hkv, "D": D,
            "page": page, "spread": 1, "window": 0, "bushy": 8, **more}


def listed():
    return [
        # one step's trees of 16 requests, the size that draft heads propose: launch latency
        _tree("tree_b16_n64", 16, 64),
        # long trees of many requests: a step that searches widely
        _tree("tree_b64_n300", 64, 300, bushy=20),
        # the tree of one short request checked over its cache, an 8B model's heads
        _cached("attn_tree_q8_1000", "attn", Q8_0, 1, 16, 1000, 1000, 32, 8, 128, 16),
        # the trees of 16 requests of any length
        _cached("attn_tree_q8_b16", "attn", Q8_0, 16, 64, 200, 8192, 32, 8, 128, 16),
        # four very long requests in a 4-bit cache, odd sizes
        _cached("attn_tree_q4_131072", "attn", Q4_0, 4, 61, 131072, 131072, 32, 8, 128, 64),
        # the walk down one request's tree, and its tokens moved, a 1B model's heads
        _cached("accept_q4_b1", "accept", Q4_0, 1, 26, 900, 900, 32, 8, 64, 32),
        # the same of 64 requests and an 8B model
        _cached("accept_q8_b64", "accept", Q8_0, 64, 64, 100, 4096, 32, 8, 128, 16),
        # what each key received in a decoding step of 64 requests of any length
        _cached("weigh_step_q8_b64", "weigh", Q8_0, 64, 1, 1, 8192, 32, 8, 128, 16),
        # prompts of three requests of a 1B model, 4-bit cache
        _cached("weigh_prompts_q4_b3", "weigh", Q4_0, 3, 2048, 700, 2048, 32, 8, 64, 16),
        # the largest: a chunk of 2048 tokens of a long prompt
        _cached("weigh_chunk_q8_30000", "weigh", Q8_0, 1, 2048, 30000, 30000, 32, 8, 128, 64),
        # caches of 64 requests cut to 1024 tokens, those that are shorter kept whole
        _cached("evict_q8_b64", "evict", Q8_0, 64, 0, 300, 8192, 32, 8, 128, 16, budget=1024, sinks=4, recent=256),
        # one very long request's 4-bit cache cut to a quarter
        _cached("evict_q4_131072", "evict", Q4_0, 1, 0, 131072, 131072, 32, 8, 128, 64, budget=32768, sinks=4, recent=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "attn", "attn", "accept", "weigh", "weigh", "evict"])
    if op == "tree":
        nodes = _log(rng, 1, 700)
        c = _tree("", _log(rng, 1, max(1, min(128, 64 * 300 // nodes))), nodes, bushy=rng.choice([1, 2, 3, 8, 30]))
    else:
        D = rng.choice([64, 128])
        Hkv = rng.choice([1, 2, 4, 8, 8, 32])
        H = Hkv * (1 if Hkv == 32 else rng.choice([1, 2, 4, 5, 8]))
        B = _log(rng, 1, 128)
        hi = _log(rng, 16, min(65536, 4 * 131072 * 8 * 128 // (B * Hkv * D)))  # no more cache than the largest listed
        lo = max(1, int(hi * rng.choice([0.02, 0.3, 1.0])))
        fmt, page = rng.choice([Q8_0, Q4_0]), rng.choice([16, 32, 64, 128, 256])
        if op == "evict":
            budget = _log(rng, 1, hi)
            sinks = rng.choice([0, min(4, budget), budget // 3])
            c = _cached("", op, fmt, B, 0, lo, hi, H, Hkv, D, page, budget=budget, sinks=sinks,
                        recent=rng.choice([0, (budget - sinks) // 4, budget - sinks]))
        else:
            new = _log(rng, 1, 200) if op != "weigh" else rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 2048)])
            # no more rows times keys than the largest listed case, nor more rows of plain scores
            while new > 1 and (B * new * hi * H > 2048 * 30000 * 32 or B * new > 8192):
                new //= 2
            lo, hi = max(lo, min(new, 4096)), max(hi, new)
            c = _cached("", op, fmt, B, new, lo, hi, H, Hkv, D, page,
                        window=_log(rng, 1, 8192) if op in ("attn", "weigh") and rng.random() < 0.25 else 0,
                        bushy=rng.choice([1, 2, 3, 8, 30]))
    c["spread"] = rng.randint(1, 10 ** 6)
    del c["name"]
    return c


def _lengths(case):
    """(kv_len, new rows) of each sequence; new = 0 stands for no rows."""
    r = random.Random(case["spread"])
    if case["op"] == "tree":
        return [case["new"] + _log(r, 1, 8192) for _ in range(case["B"])], [case["new"]] * case["B"]
    lens = [_log(r, case["lo"], case["hi"]) for _ in range(case["B"])]
    return lens, [min(n, case["new"]) for n in lens]


def _trees(case):
    """The parent of each node of each sequence (-1: none), and the child that the model goes on with from each (-1:
    none of them)."""
    r = random.Random(case["spread"] + 1)
    parents, follows = [], []
    for n in _lengths(case)[1]:
        p = [-1] + [max(0, i - 1 - int(r.expovariate(1.0 / case["bushy"]))) for i in range(1, n)]
        f = [-1] * n
        for i in range(n - 1, 0, -1):
            if f[p[i]] < 0 or r.random() < 0.4:
                f[p[i]] = i
        parents.append(p)
        follows.append([c if r.random() < 0.85 else -1 for c in f])
    return parents, follows


# ---- inputs -----------------------------------------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _half(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen).to(torch.float16)


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


def _kept_lengths(case):
    return [min(n, case["budget"]) for n in _lengths(case)[0]]


def _cache(case, gen):
    """Codes and scales of a filled cache whose pages lie in any order, its page table, and that of the pages that an
    eviction fills."""
    lens, _ = _lengths(case)
    Hkv, P, D = case["Hkv"], case["page"], case["D"]
    need = [-(-n // P) for n in lens]
    more = [-(-n // P) for n in _kept_lengths(case)] if case["op"] == "evict" else []
    N = sum(need) + sum(more) + 3
    order = torch.randperm(N, device="cuda", generator=gen).to(torch.int32)
    tables, at = [], 0
    for rows in (need, more):
        table = torch.full((len(lens), max(rows, default=0)), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(rows):
            table[b, :n] = order[at:at + n]
            at += n
        tables.append(table)
    parts = [_codes(case["fmt"], N * Hkv * P * D // 32, gen) for _ in range(2)]
    k, v = (q.reshape(N, Hkv, P, D) for q, _ in parts)
    ks, vs = (d.reshape(N, Hkv, P, D // 32) for _, d in parts)
    return k, ks, v, vs, tables


def _sequence(case, cache, b, which, dtype=torch.float64):
    """K (0) or V (1) of sequence b, [Hkv, keys, D]."""
    q, s, at = cache[2 * which], cache[2 * which + 1], cache[4][0][b]
    n = _lengths(case)[0][b]
    at = at[:-(-n // case["page"])].long()
    x = (q[at].to(dtype).unflatten(-1, (-1, 32)) * s[at].to(dtype)[..., None]).flatten(-2).half()
    return x.transpose(0, 1).flatten(1, 2)[:, :n].to(dtype)


def _seen(case, b, first, n, ancestors=None):
    """Which of the keys first + n each of the last n rows sees."""
    i = torch.arange(n, device="cuda")[:, None]
    j = torch.arange(first + n, device="cuda")[None, :]
    if ancestors is None:
        p, k, seen = first + i, j, j <= first + i
    else:
        depth = first + ancestors.sum(-1) - 1
        p, k = depth[:, None], torch.cat([torch.arange(first, device="cuda"), depth])[None, :]
        seen = torch.cat([torch.ones(n, first, dtype=torch.bool, device="cuda"), ancestors], 1)
    return seen & (k > p - case["window"]) if case["window"] else seen


def _lse(case, cache, q):
    """log of the sum of exp(score) of each row [H, T] of causal attention: what the attention call hands over."""
    lens, new = _lengths(case)
    out, at = [], 0
    for b, (L, n) in enumerate(zip(lens, new)):
        k = _sequence(case, cache, b, 0, torch.float32).repeat_interleave(case["H"] // case["Hkv"], 0)
        s = torch.matmul(q[:, at:at + n].float(), k.transpose(-1, -2).contiguous()) * case["D"] ** -0.5
        s.masked_fill_(~_seen(case, b, L - n, n), -math.inf)
        out.append(torch.logsumexp(s.double(), -1) if n * L * case["H"] < 1 << 28 else torch.logsumexp(s, -1))
        at += n
    return torch.cat(out, 1).float()


def _ancestors(parents):
    """[n, n] bool: node j is i or before it."""
    n = len(parents)
    a = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def _words(a, words):
    """Ancestor masks [n, n] as int32 [n, words]."""
    a = torch.nn.functional.pad(a, (0, 32 * words - a.shape[1])).unflatten(-1, (words, 32)).long()
    w = (a << torch.arange(32, device=a.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens, new = _lengths(case)
    op, T = case["op"], sum(new)
    t = {"kv_len": _ints(lens), "q_start": _ints([0] + [sum(new[:b + 1]) for b in range(len(new))])}
    cache = None
    if op in ("tree", "attn", "accept"):
        parents, follows = _trees(case)
        words = -(-max(new) // 32)
        if op == "tree":  # a few nodes hang elsewhere, behind another number of keys
            move = random.Random(seed)
            t["kv_len"] += _ints([move.randrange(1000) for _ in lens])
            for p in parents:
                for i in range(1, len(p)):
                    if move.random() < 0.05:
                        p[i] = move.randrange(i)
        t["parents"] = _ints([p for s in parents for p in s])
        if op == "attn":
            anc = [_ancestors(p) for p in parents]
            t["ancestors"] = [a.cuda() for a in anc]
            t["mask"] = torch.cat([_words(a, words) for a in anc]).cuda()
            t["places"] = torch.cat([L - len(p) + a.sum(-1) - 1 for L, p, a in zip(lens, parents, anc)]).int().cuda()
        if op == "accept":
            names = torch.randperm(128000, device="cuda", generator=gen)[:T].int()  # no two nodes alike
            goes = _ints([c for f in follows for c in f])
            start = torch.repeat_interleave(t["q_start"][:-1].long(), _ints(new).long())
            other = torch.randint(128000, 129000, (T,), device="cuda", generator=gen).int()
            t["tokens"], t["targets"] = names, torch.where(goes < 0, other, names[(start + goes.clamp(min=0)).long()])
    if op != "tree":
        cache = _cache(case, gen)
        t["table"], t["table_out"] = cache[-1]
    if op in ("attn", "weigh"):
        t["q"] = _half(gen, case["H"], T, case["D"])
    if op == "weigh":
        t["lse"] = _lse(case, cache, t["q"])
    if op in ("weigh", "evict"):  # what keys have received so far, many of them nothing
        shape = (cache[0].shape[0], case["Hkv"], case["page"])
        t["sums"] = torch.exp(2 * torch.randn(shape, device="cuda", generator=gen))
        t["sums"] *= torch.rand(shape, device="cuda", generator=gen) > 0.1
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
    op, (lens, new) = case["op"], _lengths(case)
    B, T = case["B"], sum(new)
    if cache is not None:
        t["pages"] = _pack(case["fmt"], *cache[:4])
    if op == "tree":
        t["mask"] = torch.empty(T, -(-max(new) // 32), dtype=torch.int32, device="cuda")
        t["places"] = torch.empty(T, dtype=torch.int32, device="cuda")
    if op == "attn":
        t["o"] = torch.empty(T, case["H"], case["D"], dtype=torch.float16, device="cuda")
        t["lse"] = torch.empty(case["H"], T, device="cuda")
    if op == "accept":
        t["path"] = torch.empty(T, dtype=torch.int32, device="cuda")
        t["count"], t["next"], t["len_out"] = (torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(3))
    if op == "evict":
        kept = _kept_lengths(case)
        t["kept"] = torch.empty(B, case["Hkv"], case["budget"], dtype=torch.int32, device="cuda")
        t["len_out"] = torch.empty(B, dtype=torch.int32, device="cuda")
        t["start_out"] = _ints([0] + [sum(kept[:b + 1]) for b in range(B)])
        T = sum(kept)
    if op in ("accept", "evict"):
        t["k_out"], t["v_out"] = (torch.empty(case["Hkv"], T, case["D"], dtype=torch.float16, device="cuda") for _ in range(2))
    if own:  # what a program keeps beside its tensors: the bridge, the cache, the batch and the trees
        m, b = _package()
        b.synchronize()
        state["b"] = b
        table = t["table"] if cache is not None else torch.zeros(B, 1, dtype=torch.int32, device="cuda")
        state["batch"] = m.KVBatch(t["q_start"], t["kv_len"], table, max_new=max(new), max_kv=max(lens))
        if op in ("tree", "attn"):
            state["tree"] = m.DraftTree(t["mask"], t["places"])
        if cache is not None:
            state["cache"] = m.PagedKVCache(case["fmt"], t["pages"].shape[0], case["page"], case["Hkv"], case["D"],
                                            pages=t["pages"])
        if op == "evict":
            state["after"] = m.KVBatch(t["start_out"], t["len_out"], t["table_out"], max_new=max(kept), max_kv=max(kept))
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _padded(state):
    """(row of each place, whether it is one) [B, most]: the rows of the sequences side by side."""
    t = state["t"]
    new = t["q_start"].diff()
    i = torch.arange(max(_lengths(state["case"])[1]), device="cuda")
    live = i < new[:, None]
    return torch.where(live, t["q_start"][:-1, None] + i, 0).long(), live


def _closure(state, parents, live):
    """Ancestors [B, n, n] as fp32 zeros and ones, of parents [B, n]: paths of length 1, 2, 4 ..."""
    n = parents.shape[1]
    eye = torch.eye(n, device="cuda")
    a = (eye + (torch.arange(n, device="cuda") == parents[..., None])).clamp(max=1) * live[..., None]
    for _ in range(max(1, (n - 1).bit_length())):
        a = torch.matmul(a, a).clamp(max=1)
    return a


def _tree_plain(state):
    t = state["t"]
    rows, live = _padded(state)
    a = _closure(state, torch.where(live, t["parents"][rows], -2), live)
    first = t["kv_len"] - t["q_start"].diff()
    places = first[:, None] + a.sum(-1).int() - 1
    return {"mask": _words(a, t["mask"].shape[1])[live], "places": places[live]}


def _accept_plain(state):
    c, t = state["case"], state["t"]
    rows, live = _padded(state)
    n = rows.shape[1]
    parents = torch.where(live, t["parents"][rows], -2).long()
    at = parents.clamp(min=0)
    token, target = t["tokens"][rows], t["targets"][rows]
    match = live & (parents >= 0) & (token == target.gather(1, at))
    earlier = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"), -1)
    twin = (match[:, None, :] & (parents[:, None, :] == parents[..., None]) & earlier).any(-1)
    ok = match & ~twin
    ok[:, 0] = True
    taken = (torch.matmul(_closure(state, parents, live), (~ok).float()[..., None])[..., 0] == 0) & live
    count = taken.sum(-1)
    i = torch.arange(n, device="cuda")
    path = torch.sort(torch.where(taken, i, n), -1).values
    inside = i < count[:, None]
    path = torch.where(inside, path, -1)
    last = path.gather(1, count[:, None] - 1)
    first = (t["kv_len"] - t["q_start"].diff())[:, None]
    _move(state, *torch.where(inside)[:1], (first + path)[inside], (first + i)[inside])
    p = (first + i)[live]
    b = torch.where(live)[0]
    raw = t["pages"][t["table"][b, p // c["page"]].long()]
    k, v = _tokens(raw, c, p % c["page"])
    return {"path": path[live].int(), "count": count.int(), "next": target.gather(1, last)[:, 0],
            "kv_len": (first[:, 0] + count).int(), "k": k, "v": v}


def _parts(pages, c):
    """K codes [.., P, bytes], V codes [.., P / 4, bytes, 4], K scales and V scales alike, views of pages [.., bytes]."""
    P, blocks = c["page"], c["D"] // 32
    width = c["D"] if c["fmt"] == Q8_0 else c["D"] // 2
    k, v, ks, vs = pages.split([P * width, P * width, 2 * P * blocks, 2 * P * blocks], -1)
    return (k.unflatten(-1, (P, width)), v.unflatten(-1, (P // 4, width, 4)), ks.unflatten(-1, (P, 2 * blocks)),
            vs.unflatten(-1, (P // 4, blocks, 4, 2)))


def _move(state, b, src, dst):
    """The tokens src of sequences b to the places dst of the same sequences, every head's."""
    c, t = state["case"], state["t"]
    P = c["page"]
    sp, dp = t["table"][b, src // P].long(), t["table"][b, dst // P].long()
    si, di = (src % P).long(), (dst % P).long()
    k, v, ks, vs = _parts(t["pages"], c)
    k[dp, :, di] = k[sp, :, si]
    v[dp, :, di // 4, :, di % 4] = v[sp, :, si // 4, :, si % 4]
    ks[dp, :, di] = ks[sp, :, si]
    vs[dp, :, di // 4, :, di % 4] = vs[sp, :, si // 4, :, si % 4]


def _tokens(raw, c, slot):
    """K and V [Hkv, T, D] fp16 of the tokens `slot` of pages [T, Hkv, bytes]."""
    k, v, ks, vs = _parts(raw, c)
    T, Hkv = raw.shape[:2]
    i = torch.arange(T, device="cuda")
    slot = slot.long()
    k, ks = k[i, :, slot], ks[i, :, slot]
    v, vs = v[i, :, slot // 4, :, slot % 4], vs[i, :, slot // 4, :, slot % 4].flatten(-2)
    if c["fmt"] == Q8_0:
        k, v = k.float() - 128, v.float() - 128
    else:
        k = torch.stack([x.unflatten(-1, (-1, 4)) for x in (k & 15, k >> 4)], -2).flatten(-3).float() - 8
        v = torch.stack([v & 15, v >> 4], -1).flatten(-2).float() - 8
    return [(x.unflatten(-1, (-1, 32)) * s.contiguous().view(torch.float16).float()[..., None]).flatten(-2).half().transpose(0, 1).contiguous()
            for x, s in ((k, ks), (v, vs))]


def _values(state, which):
    """K (0) or V (1) [B, Hkv, keys, D] in fp32, rounded to fp16 as the cache's values are, the keys padded to the
    longest sequence's pages."""
    c, t = state["case"], state["t"]
    raw = t["pages"][t["table"].clamp(min=0).long()].transpose(1, 2)  # [B, Hkv, pages, bytes]
    codes, scales = _parts(raw, c)[which], _parts(raw, c)[2 + which]
    if which:
        codes = codes.transpose(-1, -2).flatten(-3, -2)
        scales = scales.transpose(-2, -3).flatten(-4, -3).flatten(-2)
    if c["fmt"] == Q8_0:
        x = codes.float() - 128
    elif which:
        x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8
    else:
        x = codes.unflatten(-1, (-1, 4))
        x = torch.stack([x & 15, x >> 4], -2).flatten(-3).float() - 8
    d = scales.contiguous().view(torch.float16).float()
    return (x.unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2).half().float().flatten(2, 3)


def _scores(state, hidden):
    """Scores [B, Hkv, G, rows, keys] of the rows, padded, -infinity where hidden [B, rows, keys]."""
    c, t = state["case"], state["t"]
    rows, live = _padded(state)
    k = _values(state, 0)
    q = t["q"][:, rows].float().transpose(0, 1).unflatten(1, (c["Hkv"], -1))  # [B, Hkv, G, rows, D]
    s = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, q.shape[2:4])
    s *= c["D"] ** -0.5
    return s.masked_fill_(hidden[:, None, None], -math.inf)


def _attn_plain(state):
    c, t = state["case"], state["t"]
    rows, live = _padded(state)
    first = (t["kv_len"] - t["q_start"].diff())[:, None, None]
    j = torch.arange(t["table"].shape[1] * c["page"], device="cuda")
    node = (j - first)  # [B, 1, keys]: which node a key is
    place = t["places"][rows][..., None]
    at = node.clamp(0, rows.shape[1] - 1)
    words = t["mask"][rows].gather(2, (at // 32).expand(-1, rows.shape[1], -1).clamp(max=t["mask"].shape[1] - 1))
    bit = (words >> at % 32) & 1
    hidden = (node >= t["q_start"].diff()[:, None, None]) | ((node >= 0) & (bit == 0))
    if c["window"]:
        key = torch.where(node < 0, j, t["places"][rows].gather(1, at[:, 0])[:, None])
        hidden = hidden | (key <= place - c["window"])
    hidden = hidden | ~live[..., None]
    s = _scores(state, hidden)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    s -= top
    s.exp_()
    z = s.sum(-1, keepdim=True)
    lse = (top + torch.log(z))[..., 0].flatten(1, 2).transpose(1, 2)[live].T.contiguous()
    v = torch.where((j < t["kv_len"][:, None])[:, None, :, None], _values(state, 1), 0.0)
    o = torch.matmul(s.flatten(2, 3), v).unflatten(2, s.shape[2:4]) / torch.where(z > 0, z, 1.0)
    return {"o": o.flatten(1, 2).transpose(1, 2)[live].half(), "lse": lse}


def _weigh_plain(state):
    c, t = state["case"], state["t"]
    rows, live = _padded(state)
    first = (t["kv_len"] - t["q_start"].diff())[:, None]
    j = torch.arange(t["table"].shape[1] * c["page"], device="cuda")
    p = (first + torch.arange(rows.shape[1], device="cuda"))[..., None]
    hidden = (j > p) | ~live[..., None]
    if c["window"]:
        hidden = hidden | (j <= p - c["window"])
    s = _scores(state, hidden)
    s -= t["lse"][:, rows].transpose(0, 1).unflatten(1, (c["Hkv"], -1))[..., None]
    w = s.exp_().sum((2, 3))  # [B, Hkv, keys]
    there = torch.where(j < t["kv_len"][:, None])
    page, slot = t["table"][there[0], there[1] // c["page"]].long(), there[1] % c["page"]
    old = (j < first)[there]
    t["sums"][page, :, slot] = torch.where(old[:, None], t["sums"][page, :, slot], 0.0) + w[there[0], :, there[1]]
    return t["sums"]


def _chosen_plain(state):
    """The places that are kept, [B, Hkv, budget] in order, the sequence's length where there are no more."""
    c, t = state["case"], state["t"]
    P, n = c["page"], t["kv_len"][:, None, None]
    j = torch.arange(t["table"].shape[1] * P, device="cuda")
    w = t["sums"][t["table"].clamp(min=0).long()].transpose(1, 2).flatten(2)  # [B, Hkv, keys]
    w = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), math.inf, w)
    w = torch.where(j < n, w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    at = torch.where(order < n, order, n)
    at = torch.nn.functional.pad(at, (0, c["budget"] - at.shape[-1]), value=1 << 30)
    return torch.minimum(torch.sort(at, -1).values, n)


def _evict_plain(state):
    c, t = state["case"], state["t"]
    P, budget = c["page"], c["budget"]
    at = _chosen_plain(state)
    length = torch.minimum(t["kv_len"], torch.tensor(budget, device="cuda")).int()
    i = torch.arange(budget, device="cuda")
    b, to = torch.where(i < length[:, None])
    src = at[b, :, to]  # [tokens, Hkv]
    sp, si = t["table"][b[:, None], src // P].long(), (src % P).long()
    dp, di = t["table_out"][b, to // P].long()[:, None], (to % P)[:, None]
    h = torch.arange(c["Hkv"], device="cuda")
    k, v, ks, vs = _parts(t["pages"], c)
    k[dp, h, di] = k[sp, h, si]
    v[dp, h, di // 4, :, di % 4] = v[sp, h, si // 4, :, si % 4]
    ks[dp, h, di] = ks[sp, h, si]
    vs[dp, h, di // 4, :, di % 4] = vs[sp, h, si // 4, :, si % 4]
    t["sums"][dp, h, di] = t["sums"][sp, h, si]
    ko, vo = _tokens(t["pages"][dp[:, 0]], c, di[:, 0])
    return {"k": ko, "v": vo, "sums": t["sums"], "kv_len": length,
            "kept": torch.where(i < length[:, None, None], at, -1).int()}


def run(state):
    c, t, op = state["case"], state["t"], state["case"]["op"]
    if not own:
        return {"tree": _tree_plain, "attn": _attn_plain, "accept": _accept_plain, "weigh": _weigh_plain,
                "evict": _evict_plain}[op](state)
    b, batch = state["b"], state["batch"]
    if op == "tree":
        b.draft_tree(batch, t["parents"], state["tree"])
        return {"mask": t["mask"], "places": t["places"]}
    cache = state["cache"]
    if op == "attn":
        b.dispatch_paged_attn(cache, batch, t["q"], t["o"], c["D"] ** -0.5, o_token_major=True, window=c["window"],
                              tree=state["tree"], lse=t["lse"])
        return {"o": t["o"], "lse": t["lse"]}
    if op == "weigh":
        b.kv_cache_weigh(cache, batch, t["q"], t["lse"], t["sums"], c["D"] ** -0.5, window=c["window"])
        return t["sums"]
    if op == "accept":
        b.tree_accept(batch, t["parents"], t["tokens"], t["targets"], t["path"], t["count"], t["next"])
        b.kv_cache_keep(cache, batch, t["path"], t["count"], t["len_out"])
        b.kv_cache_read(cache, batch, t["k_out"], t["v_out"])
        return {"path": t["path"], "count": t["count"], "next": t["next"], "kv_len": t["len_out"], "k": t["k_out"],
                "v": t["v_out"]}
    b.kv_cache_evict(cache, batch, t["sums"], t["table_out"], t["len_out"], c["budget"], sinks=c["sinks"],
                     recent=c["recent"], kept=t["kept"])
    b.kv_cache_read(cache, state["after"], t["k_out"], t["v_out"])
    return {"k": t["k_out"], "v": t["v_out"], "sums": t["sums"], "kv_len": t["len_out"], "kept": t["kept"]}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    t, cache = _inputs(case, seed)
    op = case["op"]
    if op == "tree":
        return None
    lens, new = _lengths(case)
    G, P, scale = case["H"] // case["Hkv"], case["page"], case["D"] ** -0.5
    outs, at = [], 0
    if op == "attn":
        for b, (L, n) in enumerate(zip(lens, new)):
            k, v = _sequence(case, cache, b, 0), _sequence(case, cache, b, 1)
            seen = _seen(case, b, L - n, n, t["ancestors"][b])
            for h in range(case["H"]):
                s = torch.where(seen, t["q"][h, at:at + n].double() @ k[h // G].T * scale, -math.inf)
                outs.append((torch.softmax(s, -1) @ v[h // G], torch.logsumexp(s, -1)))
            at += n
        H = case["H"]
        return {"o": torch.cat([torch.stack([o for o, _ in outs[i:i + H]], 1) for i in range(0, len(outs), H)]),
                "lse": torch.cat([torch.stack([z for _, z in outs[i:i + H]]) for i in range(0, len(outs), H)], 1)}
    if op == "weigh":
        sums = t["sums"].double()
        for b, (L, n) in enumerate(zip(lens, new)):
            k = _sequence(case, cache, b, 0)
            seen = _seen(case, b, L - n, n)
            w = torch.zeros(case["Hkv"], L, dtype=torch.float64, device="cuda")
            for h in range(case["H"]):
                s = t["q"][h, at:at + n].double() @ k[h // G].T * scale - t["lse"][h, at:at + n, None].double()
                w[h // G] += torch.where(seen, torch.exp(s), 0.0).sum(0)
            at += n
            j = torch.arange(L, device="cuda")
            page, slot = cache[4][0][b][j // P].long(), j % P
            sums[page, :, slot] = torch.where(j[:, None] < L - n, sums[page, :, slot], 0.0) + w.T
        return sums
    if op == "accept":  # the values of the rows, those of the accepted path moved to the front
        start = t["q_start"].tolist()
        tokens, targets = t["tokens"].tolist(), t["targets"].tolist()
        for b, (L, n, parents) in enumerate(zip(lens, new, _trees(case)[0])):
            path, go = [0], True
            while go:
                fits = [i for i in range(n) if parents[i] == path[-1] and tokens[start[b] + i] == targets[start[b] + path[-1]]]
                path, go = path + fits[:1], bool(fits)
            order = torch.tensor(path + list(range(len(path), n)), device="cuda")
            outs.append([_sequence(case, cache, b, w)[:, L - n:][:, order] for w in (0, 1)])
        return {"k": torch.cat([k for k, _ in outs], 1), "v": torch.cat([v for _, v in outs], 1)}
    sums, table, to = t["sums"].double(), cache[4][0], cache[4][1]
    moved = sums.clone()
    for b, (L, n) in enumerate(zip(lens, _kept_lengths(case))):
        j = torch.arange(L, device="cuda")
        w = sums[table[b][j // P].long(), :, j % P].T.clone()  # [Hkv, L]
        w[:, (j < case["sinks"]) | (j >= L - case["recent"])] = math.inf
        keep = torch.sort(torch.argsort(w, dim=-1, descending=True, stable=True)[:, :n], -1).values
        k, v = _sequence(case, cache, b, 0), _sequence(case, cache, b, 1)
        outs.append([torch.take_along_dim(x, keep[..., None], 1) for x in (k, v)])
        i = torch.arange(n, device="cuda")
        for h in range(case["Hkv"]):
            moved[to[b][i // P].long(), h, i % P] = sums[table[b][keep[h] // P].long(), h, keep[h] % P]
    return {"k": torch.cat([k for k, _ in outs], 1), "v": torch.cat([v for _, v in outs], 1), "sums": moved}


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    op, (lens, new) = case["op"], _lengths(case)
    T = sum(new)
    if op == "tree":
        return {"bytes": 4 * T * (2 + -(-max(new) // 32)), "flops": T * 10}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    row = 2 * Hkv * (34 if case["fmt"] == Q8_0 else 18) * D // 32  # a token's K and V in the cache
    if op == "accept":  # parents, tokens, targets, path; a third of the rows moved; the rows read back
        return {"bytes": T * 16 + T // 3 * 2 * row + T * (row + 4 * Hkv * D), "flops": T * Hkv * D * 2}
    if op == "evict":  # sums, the kept tokens moved and read back
        kept = sum(_kept_lengths(case))
        return {"bytes": 4 * Hkv * sum(lens) + kept * (2 * row + 12 * Hkv) + kept * (row + 4 * Hkv * D),
                "flops": sum(lens) * Hkv + kept * Hkv * D * 2}
    keys = seen = 0
    if op == "attn":
        for L, n, parents in zip(lens, new, _trees(case)[0]):
            depth = [0] * n
            for i, p in enumerate(parents):
                depth[i] = depth[p] + 1 if p >= 0 else 0
            w = case["window"] or L + 1
            keys += min(L, n + w)
            seen += sum(min(L - n + d + 1, w) for d in depth)
        return {"bytes": keys * row + T * H * (4 * D + 4) + T * 4 * -(-max(new) // 32), "flops": 4 * H * D * seen}
    for L, n in zip(lens, new):
        w = case["window"] or L
        keys += L - max(0, L - n + 1 - w)
        seen += sum(min(p + 1, w) for p in range(L - n, L))
    return {"bytes": keys * (row // 2 + 8 * Hkv) + T * H * (2 * D + 4), "flops": 2 * H * D * seen}
