"""Plain implementations, in 64 bits on the CPU, of the serving operators: rotary positions with several axes, the
paged quantized KV cache and attention over it.  Written from the definitions in include/m4_mlx_bridge.h."""
from __future__ import annotations

import numpy as np

Q4_0, Q8_0 = 0, 6


def page_bytes(fmt, P, D):
    return 2 * P * (D if fmt == Q8_0 else D // 2) + 4 * P * (D // 32)


def quantize(fmt, x):
    """fp16 [..., D] -> (codes int [..., D] around 0, scales fp16 [..., D / 32]); each step rounds to fp32."""
    f = np.float32
    b = x.astype(f).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        if fmt == Q8_0:
            d = np.abs(b).max(-1) / f(127)
            inv = np.where(d > 0, f(1) / np.where(d > 0, d, f(1)), f(0)).astype(f)
            p = (b * inv[..., None]).astype(f)
            q = np.clip(np.sign(p) * np.floor(np.abs(p.astype(np.float64)) + 0.5), -128, 127)
        else:
            at = np.abs(b).argmax(-1)
            d = np.take_along_axis(b, at[..., None], -1)[..., 0] / f(-8)
            inv = np.where(d != 0, f(1) / np.where(d != 0, d, f(1)), f(0)).astype(f)
            q = np.clip(np.floor((b * inv[..., None]).astype(f) + f(8.5)), 0, 15) - 8
    return q.reshape(x.shape).astype(np.int32), d.astype(np.float16)


def values(q, d):
    """half(q half(d)) of codes [..., D] and scales [..., D / 32]."""
    with np.errstate(all="ignore"):
        return (q.astype(np.float64) * np.repeat(d, 32, -1).astype(np.float64)).astype(np.float16)


class Pages:
    """The cache's bytes as numpy [num_pages, Hkv, bytes], with the places of a token's parts."""

    def __init__(self, fmt, num_pages, P, Hkv, D, fill=0xFF):
        self.fmt, self.P, self.Hkv, self.D = fmt, P, Hkv, D
        self.raw = np.full((num_pages, Hkv, page_bytes(fmt, P, D)), fill, np.uint8)

    def _places(self, slot):
        P, D, nb = self.P, self.D, self.D // 32
        w = D if self.fmt == Q8_0 else D // 2
        i, j = np.arange(w), np.arange(nb)
        return (slot * w + i, P * w + ((slot // 4) * w + i) * 4 + slot % 4,
                2 * P * w + (slot * nb + j) * 2, 2 * P * w + 2 * P * nb + ((slot // 4 * nb + j) * 4 + slot % 4) * 2)

    def write(self, page, slot, k, ks, v, vs):
        """Codes [Hkv, D] and scales [Hkv, D / 32] of one token."""
        ak, av, aks, avs = self._places(slot)
        if self.fmt == Q8_0:
            kb, vb = (k + 128).astype(np.uint8), (v + 128).astype(np.uint8)
        else:
            k8 = (k + 8).reshape(self.Hkv, -1, 8).astype(np.uint8)
            kb = (k8[..., :4] | (k8[..., 4:] << 4)).reshape(self.Hkv, -1)
            v8 = (v + 8).astype(np.uint8)
            vb = v8[:, 0::2] | (v8[:, 1::2] << 4)
        self.raw[page][:, ak], self.raw[page][:, av] = kb, vb
        for at, s in ((aks, ks), (avs, vs)):
            b = np.ascontiguousarray(s).view(np.uint8).reshape(self.Hkv, -1, 2)
            self.raw[page][:, at], self.raw[page][:, at + 1] = b[..., 0], b[..., 1]

    def read(self, page, slot):
        """(K, V) values fp16 [Hkv, D] of one token."""
        ak, av, aks, avs = self._places(slot)
        r = self.raw[page]
        kb, vb = r[:, ak].astype(np.int32), r[:, av].astype(np.int32)
        if self.fmt == Q8_0:
            k, v = kb - 128, vb - 128
        else:
            kb = kb.reshape(self.Hkv, -1, 4)
            k = np.concatenate([kb & 15, kb >> 4], -1).reshape(self.Hkv, -1) - 8
            v = np.stack([vb & 15, vb >> 4], -1).reshape(self.Hkv, -1) - 8
        ks, vs = (np.ascontiguousarray(np.stack([r[:, a], r[:, a + 1]], -1)).view(np.float16)[..., 0] for a in (aks, avs))
        return values(k, ks), values(v, vs)


def rotate(x, positions, pair_axes, inv_freq, traditional):
    """x [H, T, D] in float64 by positions [axes, T]."""
    n = len(pair_axes)
    ang = np.asarray(positions, np.float64)[np.asarray(pair_axes)].T * np.asarray(inv_freq)[None, :]  # [T, n]
    cs, sn = np.cos(ang), np.sin(ang)
    y = x.astype(np.float64).copy()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if traditional else (slice(0, n), slice(n, 2 * n))
    xa, xb = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
    y[..., a], y[..., b] = xa * cs - xb * sn, xa * sn + xb * cs
    return y


def attention(q, k, v, first, window, scale, valid=None):
    """q [H, n, D] fp16 at positions first .. first + n - 1; k, v [Hkv, keys, D] fp16.  Returns the result in float64
    [H, n, D] and a bound on what a kernel may be off it by, from these roundings:
      * scores in fp32: (D + 8) 2^-24 of the sum of |q k|, the product with the scale and the base-2 exponent 2^-22
        relative to the exponent, so weights are off by e = 2 (that) + 2^-21 relatively;
      * each weight rounds to fp16 once (2^-11, or 2^-25 absolutely beside the largest, which is at least 2^7) and
        the sum is of the rounded ones, so a weight's error multiplies v - o;
      * fp32 sums over the keys: (keys + 8) 2^-24 of the sum of |w v|;
      * the result rounds to fp16: 2^-11 |o|, or 2^-25 where it is subnormal."""
    H, n, D = q.shape
    Hkv, L, _ = k.shape
    o, bound = np.zeros((H, n, D)), np.zeros((H, n, D))
    pos = first + np.arange(n)[:, None]
    j = np.arange(L)[None, :]
    seen = j <= pos
    if window:
        seen &= j > pos - window
    if valid is not None:
        seen &= valid[None, :]
    with np.errstate(all="ignore"):
        for h in range(H):
            kk, vv = k[h // (H // Hkv)].astype(np.float64), v[h // (H // Hkv)].astype(np.float64)
            qq = q[h].astype(np.float64)
            s = np.where(seen, (qq @ np.where(np.isfinite(kk), kk, 0).T) * scale, -np.inf)
            a = (np.abs(qq) @ np.abs(np.where(np.isfinite(kk), kk, 0)).T) * abs(scale)
            m = s.max(-1, keepdims=True) if L else np.full((n, 1), -np.inf)
            any_seen = np.isfinite(m)
            w = np.where(seen & any_seen, np.exp(s - np.where(any_seen, m, 0)), 0)
            z = w.sum(-1, keepdims=True)
            w = w / np.where(z > 0, z, 1)
            fin = np.where(np.isfinite(vv), vv, 0)
            o[h] = w @ fin
            e = 2 * np.where(seen, a * ((D + 8) * 2.0 ** -24 + 2.0 ** -22), 0).max(-1, initial=0)[:, None] + 2.0 ** -21
            big = w @ np.abs(fin)
            top = np.abs(fin).max(0, initial=0)[None, :]
            bound[h] = ((2.0 ** -11 + e) * (big + np.abs(o[h])) + seen.sum(-1, keepdims=True) * 2.0 ** -32 * (top + np.abs(o[h]))
                        + (L + 8) * 2.0 ** -24 * big + 2.0 ** -11 * np.abs(o[h]) + 2.0 ** -25)
            for key in np.nonzero(~np.isfinite(vv).all(-1))[0]:  # a value that is not finite reaches the rows that see it
                rows = seen[:, key]
                bad = ~np.isfinite(vv[key])
                o[h][np.ix_(rows, bad)] = np.nan
    return o, bound
