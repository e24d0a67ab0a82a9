"""The paged 8-bit cache, attention over it and sampling, restated in float64
numpy from their definitions: what the GPU tests compare with."""
import math

import numpy as np

ROWS = (32, 64, 96, 128, 192, 256)


def padded(hd):
    return next(r for r in ROWS if r >= hd)


def _table():
    v = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = (1 + m / 8) * 2.0 ** (e - 7) if e else m * 2.0 ** -9
        v[b] = np.nan if b & 127 == 127 else (-x if b & 128 else x)
    return v


E4M3 = _table()
_POS = E4M3[:127]


def encode(x):
    """Nearest E4M3 bytes, ties to the even code; |x| <= 448; NaN and infinities 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = code | np.where(np.signbit(x), 0x80, 0).astype(np.uint8)
    return np.where(np.isfinite(x), code, 0x7f).astype(np.uint8)


def bf16_bits(x):
    """float32 -> bfloat16 bits, nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + (u >> 16 & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(np.asarray(x, np.float32))
    return np.where(nan, ((u >> 16).astype(np.uint16) | 0x40), r).astype(np.uint16)


def bf16_value(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def tables(n, hd):
    """applyRoPE's angles: float32 position times float32 frequency."""
    h = hd // 2
    th = np.array([np.float32(10000.0 ** (-(2 * k) / hd)) for k in range(h)], np.float32).reshape(1, h)
    ang = (np.arange(n, dtype=np.float32)[:, None] * th).astype(np.float32).astype(np.float64)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rotate(x, cos, sin):
    """x [..., hd] float64, cos / sin [..., hd // 2]: the exact values, rounded to float32."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:2 * h]
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    y = np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * h:]], -1)
    return y.astype(np.float32).astype(np.float64)


class Cache:
    def __init__(self, pages, page, kvh, hd, table, rng):
        self.P, self.kvh, self.hd, self.R = page, kvh, hd, padded(hd)
        self.pages, self.table = pages, np.ascontiguousarray(table, np.int32)
        # bytes of any kind, NaN among them, where nothing was stored yet; scales too
        self.k = rng.integers(0, 256, (pages, kvh, page, self.R)).astype(np.uint8)
        self.v = rng.integers(0, 256, (pages, kvh, self.R, page)).astype(np.uint8)
        self.ks = np.full((pages, kvh), np.nan, np.float32)
        self.vs = np.full((pages, kvh), np.nan, np.float32)

    def append(self, b, pos, k, v):
        """k, v [n, kvh, hd] float64 at positions pos .. pos + n - 1 of sequence b."""
        n = k.shape[0]
        if n == 0:
            return
        for j in range(pos // self.P, (pos + n - 1) // self.P + 1):
            page = self.table[b, j]
            if not 0 <= page < self.pages:
                continue
            lo, hi = max(pos - j * self.P, 0), min(pos + n - j * self.P, self.P)
            at = j * self.P + lo - pos
            for x, S, cache, up in ((k, self.ks, self.k, False), (v, self.vs, self.v, True)):
                for h in range(self.kvh):
                    part = x[at:at + hi - lo, h]
                    ok = np.abs(part[np.isfinite(part)])
                    a = ok.max() if ok.size else 0.0
                    e = -100
                    if a > 0:
                        f, q = math.frexp(a / 448.0)
                        e = max(q - 1 if f == 0.5 else q, -100)
                    s = np.float32(2.0 ** e)
                    if lo:
                        old = S[page, h]
                        if old > s:
                            s = old
                        elif old < s:
                            held = cache[page, h, :, :lo] if up else cache[page, h, :lo]
                            was = E4M3[held] * (float(old) / float(s))
                            moved = np.where(held & 127 == 127, held, encode(was))
                            # a zero keeps its sign
                            held[...] = moved
                    S[page, h] = s
                    full = np.zeros((hi - lo, self.R))
                    full[:, :self.hd] = part / float(s)
                    code = encode(full)
                    if up:
                        cache[page, h, :self.hd, lo:hi] = code[:, :self.hd].T
                    else:
                        cache[page, h, lo:hi] = code

    def read(self, b, length):
        """(k, v [length, kvh, hd] float64, present [length])."""
        k, v = np.zeros((length, self.kvh, self.hd)), np.zeros((length, self.kvh, self.hd))
        here = np.zeros(length, bool)
        for p in range(length):
            page, t = self.table[b, p // self.P], p % self.P
            if 0 <= page < self.pages:
                here[p] = True
                k[p] = E4M3[self.k[page, :, t, :self.hd]] * self.ks[page].astype(np.float64)[:, None]
                v[p] = E4M3[self.v[page, :, :self.hd, t]] * self.vs[page].astype(np.float64)[:, None]
        return k, v, here


def attend(cache, b, past, q, scale, causal):
    """q [n, heads, hd] float64 -> (out, the bound's parts): see bound()."""
    n, heads, hd = q.shape
    total, G = past + n, heads // cache.kvh
    k, v, here = cache.read(b, total)
    out, size, lost = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for t in range(n):
            see = here.copy()
            if causal:
                see[past + t + 1:] = False
            if not see.any():
                continue
            for h in range(heads):
                kk, vv = k[see, h // G], v[see, h // G]
                s = (kk @ q[t, h]) * scale
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[t, h], size[t, h] = p @ vv, p @ np.abs(vv)
                # float32 rounding of a score: hd products and sums, the two factors
                lost[t, h] = 2.0 ** -24 * ((hd + 4) * np.max(np.abs(kk) @ np.abs(q[t, h])) * abs(scale) + 4 * np.max(np.abs(s)))
    return out, size, lost


def bound(out, size, lost, keys, dtype):
    """How far an output may be: scores off by `lost` move every weight by twice that;
    exp2 is good to 2 units, sums over the keys round once a term; bfloat16 weights and
    outputs add half a step (2^-8 relative)."""
    rel = 2 * lost * 1.01 + (keys + 16) * 2.0 ** -24
    if dtype == "bf16":
        rel = rel + 2.0 ** -8
    return rel[..., None] * size + np.abs(out) * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) + 1e-30


def sample(z, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One row of float64 logits -> index."""
    ok = np.flatnonzero(z > -np.inf)  # neither NaN nor -inf
    if ok.size == 0:
        return -1
    T = 1.0 if temperature is None else float(temperature)
    m = z[ok].max()
    if not T > 0:
        return int(ok[z[ok] == m][0])
    with np.errstate(invalid="ignore", over="ignore"):
        # an infinite distance stays one at an infinite temperature
        t = np.where(z[ok] == m, 0.0, np.where(np.isinf(z[ok] - m), -np.inf, (z[ok] - m) / T))
    w = np.exp(t)
    order = np.argsort(-z[ok], kind="stable")
    if top_k is not None and top_k > 0:
        order = order[:int(top_k)]
    if top_p is not None and top_p < 1:
        cum = np.cumsum(w[order])
        order = order[:int(np.searchsorted(cum, max(float(top_p), 0.0) * cum[-1], "left")) + 1]
    if min_p is not None:
        order = order[(w[order] >= float(min_p)) | (t[order] == 0)]
    at = np.sort(order)
    cum = np.cumsum(w[at])
    i = int(np.searchsorted(cum, min(max(float(u), 0.0), 1.0) * cum[-1], "right"))
    return int(ok[at[min(i, at.size - 1)]])
