"""Windowed and tree attention over the paged cache, appends at given positions,
the move of kept tokens and rules on logits, restated in float64 numpy from their
definitions: what the GPU tests compare with."""
import numpy as np

import kvref


def window_sight(past, n, sinks, window):
    """[n, past + n]: which keys each new token sees."""
    i, j = np.arange(past, past + n)[:, None], np.arange(past + n)[None]
    return (j <= i) & ((j < sinks) | (j > i - window))


def tree_sight(past, mask):
    """mask [n, n] of the new tokens."""
    n = mask.shape[0]
    return np.concatenate([np.ones((n, past), bool), mask], 1)


def ancestors(parents):
    m = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return np.array(d, np.int32)


def words(masks, stride, junk=None):
    """[N, stride] uint32 of the sequences' masks; bits behind a sequence's tokens: junk's."""
    rows = []
    for m in masks:
        n = m.shape[0]
        full = np.zeros((n, stride * 32), bool) if junk is None else junk.random((n, stride * 32)) < 0.5
        full[:, :n] = m
        rows.append(np.packbits(full, axis=1, bitorder="little"))
    return np.ascontiguousarray(np.concatenate(rows)).view("<u4").reshape(-1, stride)


def attend(cache, b, past, q, scale, sight):
    """q [n, heads, hd] float64 -> (out, size, lost) as kvref.attend's, of the keys in sight."""
    n, heads, hd = q.shape
    G = heads // cache.kvh
    k, v, here = cache.read(b, past + n)
    out, size, lost = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for t in range(n):
            see = here & sight[t]
            if not see.any():
                continue
            for h in range(heads):
                kk, vv = k[see, h // G], v[see, h // G]
                s = (kk @ q[t, h]) * scale
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[t, h], size[t, h] = p @ vv, p @ np.abs(vv)
                lost[t, h] = 2.0 ** -24 * ((hd + 4) * np.max(np.abs(kk) @ np.abs(q[t, h])) * abs(scale) + 4 * np.max(np.abs(s)))
    return out, size, lost


def keep(cache, b, past, n, path):
    """The tokens past + path[i] of a sequence become its tokens past + i."""
    path = [int(p) for p in path]
    if path == list(range(len(path))):
        return
    P, table = cache.P, cache.table[b]
    for data, S, up in ((cache.k, cache.ks, False), (cache.v, cache.vs, True)):
        for h in range(cache.kvh):
            come = []
            for p in path:
                page, t = table[(past + p) // P], (past + p) % P
                come.append(((data[page, h, :, t] if up else data[page, h, t]).copy(), float(S[page, h])))
            first = next(i for i, p in enumerate(path) if p != i)
            for j in sorted({(past + i) // P for i in range(first, len(path))}):
                page = table[j]
                mine = [i for i in range(first, len(path)) if (past + i) // P == j]
                s = max([float(S[page, h])] + [come[i][1] for i in mine])
                data[page, h] = scaled(data[page, h], float(S[page, h]) / s)
                S[page, h] = np.float32(s)
                for i in mine:
                    x = scaled(come[i][0], come[i][1] / s)
                    if up:
                        data[page, h, :, (past + i) % P] = x
                    else:
                        data[page, h, (past + i) % P] = x


def scaled(codes, ratio):
    if ratio == 1:
        return codes
    with np.errstate(invalid="ignore"):
        return np.where(codes & 127 == 127, codes, kvref.encode(kvref.E4M3[codes] * ratio))


def adjust(z, tokens=None, prompt=0, repetition=None, frequency=None, presence=None, ids=None, bias=None, allowed=None):
    """One row of float32 logits -> (float64 values, how far float32's roundings may be from them)."""
    z = np.asarray(z, np.float32).astype(np.float64)
    V, off = z.size, np.zeros(z.size)
    step = 2.0 ** -24

    def rounded(x):
        with np.errstate(invalid="ignore"):
            return step * np.abs(x) + 2.0 ** -149

    def held(x):  # float32 has no number there
        return np.where(np.abs(x) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.copysign(np.inf, x), x)

    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        text = np.asarray([] if tokens is None else tokens, np.int64)
        inside = (text >= 0) & (text < V)
        some = np.zeros(V, bool)
        some[text[inside]] = True
        later = np.bincount(text[inside & (np.arange(text.size) >= prompt)], minlength=V).astype(np.float64)
        r = None if repetition is None else float(repetition)
        if r is not None and r > 0:
            z = held(np.where(some, np.where(z > 0, z / r, z * r), z))
            off += np.where(some, rounded(z), 0)
        f, p = float(frequency or 0), float(presence or 0)
        y = held(np.where(later > 0, z - held(f * later), z))
        off += np.where(later > 0, rounded(f * later) + rounded(y), 0)
        z = held(np.where(later > 0, y - p, y))
        off += np.where(later > 0, rounded(z), 0)
        last = {}
        for i, x in zip([] if ids is None else ids, [] if bias is None else bias):
            if 0 <= i < V:
                last[int(i)] = float(x)
        for i, x in last.items():
            z[i] = held(z[i] + x)
            off[i] += rounded(z[i])
    if allowed is not None:
        z = np.where(allowed, z, -np.inf)
    # the sums above bound each step by the value it leaves; what a later step cancels stays
    return z, off
