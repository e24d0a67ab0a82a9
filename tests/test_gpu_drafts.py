"""GPU tests of drafted tokens: appends at given positions and the move of the kept ones
byte for byte against float64 restatements (kvref, viewref), and whole steps of drafting
with every operator that takes part."""
import ctypes as C
import math

import numpy as np
import pytest

import kvref
import viewref
from gpuutil import DBuf, log
from test_gpu_kv_cache import BF16, F32, OnDevice, as_dtype, spread, starts_of, values

pytestmark = pytest.mark.gpu


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


def append_at(dev, on, q, k, v, q_out, positions, past, new, heads, dtype, cos, sin, bad=None, gap=0, off=0, rope_len=None):
    """One gn_kv_append_at of rows padded by `gap` columns that start `off` elements into their buffers."""
    L, check = _lib()

    def padded(a):
        if a is None:
            return None, None, 0
        w = a.shape[1] + gap
        full = np.zeros(off + a.shape[0] * w, a.dtype)
        full[off:].reshape(a.shape[0], w)[:, :a.shape[1]] = a
        d = DBuf(dev, full)
        return d, C.c_void_p(d.p.value + off * a.itemsize), w

    (dq, pq, wq), (dk, pk, wk), (dv, pv, wv), (do, po, wo) = (padded(a) for a in (q, k, v, q_out))
    st, ln = DBuf(dev, starts_of(new)), DBuf(dev, np.asarray(past, np.int32))
    at = DBuf(dev, np.asarray(positions, np.int32)) if positions is not None else None
    dc, ds = (DBuf(dev, cos), DBuf(dev, sin)) if cos is not None else (None, None)
    check(dev.h, L.gn_kv_append_at(dev.h, C.byref(on.kv), pq, pk, pv, po, wq, wk, wv, wo, dc.p if dc else None, ds.p if ds else None,
                                   (rope_len or cos.shape[0]) if dc else 0, at.p if at else None, st.p, ln.p, len(past), k.shape[0],
                                   max(list(new) + [1]), heads, F32 if dtype == "f32" else BF16, bad.p if bad else None))
    if do is None:
        return None
    return do.get()[off:].reshape(q_out.shape[0], wo)[:, :q_out.shape[1]]


CASES = [
    # dtype, hd, page, kvh, group, past, new, gap, offset
    ("f32", 32, 16, 8, 1, [0, 5, 15, 16], [1, 1, 1, 1], 0, 0),
    ("bf16", 128, 64, 2, 4, [63, 64, 0, 130], [64, 1, 33, 70], 0, 0),
    ("f32", 80, 32, 3, 2, [0, 7, 31, 40], [70, 0, 1, 33], 0, 0),
    ("bf16", 64, 128, 1, 7, [100, 0], [29, 300], 8, 0),
    ("f32", 7, 16, 2, 2, [3, 0, 14], [20, 1, 2], 3, 1),
    ("bf16", 1, 16, 1, 1, [0, 9], [17, 1], 0, 0),
    ("f32", 256, 128, 1, 2, [10, 127], [119, 3], 0, 0),
    ("bf16", 192, 16, 2, 1, [0], [49], 1, 3),
    ("bf16", 72, 32, 4, 1, [32, 0, 31], [32, 32, 2], 0, 0),
]


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new,gap,off", CASES)
def test_append_at_is_the_definition_byte_for_byte(dev, dtype, hd, page, kvh, G, past, new, gap, off):
    log(f"append_at {dtype} hd={hd} page={page} kvh={kvh} past={past} new={new}")
    rng = np.random.default_rng(hd * 37 + page)
    B, heads, N = len(past), kvh * G, sum(new)
    max_pages = max(-(-(a + b) // page) for a, b in zip(past, new)) + 1
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    cos, sin = kvref.tables(500, hd)
    for b in range(B):
        x = rng.normal(size=(2, past[b], kvh, hd)) * 0.5
        x[:, :, ::2] *= 0.01
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    tail = 2  # rows behind the last sequence
    q, q64 = as_dtype(rng.normal(size=(N + tail, heads * hd)), dtype)
    k, k64 = as_dtype(rng.normal(size=(N + tail, kvh * hd)) * 2, dtype)
    v, v64 = as_dtype(rng.normal(size=(N + tail, kvh * hd)), dtype)
    mark, _ = as_dtype(np.full((N + tail, heads * hd), 77.0), dtype)
    at = rng.integers(0, 500, N + tail).astype(np.int32)
    at[N:] = -1
    bad = DBuf(dev, np.zeros(B, np.int32))
    got = append_at(dev, on, q, k, v, mark, at, past, new, heads, dtype, cos, sin, bad, gap, off)
    st, want = starts_of(new), np.full((N + tail, heads, hd), 77.0)
    for b in range(B):
        r = slice(st[b], st[b + 1])
        c, s = cos[at[r]][:, None], sin[at[r]][:, None]
        want[r] = kvref.rotate(q64[r].reshape(-1, heads, hd), c, s)
        ref.append(b, past[b], kvref.rotate(k64[r].reshape(-1, kvh, hd), c, s), v64[r].reshape(-1, kvh, hd))
    on.same()
    w, _ = as_dtype(want.reshape(N + tail, -1), dtype)
    assert np.array_equal(got, w) and not bad.get().any()


@pytest.mark.parametrize("dtype,hd,new", [("f32", 32, [5, 3, 1]), ("bf16", 7, [20, 2, 1]), ("f32", 1, [3, 2, 1]), ("bf16", 64, [1, 1, 1]),
                                          ("f32", 5, [1, 1, 1])])
def test_positions_outside_the_tables(dev, dtype, hd, new):
    rng = np.random.default_rng(hd)
    kvh, heads, N, past = 2, 4, sum(new), [3, 0, 20]
    pages, table = spread(rng, 3, 3)
    ref = kvref.Cache(pages, 16, kvh, hd, table, rng)
    for b in range(3):
        x = rng.normal(size=(2, past[b], kvh, hd))
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    cos, sin = kvref.tables(50, hd)
    if hd == 1:  # nothing turns, yet the tables are there
        cos = sin = np.zeros((50, 1), np.float32)
    (q, q64), (k, k64), (v, v64) = (as_dtype(rng.normal(size=(N, n * hd)), dtype) for n in (heads, kvh, kvh))
    at = rng.integers(0, 40, N).astype(np.int32)
    lost = [0, N - 2]
    at[lost] = [-1, 40] if new[0] > 1 else [2 ** 31 - 1, -2 ** 31]
    bad = DBuf(dev, np.zeros(3, np.int32))
    got = append_at(dev, on, q, k, v, q * 0, at, past, new, heads, dtype, cos, sin, bad, rope_len=40)
    st, want = starts_of(new), np.zeros((N, heads, hd))
    for b in range(3):
        r = np.arange(st[b], st[b + 1])
        p = np.where(np.isin(r, lost), 0, at[r])
        c, s = cos[p][:, None], sin[p][:, None]
        if hd == 1:
            c, s = c[..., :0], s[..., :0]
        y, z = kvref.rotate(q64[r].reshape(-1, heads, hd), c, s), kvref.rotate(k64[r].reshape(-1, kvh, hd), c, s)
        y[np.isin(r, lost)], z[np.isin(r, lost)] = np.nan, np.nan
        want[r] = y
        ref.append(b, past[b], z, v64[r].reshape(-1, kvh, hd))
    on.same()
    got, want = values(got, dtype), want.reshape(N, -1)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and bad.get().tolist() == [1, 1, 0]
    fine = ~np.isnan(want)
    w, _ = as_dtype(np.where(fine, want, 0), dtype)
    assert np.array_equal(got[fine], values(w, dtype)[fine])


def test_append_at_without_rotation_or_queries(dev):
    rng = np.random.default_rng(2)
    pages, table = spread(rng, 1, 3)
    ref = kvref.Cache(pages, 16, 2, 32, table, rng)
    on = OnDevice(dev, ref)
    (k, k64), (v, v64) = (as_dtype(rng.normal(size=(20, 64)), "f32") for _ in range(2))
    append_at(dev, on, None, k, v, None, None, [0], [20], 2, "f32", None, None)   # no tables: no positions
    ref.append(0, 0, k64.reshape(-1, 2, 32), v64.reshape(-1, 2, 32))
    on.same()
    cos, sin = kvref.tables(8, 32)
    at = np.array([7, 7, 0], np.int32)
    append_at(dev, on, None, k[:3], v[:3], None, at, [20], [3], 2, "f32", cos, sin)
    ref.append(0, 20, kvref.rotate(k64[:3].reshape(-1, 2, 32), cos[at][:, None], sin[at][:, None]), v64[:3].reshape(-1, 2, 32))
    on.same()


# ---------------------------------------------------------------- keep
KEEPS = [
    # hd, page, kvh, past, new, counts
    (32, 16, 8, [0, 5, 15, 16], [16, 16, 16, 16], [5, 0, 16, 1]),
    (128, 64, 2, [63, 64, 0, 130], [64, 1, 33, 100], [9, 1, 20, 50]),
    (80, 32, 3, [0, 7, 31, 40], [70, 0, 1, 33], [40, 0, 0, 2]),
    (64, 128, 1, [100, 0], [29, 400], [7, 300]),
    (7, 16, 2, [3, 0, 14], [20, 1, 60], [19, 1, 37]),
    (256, 128, 1, [10, 127], [300, 3], [250, 2]),
    (192, 16, 2, [0], [100], [33]),
    (1, 16, 1, [9], [300], [290]),
]


@pytest.mark.parametrize("hd,page,kvh,past,new,counts", KEEPS)
def test_keep_is_the_definition_byte_for_byte(dev, hd, page, kvh, past, new, counts):
    log(f"keep hd={hd} page={page} kvh={kvh} past={past} new={new} counts={counts}")
    L, check = _lib()
    rng = np.random.default_rng(hd + page)
    B, N = len(past), sum(new)
    max_pages = max(-(-(a + b) // page) for a, b in zip(past, new)) + 1
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    for b in range(B):
        n = past[b] + new[b]
        x = rng.normal(size=(2, n, kvh, hd))
        for p in range(0, n, page):  # blocks of unlike scales, in any order
            x[:, p:p + page] *= 2.0 ** rng.integers(-6, 6)
            ref.append(b, p, x[0, p:p + page], x[1, p:p + page])
    if hd == 32:
        ref.k[table[0, 0], 1, 3, 4] = 0x7f    # NaN moves as it is
        ref.v[table[0, 0], 2, 5, 3] = 0xff
    on = OnDevice(dev, ref)
    paths = [np.sort(rng.choice(new[b], counts[b], replace=False)) for b in range(B)]
    st, keep = starts_of(new), np.full(N + 1, -9, np.int32)
    for b in range(B):
        keep[st[b]:st[b] + counts[b]] = paths[b]
    bufs = [DBuf(dev, a) for a in (keep, np.asarray(counts, np.int32), st, np.asarray(past, np.int32), np.zeros(B, np.int32))]
    check(dev.h, L.gn_kv_keep(dev.h, C.byref(on.kv), *(x.p for x in bufs[:4]), B, N, max(new), bufs[4].p))
    for b in range(B):
        viewref.keep(ref, b, past[b], new[b], paths[b])
    on.same()
    assert not bufs[4].get().any()


def test_keep_flags_what_it_cannot_move(dev):
    L, check = _lib()
    rng = np.random.default_rng(3)
    B, page, hd, kvh = 12, 16, 32, 2
    pages, table = spread(rng, B, 3)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    new = [20] * B
    for b in range(B):
        x = rng.normal(size=(2, 25, kvh, hd))
        ref.append(b, 0, x[0], x[1])
    ref.table[5, 1] = -1                 # a page that a kept token comes from
    ref.table[6, 0] = pages              # a page that one goes to
    past, counts = [5] * B, [3] * B
    past[7], past[8] = -1, 30            # before 0, beyond the table
    counts[9], counts[10] = 21, -1       # more than there are, fewer than none
    paths = [[0, 5, 19]] * B
    paths[1] = [3, 3, 4]                 # the same twice
    paths[2] = [4, 3, 5]                 # falling
    paths[3] = [0, 1, 20]                # behind the last
    paths[4] = [-1, 1, 2]
    paths[11] = [0, 1, 2]                # all in their places: nothing moves
    st, keep = starts_of(new), np.zeros(sum(new), np.int32)
    for b in range(B):
        keep[st[b]:st[b] + 3] = paths[b]
    on = OnDevice(dev, ref)
    bufs = [DBuf(dev, a) for a in (keep, np.asarray(counts, np.int32), st, np.asarray(past, np.int32), np.zeros(B, np.int32))]
    check(dev.h, L.gn_kv_keep(dev.h, C.byref(on.kv), *(x.p for x in bufs[:4]), B, sum(new), 20, bufs[4].p))
    viewref.keep(ref, 0, 5, 20, paths[0])
    on.same()
    assert bufs[4].get().tolist() == [0] + [1] * 10 + [0]
    # more tokens than announced; no rows at all
    for N, mn in ((sum(new), 19), (0, 20)):
        bufs[4] = DBuf(dev, np.zeros(B, np.int32))
        check(dev.h, L.gn_kv_keep(dev.h, C.byref(on.kv), *(x.p for x in bufs[:4]), B, N, mn, bufs[4].p))
        on.same()
        assert bufs[4].get().tolist() == [1] * B


def test_refusals(dev):
    from goneuron_amd._lib import KVCache
    L, _ = _lib()
    ref = kvref.Cache(4, 16, 2, 32, np.arange(4).reshape(1, 4), np.random.default_rng(6))
    on = OnDevice(dev, ref)
    x, i = DBuf(dev, np.zeros(4096, np.float32)), DBuf(dev, np.zeros(8, np.int32))
    fields = {n: getattr(on.kv, n) for n, _ in KVCache._fields_}

    def app(q=x.p, k=x.p, v=x.p, qo=x.p, qs=64, ks=64, vs=64, qos=64, cos=x.p, sin=x.p, rl=64, at=i.p, st=i.p, ln=i.p, B=1, N=1, mn=1,
            heads=2, dtype=0, **kv):
        return L.gn_kv_append_at(dev.h, C.byref(KVCache(**{**fields, **kv})), q, k, v, qo, qs, ks, vs, qos, cos, sin, rl, at, st, ln,
                                 B, N, mn, heads, dtype, None)

    def kee(keep=i.p, counts=i.p, st=i.p, ln=i.p, B=1, N=1, mn=1, **kv):
        return L.gn_kv_keep(dev.h, C.byref(KVCache(**{**fields, **kv})), keep, counts, st, ln, B, N, mn, None)

    assert app() == 0 and kee() == 0
    odd = C.c_void_p(x.p.value + 2)
    for f in (app, kee):
        for kw in (dict(page_size=48), dict(pages=0), dict(kv_heads=0), dict(max_pages=0), dict(v_scale=None), dict(k_scale=None),
                   dict(table=None), dict(st=None), dict(ln=None), dict(B=-1), dict(N=-1), dict(mn=-1), dict(head_dim=0)):
            assert f(**kw) < 0, (f.__name__, kw)
        assert f(head_dim=257) == -4 and f(B=70000) == -4 and f(mn=1 << 27) == -4
        assert f(B=0) == 0 and f(N=0) == 0 and f(mn=0) == 0
    for kw in (dict(cos=None), dict(sin=None), dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(qs=63), dict(ks=63),
               dict(vs=63), dict(qos=63), dict(qos=128), dict(at=None), dict(rl=0), dict(rl=-1), dict(dtype=2), dict(heads=3),
               dict(heads=0), dict(q=odd, qo=odd)):
        assert app(**kw) == -1, kw
    assert app(cos=None, sin=None, at=None, rl=0) == 0 and app(rl=1) == 0
    assert kee(keep=None) == -1 and kee(counts=None) == -1 and kee(k=None) == -1 and kee(v=None) == -1
    on.same()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_of_drafting_together(dev, dtype):
    """Prompts, then drafted trees step after step: appended at their depths, attended to,
    their logits put under rules and drawn from, and the path that a token of each tree
    takes kept.  The cache, the answers and the draws are those of the definitions, and in
    the end the cache holds what a program without drafts would have cached."""
    L, check = _lib()
    rng = np.random.default_rng(12)
    code = F32 if dtype == "f32" else BF16
    V, heads, kvh, page, B, hd = 97, 4, 2, 16, 3, 16
    D = heads * hd
    W = (rng.normal(size=(V, D)) * 2).astype(np.float32)
    rowq, rowk, rowv = (rng.normal(size=(V, n * hd)).astype(np.float32) for n in (heads, kvh, kvh))
    pages, table = spread(rng, B, 8)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    on = OnDevice(dev, ref)
    cos, sin = kvref.tables(128, hd)
    dW, dcos, dsin = DBuf(dev, W), DBuf(dev, cos), DBuf(dev, sin)
    past = [0, 0, 0]
    text = [[], [], []]
    n = C.c_int64()
    check(None, L.gn_sample_workspace(64, V, C.byref(n)))
    draw_work = DBuf(dev, np.zeros(n.value, np.float32))
    work = DBuf(dev, np.zeros(max(1, floats_of(B, 12, 128, heads, kvh, hd)), np.float32))
    for step in range(8):
        new = [5, 17, 1] if step == 0 else [int(rng.integers(1, 12)) for _ in range(B)]
        max_new, N = max(new), sum(new)
        if step == 0:
            parents = [list(range(-1, x - 1)) for x in new]  # a prompt is a chain
            work0 = DBuf(dev, np.zeros(max(1, floats_of(B, 17, 128, heads, kvh, hd)), np.float32))
        else:
            parents = [[-1] + [int(rng.integers(-1, i)) for i in range(1, x)] for x in new]
        toks = [rng.integers(0, V, x) for x in new]
        at = np.concatenate([past[b] + viewref.depths(parents[b]) for b in range(B)]).astype(np.int32)
        ids = np.concatenate(toks)
        (q, q64), (k, k64), (v, v64) = (as_dtype(m[ids], dtype) for m in (rowq, rowk, rowv))
        bufs = [DBuf(dev, a) for a in (q, k, v, q * 0, at, starts_of(new), np.asarray(past, np.int32), np.zeros(B, np.int32))]
        dq, dk, dv, dqo, dat, st, ln, bad = bufs
        check(dev.h, L.gn_kv_append_at(dev.h, C.byref(on.kv), dq.p, dk.p, dv.p, dqo.p, D, kvh * hd, kvh * hd, D, dcos.p, dsin.p, 128,
                                       dat.p, st.p, ln.p, B, N, max_new, heads, code, bad.p))
        masks = [viewref.ancestors(p) for p in parents]
        dm, do = DBuf(dev, viewref.words(masks, 1).view(np.int32)), DBuf(dev, q * 0)
        check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dqo.p, do.p, D, D, dm.p, 1, st.p, ln.p, B, N, max_new, 128, heads,
                                            0.25, code, (work0 if step == 0 else work).p, bad.p))
        s, turned = starts_of(new), values(dqo.get(), dtype)
        got = values(do.get(), dtype)
        for b in range(B):
            r = slice(s[b], s[b + 1])
            c, sn = cos[at[r]][:, None], sin[at[r]][:, None]
            ref.append(b, past[b], kvref.rotate(k64[r].reshape(-1, kvh, hd), c, sn), v64[r].reshape(-1, kvh, hd))
            want, size, lost = viewref.attend(ref, b, past[b], turned[r].reshape(-1, heads, hd), 0.25,
                                              viewref.tree_sight(past[b], masks[b]))
            lim = kvref.bound(want, size, lost, past[b] + new[b], dtype)
            assert (np.abs(got[r].reshape(-1, heads, hd) - want) <= lim).all()
        on.same()
        assert not bad.get().any()
        # logits of every drafted token, under each row's own text, and a draw
        dh, dl = DBuf(dev, got.astype(np.float32)), DBuf(dev, np.zeros((N, V), np.float32))
        check(dev.h, L.gn_gemm(dev.h, 0, 1, N, V, D, 1.0, dh.p, D, dW.p, D, dl.p, V))
        z = dl.get()
        rows, lens = np.zeros((N, 200), np.int32), np.zeros(N, np.int32)
        for b in range(B):
            for i in range(new[b]):
                t = text[b] + [int(x) for x in toks[b][np.flatnonzero(masks[b][i])]]
                rows[s[b] + i, :len(t)], lens[s[b] + i] = t, len(t)
        allowed = rng.random((N, V)) < 0.5
        allowed[0] = False
        rep, freq = np.full(N, 1.2, np.float32), np.full(N, 0.1, np.float32)
        R, keepalive = rules(dev, repetition=rep, frequency=freq, tokens=rows, token_lens=lens,
                             allowed=bits(allowed))
        check(dev.h, L.gn_logits_adjust(dev.h, dl.p, V, dl.p, V, F32, C.byref(R), N, V))
        zz = dl.get()
        for i in range(N):
            w, off = viewref.adjust(z[i], rows[i, :lens[i]], 0, rep[i], freq[i], None, allowed=allowed[i])
            fine = np.isfinite(w)
            assert np.array_equal(np.isfinite(zz[i]), fine) and (np.abs(zz[i][fine] - w[fine]) <= off[fine]).all()
        u = rng.random(N).astype(np.float32)
        du, di = DBuf(dev, u), DBuf(dev, np.zeros(N, np.int32))
        check(dev.h, L.gn_sample(dev.h, dl.p, V, F32, None, None, None, None, du.p, di.p, N, V, draw_work.p))
        drawn = di.get()
        assert drawn[0] == -1
        for i in range(1, N):
            assert drawn[i] == kvref.sample(zz[i].astype(np.float64), u[i])
        # one path of each tree is right
        keep, counts = np.zeros(N, np.int32), np.zeros(B, np.int32)
        for b in range(B):
            i = new[b] - 1 if step == 0 else int(rng.integers(-1, new[b]))
            path = np.flatnonzero(masks[b][i]) if i >= 0 else np.zeros(0, int)
            keep[s[b]:s[b] + len(path)], counts[b] = path, len(path)
            viewref.keep(ref, b, past[b], new[b], path)
            text[b] += [int(x) for x in toks[b][path]]
        dkeep, dcount = DBuf(dev, keep), DBuf(dev, counts)
        check(dev.h, L.gn_kv_keep(dev.h, C.byref(on.kv), dkeep.p, dcount.p, st.p, ln.p, B, N, max_new, bad.p))
        on.same()
        assert not bad.get().any()
        past = [a + int(x) for a, x in zip(past, counts)]
    for b in range(B):  # what is cached: each token of the text at its place, to 8 bits
        assert past[b] == len(text[b])
        k, v, here = ref.read(b, past[b])
        _, k64 = as_dtype(rowk[text[b]], dtype)
        pos = np.arange(past[b])
        want = kvref.rotate(k64.reshape(-1, kvh, hd), cos[pos][:, None], sin[pos][:, None])
        # half a step (2^-4 relative), twice where a scale grew after, or of the smallest number
        small = 2.0 ** -9 * ref.ks[ref.table[b, pos // page]].astype(np.float64)[..., None]
        assert here.all() and (np.abs(k - want) <= 2.0 ** -4 * np.abs(want) * 1.07 + 1.5 * small).all()


def floats_of(B, max_new, max_len, heads, kvh, hd):
    L, check = _lib()
    n = C.c_int64()
    check(None, L.gn_kv_attention_workspace(B, max_new, max_len, heads, kvh, hd, C.byref(n)))
    return n.value


def bits(allowed):
    """[rows, V] truth values -> [rows, words] int32."""
    rows, V = allowed.shape
    full = np.zeros((rows, -(-V // 32) * 32), bool)
    full[:, :V] = allowed
    return np.ascontiguousarray(np.packbits(full, axis=1, bitorder="little")).view("<i4").reshape(rows, -1)


def rules(dev, tokens=None, bias=None, bias_ids=None, allowed=None, **more):
    """(gn_logit_rules of host arrays, what has to live as long)."""
    from goneuron_amd._lib import LogitRules
    held = {k: DBuf(dev, a) for k, a in dict(tokens=tokens, bias=bias, bias_ids=bias_ids, allowed=allowed, **more).items()
            if a is not None}
    kw = {k: d.p for k, d in held.items()}
    if tokens is not None:
        kw["tokens_stride"] = tokens.shape[1]
    if bias is not None:
        kw["bias_stride"] = bias.shape[1]
    if allowed is not None:
        kw.update(allowed_stride=allowed.shape[1], allowed_rows=allowed.shape[0])
    return LogitRules(**kw), held


def test_two_drafts_at_once(gn, dev):
    """Two contexts append, attend, adjust and keep in turn without a wait between."""
    other = gn.HIPDevice(0)
    try:
        on_two_streams(dev, other)
    finally:
        other.close()


def on_two_streams(dev, other):
    L, check = _lib()
    rng = np.random.default_rng(19)
    hd, kvh, H, P, T, past, V = 64, 2, 8, 32, 40, 100, 5000
    parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, T)]
    mask = viewref.ancestors(parents)
    path = np.flatnonzero(mask[T - 1])
    runs = []
    for d in (dev, other):
        ref = kvref.Cache(10, P, kvh, hd, rng.permutation(10)[:6].reshape(1, 6).astype(np.int32), rng)
        x = rng.normal(size=(2, past, kvh, hd))
        ref.append(0, 0, x[0], x[1])
        k, v, q = (rng.normal(size=(T, n * hd)).astype(np.float32) for n in (kvh, kvh, H))
        z = rng.normal(size=(2, V)).astype(np.float32)
        ok = rng.random((1, V)) < 0.3
        R, held = rules(d, allowed=bits(ok), allowed_row=np.array([0, -1], np.int32))
        runs.append(dict(d=d, ref=ref, on=OnDevice(d, ref), host=(k, v, q), k=DBuf(d, k), v=DBuf(d, v), q=DBuf(d, q), R=R, held=held,
                         out=DBuf(d, q * 0), st=DBuf(d, np.array([0, T], np.int32)), ln=DBuf(d, np.array([past], np.int32)),
                         m=DBuf(d, viewref.words([mask], 2).view(np.int32)), z=z, dz=DBuf(d, z), dy=DBuf(d, z * 0), ok=ok,
                         keep=DBuf(d, np.pad(path, (0, T - len(path))).astype(np.int32)), count=DBuf(d, np.array([len(path)], np.int32)),
                         work=DBuf(d, np.zeros(max(1, floats_of(1, T, 256, H, kvh, hd)), np.float32))))
    for r in runs:
        check(r["d"].h, L.gn_kv_append_at(r["d"].h, C.byref(r["on"].kv), None, r["k"].p, r["v"].p, None, 0, kvh * hd, kvh * hd, 0, None,
                                          None, 0, None, r["st"].p, r["ln"].p, 1, T, T, H, F32, None))
    for _ in range(3):
        for r in runs:
            check(r["d"].h, L.gn_kv_attention_tree(r["d"].h, C.byref(r["on"].kv), r["q"].p, r["out"].p, H * hd, H * hd, r["m"].p, 2,
                                                   r["st"].p, r["ln"].p, 1, T, T, 256, H, 0.125, F32, r["work"].p, None))
            check(r["d"].h, L.gn_logits_adjust(r["d"].h, r["dz"].p, V, r["dy"].p, V, F32, C.byref(r["R"]), 2, V))
    for r in runs:
        check(r["d"].h, L.gn_kv_keep(r["d"].h, C.byref(r["on"].kv), r["keep"].p, r["count"].p, r["st"].p, r["ln"].p, 1, T, T, None))
    for r in runs:
        k, v, q = r["host"]
        r["ref"].append(0, past, k.reshape(T, kvh, hd).astype(np.float64), v.reshape(T, kvh, hd).astype(np.float64))
        want, size, lost = viewref.attend(r["ref"], 0, past, q.reshape(T, H, hd).astype(np.float64), 0.125, viewref.tree_sight(past, mask))
        got = r["out"].get().reshape(T, H, hd).astype(np.float64)
        assert (np.abs(got - want) <= kvref.bound(want, size, lost, past + T, "f32")).all()
        viewref.keep(r["ref"], 0, past, T, path)
        r["on"].same()
        y = r["dy"].get()
        assert np.array_equal(y[1], r["z"][1]) and np.array_equal(y[0], np.where(r["ok"][0], r["z"][0], -np.inf))
