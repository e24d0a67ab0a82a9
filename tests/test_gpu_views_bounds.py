"""GPU tests of windows, trees, appends at positions and moves at the bounds of what they
take: loose bounds of new tokens, caches whose offsets pass 32 bits, histories of nothing."""
import ctypes as C

import numpy as np
import pytest

import kvref
import viewref
from gpuutil import DBuf, log
from test_gpu_drafts import append_at
from test_gpu_kv_cache import BF16, F32, OnDevice, as_dtype, spread, starts_of, values
from test_gpu_kv_views import case, floats, tree

pytestmark = pytest.mark.gpu


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


@pytest.mark.parametrize("dtype,hd", [("f32", 64), ("bf16", 128), ("bf16", 256), ("f32", 80)])
@pytest.mark.parametrize("view", ["window", "tree"])
def test_loose_bounds_of_new_tokens(dev, view, dtype, hd):
    """Single tokens and short sequences in calls made for many more."""
    rng = np.random.default_rng(hd)
    for new, bound in (([1, 1], 17), ([1, 3], 200), ([5, 1], 700)):
        kw = dict(masks=[tree(rng, n) for n in new]) if view == "tree" else dict(sinks=3, window=40)
        case(dev, dtype, hd, 16, 2, 2, [90, 0], new, max_new=bound, max_len=1000, **kw)


@pytest.mark.parametrize("dtype,G,hd", [("f32", 1, 64), ("f32", 4, 96), ("bf16", 4, 64), ("bf16", 8, 128), ("bf16", 2, 256), ("f32", 3, 128),
                                        ("bf16", 5, 128), ("f32", 8, 192)])
def test_trees_of_every_plan(dev, dtype, G, hd):
    """Rows that a workgroup's waves share, over one tile and many, and rows of their own;
    with and without splits."""
    rng = np.random.default_rng(G + hd)
    for past, new in (([20], [4]), ([700, 40], [24, 7]), ([2300], [40]), ([30, 5, 0], [130, 1, 66]), ([5000], [33])):
        if sum(new) * G * (sum(past) + sum(new)) > 700000:
            continue
        case(dev, dtype, hd, 32, 1, G, past, new, masks=[tree(rng, n) for n in new], seed=len(past))


def test_many_short_trees(dev):
    """So many that no split pays: the plan for a full card."""
    rng = np.random.default_rng(1)
    new = [int(x) for x in rng.integers(0, 9, 300)]
    new[0] = 8
    past = [int(x) for x in rng.integers(0, 40, 300)]
    case(dev, "bf16", 32, 16, 2, 4, past, new, masks=[tree(rng, n) for n in new])
    case(dev, "f32", 32, 16, 2, 4, past, new, sinks=2, window=11)


@pytest.mark.parametrize("dtype,hd,page", [("f32", 32, 16), ("bf16", 128, 64), ("f32", 7, 16), ("bf16", 80, 128)])
def test_append_at_and_keep_with_loose_bounds(dev, dtype, hd, page):
    L, check = _lib()
    rng = np.random.default_rng(hd)
    kvh, heads, past, new = 2, 4, [page - 1, 0, 7], [3, 0, 20]
    N = sum(new)
    pages, table = spread(rng, 3, 3)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    for b in range(3):
        x = rng.normal(size=(2, past[b], kvh, hd))
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    cos, sin = kvref.tables(64, hd)
    (q, q64), (k, k64), (v, v64) = (as_dtype(rng.normal(size=(N, n * hd)), dtype) for n in (heads, kvh, kvh))
    at = rng.integers(0, 64, N).astype(np.int32)
    w = [n * hd for n in (heads, kvh, kvh)]
    bufs = [DBuf(dev, a) for a in (q, k, v, q * 0, cos, sin, at, starts_of(new), np.asarray(past, np.int32), np.zeros(3, np.int32))]
    dq, dk, dv, do, dc, ds, da, st, ln, bad = bufs
    check(dev.h, L.gn_kv_append_at(dev.h, C.byref(on.kv), dq.p, dk.p, dv.p, do.p, w[0], w[1], w[2], w[0], dc.p, ds.p, 64, da.p, st.p,
                                   ln.p, 3, N, 500, heads, F32 if dtype == "f32" else BF16, bad.p))
    s, want = starts_of(new), np.zeros((N, heads, hd))
    for b in range(3):
        r = slice(s[b], s[b + 1])
        c, sn = cos[at[r]][:, None], sin[at[r]][:, None]
        want[r] = kvref.rotate(q64[r].reshape(-1, heads, hd), c, sn)
        ref.append(b, past[b], kvref.rotate(k64[r].reshape(-1, kvh, hd), c, sn), v64[r].reshape(-1, kvh, hd))
    on.same()
    assert np.array_equal(do.get(), as_dtype(want.reshape(N, -1), dtype)[0]) and not bad.get().any()
    paths = [[1, 2], [], [0, 4, 9, 18, 19]]
    keep, counts = np.zeros(N, np.int32), np.array([2, 0, 5], np.int32)
    for b in range(3):
        keep[s[b]:s[b] + counts[b]] = paths[b]
        viewref.keep(ref, b, past[b], new[b], paths[b])
    dk, dn = DBuf(dev, keep), DBuf(dev, counts)
    check(dev.h, L.gn_kv_keep(dev.h, C.byref(on.kv), dk.p, dn.p, st.p, ln.p, 3, N, 1000, bad.p))
    on.same()
    assert not bad.get().any()


def test_offsets_beyond_32_bits(dev):
    """K and V of 6.4 GB each, the pages in use at their end."""
    from goneuron_amd._lib import KVCache
    L, check = _lib()
    rng = np.random.default_rng(4)
    kvh, hd, P, heads, R = 8, 128, 128, 8, 128
    block = kvh * P * R
    pages, used = 49152, 4
    past, new, total = 150, 40, 190
    table = np.arange(pages - used, pages, dtype=np.int32)[[2, 0, 3, 1]].reshape(1, 4)
    small = kvref.Cache(used, P, kvh, hd, table - (pages - used), rng)
    size = pages * block
    assert size > 2 ** 32
    p = [C.c_void_p(), C.c_void_p()]
    for x in p:
        check(dev.h, L.gn_malloc(dev.h, size, C.byref(x)))
    try:
        scales = [DBuf(dev, np.full((pages, kvh), np.nan, np.float32)) for _ in range(2)]
        dt = DBuf(dev, table)
        kv = KVCache(k=p[0], v=p[1], k_scale=scales[0].p, v_scale=scales[1].p, table=dt.p, pages=pages, page_size=P, kv_heads=kvh,
                     head_dim=hd, max_pages=4)
        end = (pages - used) * block
        for x, a in zip(p, (small.k, small.v)):
            check(dev.h, L.gn_memcpy_h2d(dev.h, C.c_void_p(x.value + end), a.ctypes.data, a.nbytes))

        def same():
            for x, a in zip(p, (small.k, small.v)):
                got = np.empty_like(a)
                check(dev.h, L.gn_memcpy_d2h(dev.h, got.ctypes.data, C.c_void_p(x.value + end), got.nbytes))
                assert np.array_equal(got, a)
            for d, a in zip(scales, (small.ks, small.vs)):
                assert np.array_equal(d.get()[pages - used:], a, equal_nan=True)

        cos, sin = kvref.tables(256, hd)
        dc, ds = DBuf(dev, cos), DBuf(dev, sin)
        bad = DBuf(dev, np.zeros(1, np.int32))
        for at0, n in ((0, past), (past, new)):
            (k, k64), (v, v64), (q, q64) = (as_dtype(rng.normal(size=(n, kvh * hd)), "f32") for _ in range(3))
            at = rng.integers(0, 256, n).astype(np.int32)
            bufs = [DBuf(dev, a) for a in (q, k, v, q * 0, at, starts_of([n]), np.array([at0], np.int32))]
            w = kvh * hd
            check(dev.h, L.gn_kv_append_at(dev.h, C.byref(kv), bufs[0].p, bufs[1].p, bufs[2].p, bufs[3].p, w, w, w, w, dc.p, ds.p, 256,
                                           bufs[4].p, bufs[5].p, bufs[6].p, 1, n, n, heads, F32, bad.p))
            c, s = cos[at][:, None], sin[at][:, None]
            small.append(0, at0, kvref.rotate(k64.reshape(n, kvh, hd), c, s), v64.reshape(n, kvh, hd))
        same()
        q64 = values(bufs[3].get(), "f32").reshape(new, heads, hd)
        work = DBuf(dev, np.zeros(max(1, floats(1, new, total, heads, kvh, hd)), np.float32))
        mask = tree(rng, new)
        dm, do = DBuf(dev, viewref.words([mask], 2).view(np.int32)), DBuf(dev, np.zeros((new, w), np.float32))
        for view in ("window", "tree"):
            log(f"{view} at offsets beyond 32 bits")
            if view == "window":
                check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(kv), bufs[3].p, do.p, w, w, bufs[5].p, bufs[6].p, 1, new, new, total,
                                                      heads, 0.1, 5, 90, F32, work.p, bad.p))
                sight = viewref.window_sight(past, new, 5, 90)
            else:
                check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(kv), bufs[3].p, do.p, w, w, dm.p, 2, bufs[5].p, bufs[6].p, 1, new, new,
                                                    total, heads, 0.1, F32, work.p, bad.p))
                sight = viewref.tree_sight(past, mask)
            want, size_, lost = viewref.attend(small, 0, past, q64, float(np.float32(0.1)), sight)
            got = do.get().astype(np.float64).reshape(new, heads, hd)
            assert (np.abs(got - want) <= kvref.bound(want, size_, lost, total, "f32")).all()
        path = np.flatnonzero(mask[new - 1])
        dk, dn = DBuf(dev, np.pad(path, (0, new - len(path))).astype(np.int32)), DBuf(dev, np.array([len(path)], np.int32))
        check(dev.h, L.gn_kv_keep(dev.h, C.byref(kv), dk.p, dn.p, bufs[5].p, bufs[6].p, 1, new, new, bad.p))
        viewref.keep(small, 0, past, new, path)
        same()
        assert not bad.get().any()
    finally:
        for x in p:
            L.gn_free(dev.h, x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_stream_in_a_few_pages(dev, dtype):
    """Two streams that never end: their pages go back to a pool once they have left the
    window, and come again for later tokens.  The answers are those of a cache that holds
    everything, seen through the window; each step's logits come under rules and are drawn
    from, and the draws are the next step's tokens."""
    from test_gpu_drafts import bits, rules
    L, check = _lib()
    rng = np.random.default_rng(15)
    code = F32 if dtype == "f32" else BF16
    heads, kvh, hd, P, B, V, sinks, window, steps = 4, 2, 32, 16, 2, 61, 4, 40, 60
    D, KW = heads * hd, kvh * hd
    E = [rng.normal(size=(V, n)).astype(np.float32) for n in (D, KW, KW)]
    Wo = rng.normal(size=(V, D)).astype(np.float32) * 2
    max_pages = 40
    shadow = kvref.Cache(B * max_pages, P, kvh, hd, np.arange(B * max_pages).reshape(B, max_pages), rng)
    small = kvref.Cache(12, P, kvh, hd, np.full((B, max_pages), -1), rng)
    on = OnDevice(dev, small)
    free = list(range(12))
    table = np.full((B, max_pages), -1, np.int32)
    cos, sin = kvref.tables(max_pages * P, hd)
    dc, ds, dW = DBuf(dev, cos), DBuf(dev, sin), DBuf(dev, Wo)
    past, tokens = [0, 0], [list(rng.integers(0, V, 23)), list(rng.integers(0, V, 3))]
    text, recycled = [[], []], 0
    n = C.c_int64()
    check(None, L.gn_sample_workspace(B, V, C.byref(n)))
    draw = DBuf(dev, np.zeros(n.value, np.float32))
    for step in range(steps):
        new = [len(t) for t in tokens]
        for b in range(B):
            for j in range(max_pages):  # what the coming queries do not see goes back
                if table[b, j] >= 0 and j * P >= sinks and (j + 1) * P <= past[b] - window + 1:
                    free.append(int(table[b, j]))
                    table[b, j] = rng.choice([-1, 99, table[b, j]])
                    if table[b, j] == free[-1]:
                        table[b, j] = -5
            for j in range(past[b] // P, (past[b] + new[b] - 1) // P + 1):
                if table[b, j] < 0 or j * P >= past[b]:
                    if j * P >= past[b]:
                        recycled += step > 0
                        table[b, j] = free.pop(0)
        dt = DBuf(dev, table)
        on.kv.table = dt.p
        ids = np.concatenate(tokens)
        N, mx = len(ids), max(new)
        (q, q64), (k, k64), (v, v64) = (as_dtype(e[ids], dtype) for e in E)
        bufs = [DBuf(dev, a) for a in (q, k, v, q * 0, q * 0, starts_of(new), np.asarray(past, np.int32), np.zeros(B, np.int32))]
        dq, dk, dv, dqo, do, st, ln, bad = bufs
        check(dev.h, L.gn_kv_append(dev.h, C.byref(on.kv), dq.p, dk.p, dv.p, dqo.p, D, KW, KW, D, dc.p, ds.p, max_pages * P, st.p, ln.p,
                                    B, N, mx, heads, code, bad.p))
        check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dqo.p, do.p, D, D, st.p, ln.p, B, N, mx, max_pages * P, heads, 0.2,
                                              sinks, window, code, None, bad.p))
        assert not bad.get().any()
        s, turned, got = starts_of(new), values(dqo.get(), dtype), values(do.get(), dtype)
        for b in range(B):
            r, pos = slice(s[b], s[b + 1]), np.arange(past[b], past[b] + new[b])
            shadow.append(b, past[b], kvref.rotate(k64[r].reshape(-1, kvh, hd), cos[pos][:, None], sin[pos][:, None]),
                          v64[r].reshape(-1, kvh, hd))
            want, size, lost = viewref.attend(shadow, b, past[b], turned[r].reshape(-1, heads, hd), float(np.float32(0.2)),
                                              viewref.window_sight(past[b], new[b], sinks, window))
            lim = kvref.bound(want, size, lost, past[b] + new[b], dtype)
            assert (np.abs(got[r].reshape(-1, heads, hd) - want) <= lim).all(), (step, b)
            text[b] += [int(x) for x in tokens[b]]
        dh, dl = DBuf(dev, got[[s[1] - 1, s[2] - 1]].astype(np.float32)), DBuf(dev, np.zeros((B, V), np.float32))
        check(dev.h, L.gn_gemm(dev.h, 0, 1, B, V, D, 1.0, dh.p, D, dW.p, D, dl.p, V))
        z = dl.get()
        rows = np.zeros((B, 700), np.int32)
        for b in range(B):
            rows[b, :len(text[b])] = text[b]
        ok = rng.random((1, V)) < 0.7
        R, held = rules(dev, tokens=rows, token_lens=np.array([len(t) for t in text], np.int32), repetition=np.full(B, 1.1, np.float32),
                        presence=np.full(B, 0.3, np.float32), allowed=bits(ok), allowed_row=np.array([0, -1], np.int32))
        check(dev.h, L.gn_logits_adjust(dev.h, dl.p, V, dl.p, V, F32, C.byref(R), B, V))
        y = dl.get()
        u = rng.random(B).astype(np.float32)
        du, di = DBuf(dev, u), DBuf(dev, np.zeros(B, np.int32))
        check(dev.h, L.gn_sample(dev.h, dl.p, V, F32, None, None, None, None, du.p, di.p, B, V, draw.p))
        drawn = di.get()
        for b in range(B):
            w, off = viewref.adjust(z[b], text[b], 0, np.float32(1.1), None, np.float32(0.3), allowed=ok[0] if b == 0 else None)
            fine = np.isfinite(w)
            assert np.array_equal(np.isfinite(y[b]), fine) and (np.abs(y[b][fine] - w[fine]) <= off[fine]).all()
            assert drawn[b] == kvref.sample(y[b].astype(np.float64), u[b])
        past = [a + x for a, x in zip(past, new)]
        # a drawn token, and now and then some that a user adds
        tokens = [[int(drawn[b])] + list(rng.integers(0, V, int(rng.integers(0, 12)) if rng.random() < 0.2 else 0)) for b in range(B)]
    assert recycled > 6 and max(past) > 60


@pytest.mark.parametrize("dtype,hd,G,new0", [("f32", 64, 2, 45), ("bf16", 128, 4, 30), ("f32", 192, 2, 20), ("bf16", 96, 2, 70),
                                             ("bf16", 32, 5, 6), ("f32", 128, 3, 33), ("bf16", 256, 2, 12), ("f32", 32, 1, 90)])
@pytest.mark.parametrize("view", ["window", "tree"])
@pytest.mark.parametrize("kind", ["plain", "nan", "missing"])
def test_a_card_full_of_sequences(dev, view, kind, dtype, hd, G, new0):
    """Enough sequences that waves take rows of their own: a few longer ones among many of a
    token or two, with NaN in and out of sight, pages that are not there, and pages that have
    left the windows."""
    rng = np.random.default_rng(hd + new0)
    B, kvh, P = 258, 2, 16
    past, new = [int(x) for x in rng.integers(0, 30, B)], [int(x) for x in rng.integers(0, 3, B)]
    for b, (a, n) in zip((0, 7, 100, 257), ((190, new0), (0, new0), (333, new0 // 2 + 1), (64, 1))):
        past[b], new[b] = a, n

    def spoil(ref):
        if kind == "nan":
            for b in (0, 7, 100):
                for p in {3, 50, past[b] // 2, past[b], past[b] + new[b] - 1}:
                    if p >= past[b] + new[b]:
                        continue
                    page, t = ref.table[b, p // P], p % P
                    ref.v[page, 0, (p * 5) % hd, t] = 0x7f
                    ref.v[page, 1, 2, t] = 0xff
                    if p % 2:
                        ref.k[page, 1, t, 5] = 0x7f
        if kind == "missing":
            ref.table[0, 11] = -1
            ref.table[7, 0] = ref.pages
            ref.table[100, 20] = 2 ** 31 - 1

    kw = dict(masks=[tree(rng, n) for n in new]) if view == "tree" else dict(sinks=5, window=41, gone=kind != "missing")
    bad = case(dev, dtype, hd, P, kvh, G, past, new, spoil=None if kind == "plain" else spoil, **kw)
    assert sorted(np.flatnonzero(bad)) == ([0, 7, 100] if kind == "missing" else [])
