"""GPU tests of the paged 8-bit cache: gn_kv_append byte for byte and
gn_kv_attention within derived bounds against float64 restatements (kvref),
gn_mha_cached_forward against the layer's formulas, and a few steps of all of
them with gn_sample as a generating program runs them."""
import ctypes as C
import math

import numpy as np
import pytest

import kvref
from gpuutil import DBuf, log

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 1


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


def as_dtype(x, dtype):
    """float32 values -> (device array, the values it holds as float64)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x.astype(np.float64)
    b = kvref.bf16_bits(x)
    return b, kvref.bf16_value(b).astype(np.float64)


def values(a, dtype):
    return (a if dtype == "f32" else kvref.bf16_value(a)).astype(np.float64)


class OnDevice:
    """A kvref.Cache's memory on the GPU."""

    def __init__(self, dev, ref):
        from goneuron_amd._lib import KVCache
        self.ref = ref
        self.k, self.v = DBuf(dev, ref.k), DBuf(dev, ref.v)
        self.ks, self.vs, self.table = DBuf(dev, ref.ks), DBuf(dev, ref.vs), DBuf(dev, ref.table)
        self.kv = KVCache(k=self.k.p, v=self.v.p, k_scale=self.ks.p, v_scale=self.vs.p, table=self.table.p,
                          pages=ref.pages, page_size=ref.P, kv_heads=ref.kvh, head_dim=ref.hd,
                          max_pages=ref.table.shape[1])

    def same(self):
        for name, d, r in (("k", self.k, self.ref.k), ("v", self.v, self.ref.v)):
            got = d.get()
            assert np.array_equal(got, r), (name, int((got != r).sum()), np.argwhere(got != r)[:4].tolist())
        for name, d, r in (("k_scale", self.ks, self.ref.ks), ("v_scale", self.vs, self.ref.vs)):
            assert np.array_equal(d.get(), r, equal_nan=True), name


def spread(rng, B, max_pages, extra=2):
    """Page tables over pages in any order."""
    pages = B * max_pages + extra
    return pages, rng.permutation(pages)[:B * max_pages].reshape(B, max_pages).astype(np.int32)


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def append(dev, on, q, k, v, past, new, heads, dtype, cos=None, sin=None, q_out=None, gap=0, bad=None, N=None,
           max_new=None, starts=None, rope_len=None, off=0):
    """One gn_kv_append; q, k, v: device-typed arrays of rows (may be padded by `gap`
    columns, and start `off` elements into their buffer)."""
    L, check = _lib()
    ref = on.ref
    N = N if N is not None else k.shape[0]

    def padded(a):
        if a is None:
            return None, None, 0
        w = a.shape[1] + gap
        full = np.zeros(off + a.shape[0] * w, a.dtype)
        full[off:].reshape(a.shape[0], w)[:, :a.shape[1]] = a
        d = DBuf(dev, full)
        return d, C.c_void_p(d.p.value + off * a.itemsize), w

    dq, pq, wq = padded(q)
    dk, pk, wk = padded(k)
    dv, pv, wv = padded(v)
    do, po, wo = padded(q_out)
    st = DBuf(dev, starts if starts is not None else starts_of(new))
    ln = DBuf(dev, np.asarray(past, np.int32))
    dc = DBuf(dev, cos) if cos is not None else None
    ds = DBuf(dev, sin) if sin is not None else None
    B = len(past)
    check(dev.h, L.gn_kv_append(dev.h, C.byref(on.kv), pq, pk, pv, po, wq, wk, wv, wo, dc.p if dc else None,
                                ds.p if ds else None, (rope_len if rope_len is not None else cos.shape[0]) if dc else 0,
                                st.p, ln.p, B, N, max_new if max_new is not None else max(list(new) + [1]), heads,
                                F32 if dtype == "f32" else BF16, bad.p if bad else None))
    if do is None:
        return None
    full = do.get()
    return full[off:].reshape(q_out.shape[0], wo)[:, :q_out.shape[1]]


CASES = [
    # dtype, hd, page, kvh, group, past, new, gap, offset
    ("f32", 32, 16, 8, 1, [0, 5, 15, 16], [1, 1, 1, 1], 0, 0),
    ("bf16", 128, 64, 2, 4, [63, 64, 0, 130], [1, 1, 1, 1], 0, 0),
    ("f32", 80, 32, 3, 2, [0, 7, 31, 40], [70, 0, 1, 33], 0, 0),
    ("bf16", 64, 128, 1, 7, [100, 0], [29, 300], 8, 0),
    ("f32", 7, 16, 2, 2, [3, 0, 14], [20, 1, 2], 3, 1),          # odd head: the last column does not turn
    ("bf16", 1, 16, 1, 1, [0, 9], [17, 1], 0, 0),
    ("f32", 256, 128, 1, 2, [10, 127], [119, 3], 0, 0),           # the largest block
    ("bf16", 192, 16, 2, 1, [0], [49], 1, 3),                     # rows at odd addresses
    ("f32", 100, 64, 2, 1, [1, 2, 3], [64, 62, 61], 0, 0),
    ("bf16", 72, 32, 4, 1, [32, 0, 31], [32, 32, 2], 0, 0),
]


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new,gap,off", CASES)
def test_append_is_the_definition_byte_for_byte(dev, dtype, hd, page, kvh, G, past, new, gap, off):
    log(f"append {dtype} hd={hd} page={page} kvh={kvh} past={past} new={new}")
    rng = np.random.default_rng(hd * 31 + page)
    B, heads, N = len(past), kvh * G, sum(new)
    max_pages = max(-(-(a + b) // page) for a, b in zip(past, new)) + 1
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    cos, sin = kvref.tables(max_pages * page, hd)
    hist = [rng.normal(size=(2, n, kvh, hd)) * 0.5 for n in past]
    for b in range(B):  # what earlier steps left, at a smaller scale for some heads
        hist[b][:, :, ::2] *= 0.01
        ref.append(b, 0, hist[b][0], hist[b][1])
    on = OnDevice(dev, ref)
    tail = 2  # rows behind the last sequence
    q, q64 = as_dtype(rng.normal(size=(N + tail, heads * hd)), dtype)
    k, k64 = as_dtype(rng.normal(size=(N + tail, kvh * hd)) * 2, dtype)
    v, v64 = as_dtype(rng.normal(size=(N + tail, kvh * hd)), dtype)
    mark, _ = as_dtype(np.full((N + tail, heads * hd), 77.0), dtype)
    got = append(dev, on, q, k, v, past, new, heads, dtype, cos, sin, mark, gap, off=off)
    st, want = starts_of(new), np.full((N + tail, heads, hd), 77.0)
    for b in range(B):
        r = slice(st[b], st[b + 1])
        pos = np.arange(past[b], past[b] + new[b])
        c, s = cos[pos][:, None], sin[pos][:, None]
        want[r] = kvref.rotate(q64[r].reshape(-1, heads, hd), c, s)
        ref.append(b, past[b], kvref.rotate(k64[r].reshape(-1, kvh, hd), c, s), v64[r].reshape(-1, kvh, hd))
    on.same()
    want = want.reshape(N + tail, -1)
    if dtype == "bf16":
        want = kvref.bf16_value(kvref.bf16_bits(want.astype(np.float32)))
    assert np.array_equal(values(got, dtype), want)


def test_append_without_rotation_queries_or_in_place(dev):
    rng = np.random.default_rng(3)
    pages, table = spread(rng, 2, 3)
    cos, sin = kvref.tables(96, 48)
    for rotate, with_q in ((False, True), (False, False), (True, False)):
        ref = kvref.Cache(pages, 32, 2, 48, table, rng)
        on = OnDevice(dev, ref)
        k, k64 = as_dtype(rng.normal(size=(40, 96)), "f32")
        v, v64 = as_dtype(rng.normal(size=(40, 96)), "f32")
        q, q64 = as_dtype(rng.normal(size=(40, 4 * 48)), "f32")
        out = append(dev, on, q if with_q else None, k, v, [0, 0], [33, 7], 4, "f32", cos if rotate else None,
                     sin if rotate else None, q * 0 if with_q else None)
        for b, r in ((0, slice(0, 33)), (1, slice(33, 40))):
            kk = k64[r].reshape(-1, 2, 48)
            if rotate:
                kk = kvref.rotate(kk, cos[:kk.shape[0], None], sin[:kk.shape[0], None])
            ref.append(b, 0, kk, v64[r].reshape(-1, 2, 48))
        on.same()
        if with_q:
            assert np.array_equal(out, q)
    # queries rotated where they lie
    L, check = _lib()
    ref = kvref.Cache(pages, 32, 2, 48, table, rng)
    on = OnDevice(dev, ref)
    dq, dk, dv = DBuf(dev, q), DBuf(dev, k), DBuf(dev, v)
    dc, ds, st, ln = DBuf(dev, cos), DBuf(dev, sin), DBuf(dev, starts_of([33, 7])), DBuf(dev, np.zeros(2, np.int32))
    check(dev.h, L.gn_kv_append(dev.h, C.byref(on.kv), dq.p, dk.p, dv.p, dq.p, 192, 96, 96, 192, dc.p, ds.p, 96, st.p, ln.p,
                                2, 40, 33, 4, F32, None))
    pos = np.concatenate([np.arange(33), np.arange(7)])
    assert np.array_equal(dq.get(), kvref.rotate(q64.reshape(40, 4, 48), cos[pos][:, None], sin[pos][:, None])
                          .reshape(40, -1).astype(np.float32))


def test_append_numbers_that_are_not_finite_large_and_small(dev):
    rng = np.random.default_rng(4)
    pages, table = spread(rng, 1, 4)
    ref = kvref.Cache(pages, 16, 1, 32, table, rng)
    on = OnDevice(dev, ref)
    at = 0
    rows = [np.full((1, 32), 1e-40), np.full((2, 32), 3e38), np.zeros((1, 32)), rng.normal(size=(17, 32)) * 1e-33,
            rng.normal(size=(3, 32)) * 448, np.full((1, 32), 448.0), np.full((1, 32), -448.0 * 2.0 ** 7),
            np.full((1, 32), np.float32(448.00003))]
    rows[4][0, 3], rows[4][1, 4], rows[4][2, 5] = np.nan, np.inf, -np.inf
    for x in rows:
        k, k64 = as_dtype(x, "f32")
        append(dev, on, None, k, k, [at], [x.shape[0]], 1, "f32")
        ref.append(0, at, k64.reshape(-1, 1, 32), k64.reshape(-1, 1, 32))
        on.same()
        at += x.shape[0]


def test_append_skips_and_flags_what_it_cannot_store(dev):
    rng = np.random.default_rng(5)
    B, page = 9, 16
    pages, table = spread(rng, B, 4)
    table[2, 1] = -1          # a page that is not there
    table[3, 0] = pages
    ref = kvref.Cache(pages, page, 1, 32, table, rng)
    on = OnDevice(dev, ref)
    new = [3, 20, 20, 5, 4, 4, 4, 4, 4]
    past = [0, 0, 0, 0, -1, 61, 0, 2147483647, 0]   # 4, 5, 7: before 0, beyond the table
    st = starts_of(new)
    st[8], st[9] = 64, 60     # 8: an end before its start; 7 grows to its start
    N = 60
    k, k64 = as_dtype(rng.normal(size=(N, 32)), "f32")
    bad = DBuf(dev, np.zeros(B, np.int32))
    cos, sin = kvref.tables(64, 32)
    append(dev, on, None, k, k, past, new, 1, "f32", cos, sin, bad=bad, N=N, max_new=20, starts=st)
    for b in (0, 1, 2, 3, 6):
        r = slice(st[b], st[b + 1])
        pos = np.arange(new[b])
        ref.append(b, 0, kvref.rotate(k64[r].reshape(-1, 1, 32), cos[pos][:, None], sin[pos][:, None]),
                   k64[r].reshape(-1, 1, 32))
    on.same()
    assert bad.get().tolist() == [0, 0, 1, 1, 1, 1, 0, 1, 1]
    # more tokens than announced, positions beyond the rotation tables
    bad = DBuf(dev, np.zeros(B, np.int32))
    ok = [0] * B
    append(dev, on, None, k, k, ok, [3] * B, 1, "f32", cos, sin, bad=bad, N=N, max_new=2, starts=starts_of([3] * B))
    on.same()
    assert bad.get().tolist() == [1] * B
    bad = DBuf(dev, np.zeros(B, np.int32))
    append(dev, on, None, k, k, [2] + [0] * (B - 1), [3] + [0] * (B - 1), 1, "f32", cos, sin, bad=bad, rope_len=4)
    on.same()
    assert bad.get().tolist() == [1] + [0] * (B - 1)


def test_refusals(dev):
    from goneuron_amd._lib import KVCache
    L, _ = _lib()
    rng = np.random.default_rng(6)
    ref = kvref.Cache(4, 16, 2, 32, np.arange(4).reshape(1, 4), rng)
    on = OnDevice(dev, ref)
    x, i = DBuf(dev, np.zeros(4096, np.float32)), DBuf(dev, np.zeros(8, np.int32))
    fields = {n: getattr(on.kv, n) for n, _ in KVCache._fields_}

    def app(q=x.p, k=x.p, v=x.p, qo=x.p, qs=64, ks=64, vs=64, qos=64, cos=x.p, sin=x.p, rl=64, st=i.p, ln=i.p, B=1, N=1, mn=1,
            heads=2, dtype=0, **kv):
        return L.gn_kv_append(dev.h, C.byref(KVCache(**{**fields, **kv})), q, k, v, qo, qs, ks, vs, qos, cos, sin, rl, st, ln, B,
                              N, mn, heads, dtype, None)

    def att(q=x.p, out=x.p, qs=64, os=64, st=i.p, ln=i.p, B=1, N=1, mn=1, ml=64, heads=2, scale=1.0, dtype=0, work=x.p, **kv):
        return L.gn_kv_attention(dev.h, C.byref(KVCache(**{**fields, **kv})), q, out, qs, os, st, ln, B, N, mn, ml, heads,
                                 scale, 1, dtype, work, None)

    assert app() == 0 and att() == 0      # no new token: nothing runs amiss
    odd = C.c_void_p(x.p.value + 2)
    for f in (app, att):
        for kw in (dict(page_size=48), dict(page_size=0), dict(pages=0), dict(kv_heads=0), dict(max_pages=0), dict(heads=3),
                   dict(heads=0), dict(k=None), dict(v=None), dict(k_scale=None), dict(table=None), dict(st=None),
                   dict(ln=None), dict(B=-1), dict(N=-1), dict(mn=-1), dict(dtype=2), dict(q=odd), dict(qs=63),
                   dict(head_dim=0)):
            if f is app and "k" in kw or f is app and "v" in kw:
                continue
            assert f(**kw) < 0, (f.__name__, kw)
        assert f(head_dim=257) == -4
        assert f(B=70000) == -4 and f(mn=1 << 27) == -4
        assert f(B=0) == 0 and f(N=0) == 0 and f(mn=0) == 0
    assert app(cos=None) == -1 and app(q=None) == -1 and app(qo=None) == -1 and app(k=None) == -1 and app(v=None) == -1
    assert app(ks=63) == -1 and app(vs=63) == -1 and app(qos=63) == -1 and app(qos=128) == -1
    assert att(out=None) == -1 and att(os=63) == -1 and att(scale=math.inf) == -1 and att(scale=math.nan) == -1
    assert att(ml=-1) == -1 and att(ml=8192, work=None) == -1
    assert L.gn_kv_append(dev.h, None, x.p, x.p, x.p, x.p, 64, 64, 64, 64, x.p, x.p, 64, i.p, i.p, 1, 1, 1, 2, 0, None) == -1
    assert L.gn_kv_attention(None, C.byref(on.kv), x.p, x.p, 64, 64, i.p, i.p, 1, 1, 1, 64, 2, 1.0, 1, 0, x.p, None) == -1
    assert L.gn_rope_tables(dev.h, None, x.p, 4, 32) == -1 and L.gn_rope_tables(dev.h, x.p, x.p, 0, 32) == -1
    on.same()


# ---------------------------------------------------------------- attention
ATT = [
    # dtype, hd, page, kvh, group, past, new, causal
    ("f32", 32, 16, 8, 1, [127, 0, 1, 63, 64], [1] * 5, 1),
    ("bf16", 128, 64, 2, 4, [0, 200, 63], [1, 1, 1], 1),
    ("f32", 128, 64, 1, 16, [700, 5], [1, 1], 1),
    ("bf16", 64, 128, 1, 17, [300, 129], [1, 1], 1),              # more heads a key than a tile has rows
    ("f32", 80, 32, 4, 3, [0, 17, 90, 3], [70, 0, 33, 1], 1),
    ("bf16", 96, 16, 2, 2, [40, 0], [100, 61], 1),
    ("f32", 7, 16, 1, 1, [0, 30], [19, 2], 1),
    ("bf16", 1, 16, 2, 1, [5], [40], 1),
    ("f32", 192, 64, 1, 2, [33, 0], [3, 70], 1),
    ("bf16", 256, 128, 1, 3, [100, 0], [1, 45], 1),
    ("f32", 256, 16, 1, 1, [20, 0], [1, 17], 0),
    ("bf16", 128, 32, 2, 2, [10, 64, 0], [90, 1, 64], 0),
    ("f32", 48, 64, 3, 1, [0, 0, 0], [1, 2, 3], 0),
    ("bf16", 72, 16, 1, 5, [2], [130], 1),
]


def attention_case(dev, dtype, hd, page, kvh, G, past, new, causal, max_len=None, spoil=None, gap=0):
    rng = np.random.default_rng(hd * 17 + page + sum(past))
    B, heads, N = len(past), kvh * G, sum(new)
    max_pages = max(-(-(a + b) // page) for a, b in zip(past, new)) + 1
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    for b in range(B):
        n = past[b] + new[b]
        x = rng.normal(size=(2, n, kvh, hd))
        ref.append(b, 0, x[0] * 1.5, x[1])
    if spoil:
        spoil(ref)
    on = OnDevice(dev, ref)
    q, q64 = as_dtype(rng.normal(size=(N + 2, heads * hd + gap)), dtype)
    scale = float(np.float32(1 / math.sqrt(hd)))
    L, check = _lib()
    longest = max(a + b for a, b in zip(past, new))
    max_len = max_len or longest
    n = C.c_int64()
    check(None, L.gn_kv_attention_workspace(B, max(new), max_len, heads, kvh, hd, C.byref(n)))
    work = DBuf(dev, np.full(max(1, n.value), np.nan, np.float32))
    mark, _ = as_dtype(np.full((N + 2, heads * hd + gap), 77.0), dtype)
    dq, do, st, ln = DBuf(dev, q), DBuf(dev, mark), DBuf(dev, starts_of(new)), DBuf(dev, np.asarray(past, np.int32))
    bad = DBuf(dev, np.zeros(B, np.int32))
    w = heads * hd + gap
    for _ in range(2):  # the second call finds the first one's workspace
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, w, w, st.p, ln.p, B, N + 2, max(new), max_len, heads,
                                       scale, causal, F32 if dtype == "f32" else BF16, work.p, bad.p))
    on.same()
    got = values(do.get(), dtype)
    assert (got[N:] == 77).all() and (got[:, heads * hd:] == 77).all()
    got, s = got[:N, :heads * hd].reshape(N, heads, hd), starts_of(new)
    worst = 0.0
    for b in range(B):
        if not new[b]:
            continue
        q1 = q64[s[b]:s[b + 1], :heads * hd].reshape(-1, heads, hd)
        want, size, lost = kvref.attend(ref, b, past[b], q1, scale, causal)
        lim = kvref.bound(want, size, lost, past[b] + new[b], dtype)
        o = got[s[b]:s[b + 1]]
        assert np.array_equal(np.isnan(o), np.isnan(want)), (b, np.argwhere(np.isnan(o) != np.isnan(want))[:5])
        fine = ~np.isnan(want)
        over = np.abs(o - want)[fine] / lim[fine]
        worst = max(worst, float(over.max(initial=0)))
    log(f"attention {dtype} hd={hd} page={page} kvh={kvh} G={G} past={past} new={new}: {worst:.3f} of the bound")
    assert worst <= 1
    return bad.get()


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new,causal", ATT)
def test_attention(dev, dtype, hd, page, kvh, G, past, new, causal):
    assert attention_case(dev, dtype, hd, page, kvh, G, past, new, causal).tolist() == [0] * len(past)


@pytest.mark.parametrize("dtype,G,new,past", [("f32", 2, 1, [2999, 511, 512, 0]), ("bf16", 1, 1, [4100]), ("bf16", 4, 9, [1500, 700]),
                                              ("f32", 1, 3, [1027]), ("bf16", 3, 40, [1300, 0])])
def test_attention_split_along_the_keys(dev, dtype, G, new, past):
    """Long histories of few sequences, also far below the announced length."""
    attention_case(dev, dtype, 64, 32, 1, G, past, [new] * len(past), 1)
    attention_case(dev, dtype, 64, 32, 1, G, past, [new] * len(past), 0, max_len=20000)


def test_attention_rows_with_a_stride(dev):
    attention_case(dev, "f32", 40, 16, 2, 2, [9, 50], [5, 1], 1, gap=3)
    attention_case(dev, "bf16", 128, 64, 2, 2, [9, 50], [5, 70], 1, gap=1)


@pytest.mark.parametrize("dtype,new", [("f32", 1), ("bf16", 1), ("f32", 37), ("bf16", 90)])
def test_attention_leaves_out_pages_that_are_not_there(dev, dtype, new):
    def spoil(ref):
        ref.table[0, 1], ref.table[1, 0], ref.table[2, :] = -5, ref.pages + 3, -1
    bad = attention_case(dev, dtype, 64, 16, 2, 2, [40, 30, 20, 9], [new] * 4, 1, spoil=spoil)
    assert bad.tolist() == [1, 1, 1, 0]


@pytest.mark.parametrize("dtype,new", [("f32", 2), ("bf16", 40), ("f32", 70)])
def test_attention_nan_stays_with_the_rows_that_see_it(dev, dtype, new):
    past = [20, 3]

    def spoil(ref):
        for b, p in ((0, 20 + new - 1), (1, 3 + new // 2)):
            page, t = ref.table[b, p // 16], p % 16
            ref.v[page, 0, 5, t] = 0x7f
            ref.v[page, 1, 2, t] = 0xff
        page = ref.table[0, 10 // 16]
        ref.k[page, 1, 10 % 16, 3] = 0x7f    # a key of NaN: every row of that head that sees it
    attention_case(dev, dtype, 32, 16, 2, 2, past, [new] * 2, 1, spoil=spoil)


def test_attention_flags_sequences_out_of_bounds(dev):
    rng = np.random.default_rng(8)
    pages, table = spread(rng, 4, 4)
    ref = kvref.Cache(pages, 16, 1, 32, table, rng)
    ref.append(0, 0, rng.normal(size=(9, 1, 32)), rng.normal(size=(9, 1, 32)))
    on = OnDevice(dev, ref)
    L, check = _lib()
    q, o = DBuf(dev, rng.normal(size=(4, 32)).astype(np.float32)), DBuf(dev, np.full((4, 32), 5, np.float32))
    st, ln, bad = DBuf(dev, np.arange(5, dtype=np.int32)), DBuf(dev, np.array([8, 64, 40, -3], np.int32)), DBuf(dev, np.zeros(4, np.int32))
    check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), q.p, o.p, 32, 32, st.p, ln.p, 4, 4, 1, 40, 1, 0.2, 1, F32, None, bad.p))
    assert bad.get().tolist() == [0, 1, 1, 1]
    assert (o.get()[1:] == 5).all() and (o.get()[0] != 5).all()


# ---------------------------------------------------------------- the layer
@pytest.mark.parametrize("D,heads,page,rope,steps", [(64, 2, 16, 1, [[7, 20], [1, 1], [3, 0], [1, 1]]),
                                                     (256, 8, 64, 0, [[70, 1], [1, 1]]),
                                                     (160, 2, 32, 1, [[1, 33], [1, 1]])])
def test_mha_cached_layer(dev, D, heads, page, rope, steps):
    """Steps of the MultiHeadAttention layer over a cache.  A projected key within
    float32 rounding of an E4M3 border may take either side, so the cache is held
    to half an E4M3 step of the float64 projections (2^-4 relative, 2^-10 of the
    scale near 0) and the output to the formulas on the cache as it is."""
    L, check = _lib()
    rng = np.random.default_rng(D)
    hd, B = D // heads, 2
    nd = D * D + D
    params = (rng.normal(size=4 * nd) / math.sqrt(D)).astype(np.float32)
    W = [(params[i * nd:i * nd + D * D].reshape(D, D).astype(np.float64), params[i * nd + D * D:(i + 1) * nd].astype(np.float64))
         for i in range(4)]
    pages, table = spread(rng, B, 4)
    ref = kvref.Cache(pages, page, heads, hd, table, rng)
    on = OnDevice(dev, ref)
    dcos, dsin = DBuf(dev, np.zeros((4 * page, hd // 2), np.float32)), DBuf(dev, np.zeros((4 * page, hd // 2), np.float32))
    check(dev.h, L.gn_rope_tables(dev.h, dcos.p, dsin.p, 4 * page, hd))
    cos, sin = kvref.tables(4 * page, hd)
    assert np.abs(dcos.get() - cos).max() <= 2.0 ** -23 and np.abs(dsin.get() - sin).max() <= 2.0 ** -23
    cos, sin = dcos.get(), dsin.get()
    dp, past = DBuf(dev, params), [0, 0]
    for new in steps:
        N = sum(new)
        x = rng.normal(size=(N, D)).astype(np.float32)
        n = C.c_int64()
        ml = max(a + b for a, b in zip(past, new))
        check(None, L.gn_mha_cached_workspace(B, N, max(new), ml, D, heads, C.byref(n)))
        dx, do, work = DBuf(dev, x), DBuf(dev, x * 0), DBuf(dev, np.full(n.value, np.nan, np.float32))
        st, ln, bad = DBuf(dev, starts_of(new)), DBuf(dev, np.asarray(past, np.int32)), DBuf(dev, np.zeros(B, np.int32))
        check(dev.h, L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, do.p, dcos.p if rope else None,
                                             dsin.p if rope else None, 4 * page if rope else 0, st.p, ln.p, B, N, max(new), ml,
                                             D, work.p, bad.p))
        assert not bad.get().any()
        ref.k, ref.v, ref.ks, ref.vs = on.k.get(), on.v.get(), on.ks.get(), on.vs.get()
        q, k, v = (x.astype(np.float64) @ W[i][0].T + W[i][1] for i in range(3))
        # D products and sums in float32 for a projected number; a rotation adds two such errors
        dq, dk, dv = (1.5 * 2.0 ** -24 * (D + 4) * (np.abs(x).astype(np.float64) @ np.abs(W[i][0]).T + np.abs(W[i][1]))
                      for i in range(3))
        if rope:
            dq, dk = (a + np.roll(a.reshape(-1, heads, hd), hd // 2, 2).reshape(a.shape) for a in (dq, dk))
        got, s = do.get(), starts_of(new)
        for b in range(B):
            r, pos = slice(s[b], s[b + 1]), np.arange(past[b], past[b] + new[b])
            if not new[b]:
                continue
            q1, k1, v1 = (a[r].reshape(-1, heads, hd) for a in (q, k, v))
            if rope:
                q1, k1 = (kvref.rotate(a, cos[pos][:, None], sin[pos][:, None]) for a in (q1, k1))
            kc, vc, _ = ref.read(b, past[b] + new[b])
            for a, c, sc, off in ((k1, kc, ref.ks, dk), (v1, vc, ref.vs, dv)):
                slack = 2 * off[r].reshape(a.shape)
                step = sc[table[b, pos // page]].astype(np.float64)[..., None] * 2.0 ** -10
                assert (np.abs(c[pos] - a) <= np.maximum(np.abs(a) * 2.0 ** -4, step) * (1 + 2.0 ** -10) + slack).all()
            o, size, lost = kvref.attend(ref, b, past[b], q1, 1 / math.sqrt(hd), 1)
            off = np.einsum("thd,lhd->thl", dq[r].reshape(-1, heads, hd), np.abs(kc)).max(2) / math.sqrt(hd)
            lim = kvref.bound(o, size, lost + off, past[b] + new[b], "f32")
            want = o.reshape(-1, D) @ W[3][0].T + W[3][1]
            lim = lim.reshape(-1, D) @ np.abs(W[3][0]).T + 2.0 ** -24 * (D + 4) * (np.abs(o.reshape(-1, D)) @ np.abs(W[3][0]).T + 1)
            assert (np.abs(got[r] - want) <= lim).all(), (b, float((np.abs(got[r] - want) / lim).max()))
        past = [a + b for a, b in zip(past, new)]


def test_mha_cached_is_the_layer(dev):
    """All tokens at once over an empty cache: gn_mha_forward's causal layer but for
    the 8-bit rounding of keys and values (2^-4 each at most: a few percent of the output)."""
    L, check = _lib()
    rng = np.random.default_rng(11)
    B, T, D, heads = 2, 48, 64, 4
    params = (rng.normal(size=4 * (D * D + D)) / math.sqrt(D)).astype(np.float32)
    x = rng.normal(size=(B * T, D)).astype(np.float32)
    dx, dp, a, b = DBuf(dev, x), DBuf(dev, params), DBuf(dev, x * 0), DBuf(dev, x * 0)
    n = C.c_int64()
    check(None, L.gn_mha_workspace(B, T, D, heads, 1, C.byref(n)))
    w = DBuf(dev, np.zeros(n.value, np.float32))
    check(dev.h, L.gn_mha_forward(dev.h, dx.p, dp.p, a.p, w.p, B, T, D, heads, 1, 1))
    pages, table = spread(rng, B, 3)
    ref = kvref.Cache(pages, 16, heads, D // heads, table, rng)
    on = OnDevice(dev, ref)
    dcos, dsin = DBuf(dev, np.zeros((T, 8), np.float32)), DBuf(dev, np.zeros((T, 8), np.float32))
    check(dev.h, L.gn_rope_tables(dev.h, dcos.p, dsin.p, T, D // heads))
    check(None, L.gn_mha_cached_workspace(B, B * T, T, T, D, heads, C.byref(n)))
    w = DBuf(dev, np.zeros(n.value, np.float32))
    st, ln = DBuf(dev, np.array([0, T, 2 * T], np.int32)), DBuf(dev, np.zeros(2, np.int32))
    check(dev.h, L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, b.p, dcos.p, dsin.p, T, st.p, ln.p, B, B * T, T, T, D,
                                         w.p, None))
    d = np.linalg.norm(a.get() - b.get()) / np.linalg.norm(a.get())
    log(f"cached against whole layer: {d:.4f}")
    assert d <= 2.0 ** -4
    # sizes that do not fit the cache
    assert L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, b.p, dcos.p, dsin.p, T, st.p, ln.p, B, B * T, T, T, D + 4,
                                   w.p, None) == -5
    assert L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, b.p, dcos.p, dsin.p, T, st.p, ln.p, B, B * T, T, T, D,
                                   None, None) == -1


def test_generating_steps_together(dev):
    """Prompts and then token after token: queries, keys and values appended, attended,
    projected to logits by gn_gemm and sampled, each step's tokens the next one's input."""
    L, check = _lib()
    rng = np.random.default_rng(12)
    V, D, heads, kvh, page, B = 300, 64, 4, 2, 16, 3
    hd, KW = D // heads, kvh * (D // heads)
    E = rng.normal(size=(V, D)).astype(np.float32)
    Wqkv = (rng.normal(size=(D + 2 * KW, D)) / math.sqrt(D)).astype(np.float32)
    pages, table = spread(rng, B, 4)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    on = OnDevice(dev, ref)
    cos, sin = kvref.tables(64, hd)
    dcos, dsin, dE, dW = DBuf(dev, cos), DBuf(dev, sin), DBuf(dev, E), DBuf(dev, Wqkv)
    tokens = [list(rng.integers(0, V, n)) for n in (5, 17, 1)]
    past = [0, 0, 0]
    for step in range(20):
        new = [len(tokens[b]) - past[b] for b in range(B)]
        N = sum(new)
        x = np.concatenate([E[tokens[b][past[b]:]] for b in range(B)])
        dx, dqkv, dq, do = DBuf(dev, x), DBuf(dev, np.zeros((N, D + 2 * KW), np.float32)), DBuf(dev, x * 0), DBuf(dev, x * 0)
        check(dev.h, L.gn_gemm(dev.h, 0, 1, N, D + 2 * KW, D, 1.0, dx.p, D, dW.p, D, dqkv.p, D + 2 * KW))
        w, base = D + 2 * KW, dqkv.p.value
        st, ln, bad = DBuf(dev, starts_of(new)), DBuf(dev, np.asarray(past, np.int32)), DBuf(dev, np.zeros(B, np.int32))
        check(dev.h, L.gn_kv_append(dev.h, C.byref(on.kv), C.c_void_p(base), C.c_void_p(base + 4 * D), C.c_void_p(base + 4 * (D + KW)),
                                    dq.p, w, w, w, D, dcos.p, dsin.p, 64, st.p, ln.p, B, N, max(new), heads, F32, bad.p))
        qkv = dqkv.get().astype(np.float64)
        s, last, want_o, lim = starts_of(new), [], np.zeros((N, D)), np.zeros((N, D))
        for b in range(B):
            r, pos = slice(s[b], s[b + 1]), np.arange(past[b], past[b] + new[b])
            c, sn = cos[pos][:, None], sin[pos][:, None]
            ref.append(b, past[b], kvref.rotate(qkv[r, D:D + KW].reshape(-1, kvh, hd), c, sn), qkv[r, D + KW:].reshape(-1, kvh, hd))
            q = kvref.rotate(qkv[r, :D].reshape(-1, heads, hd), c, sn)
            w1, size, lost = kvref.attend(ref, b, past[b], q, 0.25, 1)
            want_o[r], lim[r] = w1.reshape(-1, D), kvref.bound(w1, size, lost, len(tokens[b]), "f32").reshape(-1, D)
            last.append(s[b + 1] - 1)
        on.same()
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, D, D, st.p, ln.p, B, N, max(new), 64, heads, 0.25, 1, F32,
                                       None, bad.p))
        o = do.get()
        assert (np.abs(o - want_o) <= lim).all() and not bad.get().any()
        dl, dh = DBuf(dev, np.zeros((B, V), np.float32)), DBuf(dev, o[last])
        check(dev.h, L.gn_gemm(dev.h, 0, 1, B, V, D, 1.0, dh.p, D, dE.p, D, dl.p, V))
        u, T = rng.random(B).astype(np.float32), np.array([0.7, 1.0, 0.0], np.float32)
        k, p = np.array([40, 0, 5], np.int32), np.array([0.9, 0.95, 1.0], np.float32)
        n = C.c_int64()
        check(None, L.gn_sample_workspace(B, V, C.byref(n)))
        bufs = [DBuf(dev, a) for a in (T, k, p, u, np.zeros(B, np.int32), np.zeros(n.value, np.float32))]
        check(dev.h, L.gn_sample(dev.h, dl.p, V, F32, bufs[0].p, bufs[1].p, bufs[2].p, None, bufs[3].p, bufs[4].p, B, V, bufs[5].p))
        z, ids = dl.get().astype(np.float64), bufs[4].get()
        past = [len(t) for t in tokens]
        for b in range(B):
            assert ids[b] == kvref.sample(z[b], u[b], T[b], k[b], p[b])
            tokens[b].append(int(ids[b]))


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_attention_with_loose_bounds(dev, new):
    """Lengths' bounds far beyond the sequences, up to the largest number there is."""
    for max_len in (5000, 2 ** 30, 2 ** 31 - 1):
        attention_case(dev, "bf16", 64, 16, 2, 2, [77, 0], new, 1, max_len=max_len)


def test_more_rows_than_32_bits_count(dev):
    L, _ = _lib()
    n = C.c_int64()
    assert L.gn_kv_attention_workspace(1, 1 << 20, 64, 4096, 1, 32, C.byref(n)) == -1
    assert L.gn_mha_cached_workspace(64, 1, 1 << 20, 64, 64, 64, C.byref(n)) == -1
    ref = kvref.Cache(4, 16, 2, 32, np.arange(4).reshape(1, 4), np.random.default_rng(1))
    on = OnDevice(dev, ref)
    x, i = DBuf(dev, np.zeros(4096, np.float32)), DBuf(dev, np.zeros(8, np.int32))
    w = 4096 * 32
    assert L.gn_kv_attention(dev.h, C.byref(on.kv), x.p, x.p, w, w, i.p, i.p, 1, 1, 1 << 20, 64, 4096, 1.0, 1, 0, x.p, None) == -4
    assert L.gn_kv_append(dev.h, C.byref(on.kv), x.p, x.p, x.p, x.p, w, w, w, w, None, None, 0, i.p, i.p, 1, 1, 1 << 20, 4096, 0,
                          None) == -4


def test_two_contexts_at_once(gn, dev):
    """Two streams append to caches of their own, attend over them and draw, their work
    queued in turn without a wait between."""
    other = gn.HIPDevice(0)
    try:
        on_two_streams(dev, other)   # its buffers go before their context
    finally:
        other.close()


def on_two_streams(dev, other):
    L, check = _lib()
    rng = np.random.default_rng(9)
    hd, kvh, H, P, T = 64, 2, 8, 32, 200
    V = 20000
    runs = []
    for d in (dev, other):
        ref = kvref.Cache(10, P, kvh, hd, rng.permutation(10)[:8].reshape(1, 8).astype(np.int32), rng)
        on = OnDevice(d, ref)
        k, v, q = (rng.normal(size=(T, n * hd)).astype(np.float32) for n in (kvh, kvh, H))
        n = C.c_int64()
        check(None, L.gn_kv_attention_workspace(1, T, 256, H, kvh, hd, C.byref(n)))
        work = DBuf(d, np.full(max(1, n.value), np.nan, np.float32))
        check(None, L.gn_sample_workspace(1, V, C.byref(n)))
        draw = DBuf(d, np.full(n.value, np.nan, np.float32))
        z = rng.normal(size=(1, V)).astype(np.float32) * 3
        runs.append(dict(d=d, ref=ref, on=on, host=(k, v, q), k=DBuf(d, k), v=DBuf(d, v), q=DBuf(d, q),
                         out=DBuf(d, np.zeros((T, H * hd), np.float32)), st=DBuf(d, np.array([0, T], np.int32)),
                         ln=DBuf(d, np.zeros(1, np.int32)), work=work, draw=draw, z=z, dz=DBuf(d, z),
                         u=DBuf(d, np.array([0.37], np.float32)), p=DBuf(d, np.array([0.9], np.float32)),
                         ids=DBuf(d, np.full(1, -7, np.int32))))
    for r in runs:
        check(r["d"].h, L.gn_kv_append(r["d"].h, C.byref(r["on"].kv), None, r["k"].p, r["v"].p, None, 0, kvh * hd, kvh * hd, 0,
                                       None, None, 0, r["st"].p, r["ln"].p, 1, T, T, H, F32, None))
    for _ in range(3):
        for r in runs:
            check(r["d"].h, L.gn_kv_attention(r["d"].h, C.byref(r["on"].kv), r["q"].p, r["out"].p, H * hd, H * hd, r["st"].p,
                                              r["ln"].p, 1, T, T, 256, H, 0.125, 1, F32, r["work"].p, None))
            check(r["d"].h, L.gn_sample(r["d"].h, r["dz"].p, V, F32, None, None, r["p"].p, None, r["u"].p, r["ids"].p, 1, V,
                                        r["draw"].p))
    for r in runs:
        k, v, q = r["host"]
        r["ref"].append(0, 0, k.reshape(T, kvh, hd), v.reshape(T, kvh, hd))
        want, size, lost = kvref.attend(r["ref"], 0, 0, q.reshape(T, H, hd).astype(np.float64), 0.125, 1)
        got = r["out"].get().reshape(T, H, hd).astype(np.float64)
        assert (np.abs(got - want) <= kvref.bound(want, size, lost, T, "f32")).all()
        assert int(r["ids"].get()[0]) == kvref.sample(r["z"][0].astype(np.float64), np.float32(0.37), top_p=np.float32(0.9))
