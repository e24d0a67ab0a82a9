"""GPU tests of attention over the paged cache with a sliding window and first tokens
(gn_kv_attention_window) and of trees of drafted tokens (gn_kv_attention_tree), within
derived bounds against float64 restatements (viewref)."""
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


def floats(B, max_new, max_len, heads, kvh, hd):
    L, check = _lib()
    n = C.c_int64()
    check(None, L.gn_kv_attention_workspace(B, max_new, max_len, heads, kvh, hd, C.byref(n)))
    return n.value


def case(dev, dtype, hd, page, kvh, G, past, new, sinks=0, window=0, masks=None, max_len=None, spoil=None, gap=0, seed=0,
         max_new=None, scale=None, gone=False):
    """One call, twice; masks: a tree each (else a window).  gone: pages that no query sees
    have entries of any kind."""
    rng = np.random.default_rng(hd * 19 + page + sum(past) + seed)
    B, heads, N = len(past), kvh * G, sum(new)
    max_pages = max(-(-(a + b) // page) for a, b in zip(past, new)) + 1
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    for b in range(B):
        n = past[b] + new[b]
        x = rng.normal(size=(2, n, kvh, hd))
        ref.append(b, 0, x[0] * 1.5, x[1])
    sight = [viewref.tree_sight(past[b], masks[b]) if masks is not None else viewref.window_sight(past[b], new[b], sinks, window)
             for b in range(B)]
    if spoil:
        spoil(ref)
    if gone:
        for b in range(B):
            for j in range(max_pages):
                if not sight[b][:, j * page:(j + 1) * page].any():
                    ref.table[b, j] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31, 0])
    on = OnDevice(dev, ref)
    q, q64 = as_dtype(rng.normal(size=(N + 2, heads * hd + gap)), dtype)
    scale = float(np.float32(1 / math.sqrt(hd))) if scale is None else scale
    L, check = _lib()
    max_len = max_len or max(a + b for a, b in zip(past, new))
    max_new = max_new or max(new)
    work = DBuf(dev, np.full(max(1, floats(B, max_new, max_len, heads, kvh, hd)), np.nan, np.float32))
    mark, _ = as_dtype(np.full((N + 2, heads * hd + gap), 77.0), dtype)
    dq, do, st, ln = DBuf(dev, q), DBuf(dev, mark), DBuf(dev, starts_of(new)), DBuf(dev, np.asarray(past, np.int32))
    bad = DBuf(dev, np.zeros(B, np.int32))
    w = heads * hd + gap
    code = F32 if dtype == "f32" else BF16
    if masks is not None:
        stride = -(-max_new // 32) + 1
        dm = DBuf(dev, viewref.words(masks, stride, rng).view(np.int32))
    for _ in range(2):  # the second call finds the first one's workspace
        if masks is not None:
            check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, do.p, w, w, dm.p, stride, st.p, ln.p, B, N + 2, max_new,
                                                max_len, heads, scale, code, work.p, bad.p))
        else:
            check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, do.p, w, w, st.p, ln.p, B, N + 2, max_new, max_len,
                                                  heads, scale, sinks, window, code, work.p, bad.p))
    on.same()
    got = values(do.get(), dtype)
    assert (got[N:] == 77).all() and (got[:, heads * hd:] == 77).all()
    got, s = got[:N, :heads * hd].reshape(N, heads, hd), starts_of(new)
    worst = 0.0
    for b in range(B):
        if not new[b]:
            continue
        q1 = q64[s[b]:s[b + 1], :heads * hd].reshape(-1, heads, hd)
        want, size, lost = viewref.attend(ref, b, past[b], q1, scale, sight[b])
        lim = kvref.bound(want, size, lost, past[b] + new[b], dtype)
        o = got[s[b]:s[b + 1]]
        apart = np.argwhere(np.isnan(o) != np.isnan(want))
        assert not len(apart), (b, apart[:5])
        fine = ~np.isnan(want)
        worst = max(worst, float((np.abs(o - want)[fine] / lim[fine]).max(initial=0)))
    log(f"{'tree' if masks is not None else 'window'} {dtype} hd={hd} page={page} kvh={kvh} G={G} past={past} new={new} "
        f"sinks={sinks} window={window}: {worst:.3f} of the bound")
    assert worst <= 1
    return bad.get()


# ---------------------------------------------------------------- windows
WINDOWS = [
    # dtype, hd, page, kvh, group, past, new, sinks, window
    ("f32", 32, 16, 8, 1, [127, 0, 1, 63, 64, 300], [1] * 6, 4, 64),
    ("bf16", 128, 64, 2, 4, [0, 900, 63, 511], [1, 1, 1, 1], 4, 200),
    ("f32", 128, 64, 1, 16, [1700, 5], [1, 1], 100, 1000),
    ("bf16", 64, 128, 1, 17, [300, 129], [1, 1], 1, 17),
    ("f32", 80, 32, 4, 3, [0, 17, 400, 3], [70, 0, 33, 1], 5, 40),
    ("bf16", 96, 16, 2, 2, [40, 0], [300, 61], 0, 100),
    ("f32", 7, 16, 1, 1, [200, 30], [19, 2], 3, 9),
    ("bf16", 1, 16, 2, 1, [500], [40], 64, 1),
    ("f32", 192, 64, 1, 2, [333, 0], [3, 70], 65, 30),
    ("bf16", 256, 128, 1, 3, [700, 0], [1, 145], 10, 128),
    ("f32", 256, 16, 1, 1, [320, 0], [1, 117], 0, 33),
    ("bf16", 128, 32, 2, 4, [1000, 64, 0], [190, 1, 64], 4, 63),
    ("f32", 48, 64, 3, 1, [0, 0, 0], [1, 2, 3], 1, 1),
    ("bf16", 72, 16, 1, 5, [2], [430], 7, 128),
    ("bf16", 192, 64, 2, 2, [600], [5], 4, 100),
]


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new,sinks,window", WINDOWS)
def test_window(dev, dtype, hd, page, kvh, G, past, new, sinks, window):
    bad = case(dev, dtype, hd, page, kvh, G, past, new, sinks, window, gone=True)
    assert bad.tolist() == [0] * len(past)


@pytest.mark.parametrize("dtype,new", [("f32", [1, 1]), ("bf16", [1, 1]), ("f32", [50, 3]), ("bf16", [130, 66])])
@pytest.mark.parametrize("sinks,window", [(0, 0), (0, 1), (1, 0), (2 ** 31 - 1, 0), (0, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1),
                                          (64, 64), (63, 65), (128, 1)])
def test_window_of_every_kind(dev, dtype, new, sinks, window):
    case(dev, dtype, 64, 16, 2, 2, [260, 70], new, sinks, window, gone=True, seed=new[0])


@pytest.mark.parametrize("dtype,G,new,past,window", [("f32", 2, 1, [9000, 511, 4512, 0], 6000), ("bf16", 1, 1, [7100], 5000),
                                                     ("bf16", 4, 9, [3500, 700], 1500), ("f32", 1, 20, [5000, 30], 3000)])
def test_window_split_along_the_keys(dev, dtype, G, new, past, window):
    case(dev, dtype, 64, 64, 2, G, past, [new] * len(past), 70, window)


def test_window_that_holds_all_is_attention_without(dev):
    """gn_kv_attention's answers.  Each call is within the bound of the exact value, so they are
    within twice it of each other; they may walk the keys in different orders."""
    L, check = _lib()
    rng = np.random.default_rng(3)
    for dtype, new, past in (("f32", 1, 700), ("bf16", 90, 200), ("f32", 40, 0), ("bf16", 1, 5000)):
        hd, kvh, H, P = 64, 2, 4, 32
        total = past + new
        pages, table = spread(rng, 1, -(-total // P))
        ref = kvref.Cache(pages, P, kvh, hd, table, rng)
        x = rng.normal(size=(2, total, kvh, hd))
        ref.append(0, 0, x[0], x[1])
        on = OnDevice(dev, ref)
        q, _ = as_dtype(rng.normal(size=(new, H * hd)), dtype)
        work = DBuf(dev, np.zeros(max(1, floats(1, new, total, H, kvh, hd)), np.float32))
        dq, st, ln = DBuf(dev, q), DBuf(dev, starts_of([new])), DBuf(dev, np.array([past], np.int32))
        a, b = DBuf(dev, q * 0), DBuf(dev, q * 0)
        code = F32 if dtype == "f32" else BF16
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, a.p, H * hd, H * hd, st.p, ln.p, 1, new, new, total, H, 0.125, 1,
                                       code, work.p, None))
        check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, b.p, H * hd, H * hd, st.p, ln.p, 1, new, new, total, H,
                                              0.125, 3, total, code, work.p, None))
        va, vb = (values(y.get(), dtype).reshape(new, H, hd) for y in (a, b))
        want, size, lost = kvref.attend(ref, 0, past, values(q, dtype).reshape(new, H, hd), 0.125, 1)
        lim = kvref.bound(want, size, lost, total, dtype)
        assert (np.abs(vb - want) <= lim).all() and (np.abs(va - vb) <= 2 * lim).all() and np.abs(va).max() > 0


# ---------------------------------------------------------------- trees
def tree(rng, n):
    p = [-1] * n
    for i in range(1, n):
        p[i] = i - 1 if rng.random() < 0.6 else int(rng.integers(-1, i))
    return viewref.ancestors(p)


TREES = [
    # dtype, hd, page, kvh, group, past, new
    ("f32", 32, 16, 8, 1, [120, 0, 1, 63, 64], [16] * 5),
    ("bf16", 128, 64, 2, 4, [0, 200, 63], [64, 1, 33]),
    ("f32", 128, 64, 1, 16, [700, 5], [1, 3]),
    ("bf16", 64, 128, 1, 17, [300, 129], [4, 9]),
    ("f32", 80, 32, 4, 3, [0, 17, 90, 3], [70, 0, 33, 1]),
    ("bf16", 96, 16, 2, 2, [40, 0], [100, 61]),
    ("f32", 7, 16, 1, 1, [0, 30], [19, 2]),
    ("bf16", 1, 16, 2, 1, [5], [40]),
    ("f32", 192, 64, 1, 2, [33, 0], [3, 70]),
    ("bf16", 256, 128, 1, 3, [100, 0], [1, 45]),
    ("f32", 256, 16, 1, 1, [20, 0], [5, 17]),
    ("bf16", 128, 32, 2, 2, [10, 64, 0], [190, 1, 64]),
    ("f32", 48, 64, 3, 1, [0, 0, 0], [1, 2, 3]),
    ("bf16", 72, 16, 1, 5, [2], [130]),
    ("bf16", 192, 64, 1, 2, [70], [8]),
]


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new", TREES)
def test_tree(dev, dtype, hd, page, kvh, G, past, new):
    rng = np.random.default_rng(hd + sum(new))
    bad = case(dev, dtype, hd, page, kvh, G, past, new, masks=[tree(rng, n) for n in new])
    assert bad.tolist() == [0] * len(past)


@pytest.mark.parametrize("dtype,G,past,new", [("f32", 1, [0, 40, 7], [16, 5, 1]), ("bf16", 4, [0, 40, 7], [4, 2, 1]),
                                              ("f32", 2, [0, 70, 63], [90, 33, 64]), ("bf16", 2, [0, 70, 1], [200, 33, 65])])
def test_tree_masks_of_any_kind(dev, dtype, G, past, new):
    """Rows that see nothing (no cached token, no bit), themselves alone, all, or others at random."""
    rng = np.random.default_rng(len(past) + new[0])
    masks = [rng.random((n, n)) < 0.4 for n in new]
    for m in masks:
        m[0] = False
        m[-1] = True
        m[len(m) // 2] = False
    case(dev, dtype, 64, 32, 2, G, past, new, masks=masks, max_new=max(new) + 3)


@pytest.mark.parametrize("dtype,G,new,past", [("f32", 2, 7, [2999, 511, 512, 0]), ("bf16", 1, 12, [4100]), ("bf16", 4, 60, [1500, 700]),
                                              ("f32", 1, 37, [5000, 30])])
def test_tree_split_along_the_keys(dev, dtype, G, new, past):
    rng = np.random.default_rng(new)
    case(dev, dtype, 64, 64, 2, G, past, [new] * len(past), masks=[tree(rng, new) for _ in past])


def test_a_chain_is_causal_attention(dev):
    L, check = _lib()
    rng = np.random.default_rng(5)
    for dtype, new, past in (("f32", 8, 700), ("bf16", 90, 200), ("f32", 40, 0)):
        hd, kvh, H, P, total = 64, 2, 4, 32, past + new
        pages, table = spread(rng, 1, -(-total // P))
        ref = kvref.Cache(pages, P, kvh, hd, table, rng)
        x = rng.normal(size=(2, total, kvh, hd))
        ref.append(0, 0, x[0], x[1])
        on = OnDevice(dev, ref)
        q, _ = as_dtype(rng.normal(size=(new, H * hd)), dtype)
        work = DBuf(dev, np.zeros(max(1, floats(1, new, total, H, kvh, hd)), np.float32))
        dq, st, ln = DBuf(dev, q), DBuf(dev, starts_of([new])), DBuf(dev, np.array([past], np.int32))
        a, b = DBuf(dev, q * 0), DBuf(dev, q * 0)
        m = DBuf(dev, viewref.words([viewref.ancestors(list(range(-1, new - 1)))], 3).view(np.int32))
        code = F32 if dtype == "f32" else BF16
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, a.p, H * hd, H * hd, st.p, ln.p, 1, new, new, total, H, 0.125, 1,
                                       code, work.p, None))
        check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, b.p, H * hd, H * hd, m.p, 3, st.p, ln.p, 1, new, new, total,
                                            H, 0.125, code, work.p, None))
        va, vb = (values(y.get(), dtype).reshape(new, H, hd) for y in (a, b))
        # each is within the bound of the exact value, so within twice it of the other: the
        # two walk the keys in different orders and round elsewhere
        want, size, lost = kvref.attend(ref, 0, past, values(q, dtype).reshape(new, H, hd), 0.125, 1)
        lim = kvref.bound(want, size, lost, total, dtype)
        assert (np.abs(vb - want) <= lim).all() and (np.abs(va - vb) <= 2 * lim).all()


# ---------------------------------------------------------------- both
@pytest.mark.parametrize("dtype,new", [("f32", 1), ("bf16", 1), ("f32", 37), ("bf16", 90)])
@pytest.mark.parametrize("view", ["window", "tree"])
def test_pages_that_are_not_there(dev, view, dtype, new):
    rng = np.random.default_rng(new)

    def spoil(ref):
        ref.table[0, 1] = -1
        ref.table[1, 1] = ref.pages
        ref.table[2, :] = -7

    kw = dict(masks=[tree(rng, new) for _ in range(4)]) if view == "tree" else dict(sinks=20, window=2000)
    bad = case(dev, dtype, 64, 16, 2, 2, [100, 30, 50, 40], [new] * 4, spoil=spoil, **kw)
    assert bad.tolist() == [1, 1, 1, 0]


@pytest.mark.parametrize("dtype,new", [("f32", 2), ("bf16", 40), ("f32", 70), ("bf16", 1), ("f32", 30)])
@pytest.mark.parametrize("view", ["window", "tree"])
@pytest.mark.parametrize("hd", [64, 32, 192])
def test_nan_stays_with_the_rows_that_see_it(dev, view, dtype, new, hd):
    rng = np.random.default_rng(new + hd)
    past = [100, 300]

    def spoil(ref):
        # keys and values of cached and of new tokens, in and out of windows
        for b, at in ((0, (3, 50, 101)), (1, (7, 140, 290, 300))):
            for p in at:
                if p >= past[b] + new:
                    continue
                page, t = ref.table[b, p // 16], p % 16
                ref.v[page, 0, (p * 7) % hd, t] = 0x7f
                ref.v[page, 1, 3, t] = 0xff
                if p % 2:
                    ref.k[page, 1, t, 5] = 0x7f

    kw = dict(masks=[tree(rng, new) for _ in past]) if view == "tree" else dict(sinks=5, window=30)
    case(dev, dtype, hd, 16, 2, 2, past, [new, new], spoil=spoil, **kw)


@pytest.mark.parametrize("view", ["window", "tree"])
def test_rows_with_a_stride_and_loose_bounds(dev, view):
    rng = np.random.default_rng(8)
    for max_len in (None, 5000, 2 ** 30, 2 ** 31 - 1):
        for dtype, new in (("bf16", [1, 1]), ("f32", [40, 3])):
            kw = dict(masks=[tree(rng, n) for n in new]) if view == "tree" else dict(sinks=5, window=30)
            case(dev, dtype, 64, 16, 2, 2, [77, 0], new, max_len=max_len, gap=5, **kw)


@pytest.mark.parametrize("view", ["window", "tree"])
def test_score_scales(dev, view):
    rng = np.random.default_rng(8)
    for scale in (0.0, -0.3, 1e-30, 3.0):
        kw = dict(masks=[tree(rng, n) for n in (1, 33)]) if view == "tree" else dict(sinks=2, window=20)
        case(dev, "f32", 64, 16, 2, 2, [77, 3], [1, 33], scale=float(np.float32(scale)), **kw)


def test_sequences_out_of_bounds(dev):
    L, check = _lib()
    rng = np.random.default_rng(7)
    B, hd, P = 6, 32, 16
    pages, table = spread(rng, B, 4)
    ref = kvref.Cache(pages, P, 1, hd, table, rng)
    for b in range(B):
        x = rng.normal(size=(2, 40, 1, hd))
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    # 1: before 0, 2: beyond max_len, 3: more than max_new, 4: the largest number, 5: rows that overlap none
    past = np.array([30, -1, 39, 10, 2 ** 31 - 1, 20], np.int32)
    st = DBuf(dev, np.array([0, 2, 4, 6, 11, 13, 12], np.int32))
    ln = DBuf(dev, past)
    q, q64 = as_dtype(rng.normal(size=(14, hd)), "f32")
    mask = DBuf(dev, np.full((14, 1), 3, np.int32))
    for view in ("window", "tree"):
        do, bad, dq = DBuf(dev, np.full((14, hd), 77, np.float32)), DBuf(dev, np.zeros(B, np.int32)), DBuf(dev, q)
        if view == "window":
            check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, do.p, hd, hd, st.p, ln.p, B, 14, 4, 40, 1, 0.2, 2, 9, F32,
                                                  None, bad.p))
        else:
            check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, do.p, hd, hd, mask.p, 1, st.p, ln.p, B, 14, 4, 40, 1, 0.2,
                                                F32, None, bad.p))
        assert bad.get().tolist() == [0, 1, 1, 1, 1, 1]
        got = do.get()
        assert (got[2:] == 77).all() and (got[:2] != 77).all()
        # no rows at all: the sequences are still looked at
        bad = DBuf(dev, np.zeros(B, np.int32))
        if view == "window":
            check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, do.p, hd, hd, st.p, ln.p, B, 0, 4, 40, 1, 0.2, 2, 9, F32,
                                                  None, bad.p))
        else:
            check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, do.p, hd, hd, mask.p, 1, st.p, ln.p, B, 0, 4, 40, 1, 0.2,
                                                F32, None, bad.p))
        assert bad.get().tolist() == [1] * B


def test_one_workspace_for_every_view(dev):
    """gn_kv_attention's workspace for the largest sizes, with marks behind it."""
    L, check = _lib()
    rng = np.random.default_rng(11)
    kvh, H, hd, P = 2, 4, 64, 64
    lens = [8300, 700, 4200]
    max_pages = -(-8300 // P)
    pages, table = spread(rng, 3, max_pages)
    ref = kvref.Cache(pages, P, kvh, hd, table, rng)
    for b, n in enumerate(lens):
        x = rng.normal(size=(2, n, kvh, hd))
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    need = floats(3, 64, 8300, H, kvh, hd)
    work = DBuf(dev, np.full(need + 4096, 3.25, np.float32))
    for B, new, window in ((3, 1, 5000), (1, 1, 8000), (1, 1, 100), (2, 30, 3000), (1, 64, 8300), (1, 7, 4500)):
        past = [n - new for n in lens[:B]]
        q, q64 = as_dtype(rng.normal(size=(B * new, H * hd)), "f32")
        dq, st, ln = DBuf(dev, q), DBuf(dev, starts_of([new] * B)), DBuf(dev, np.asarray(past, np.int32))
        m = [tree(rng, new) for _ in range(B)]
        dm = DBuf(dev, viewref.words(m, 2).view(np.int32))
        for view in ("window", "tree"):
            log(f"{view} in a larger workspace: B={B} new={new} window={window}")
            do = DBuf(dev, q * 0)
            if view == "window":
                check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, do.p, H * hd, H * hd, st.p, ln.p, B, B * new, new, 8300,
                                                      H, 0.125, 70, window, F32, work.p, None))
            else:
                check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, do.p, H * hd, H * hd, dm.p, 2, st.p, ln.p, B, B * new,
                                                    new, 8300, H, 0.125, F32, work.p, None))
            assert (work.get()[need:] == 3.25).all()
            got = do.get().astype(np.float64).reshape(B, new, H, hd)
            for b in range(B):
                sight = viewref.tree_sight(past[b], m[b]) if view == "tree" else viewref.window_sight(past[b], new, 70, window)
                qs = q64.reshape(B, new, H, hd)[b]
                for t in {0, new - 1}:  # the first and the last of the new tokens
                    row = np.zeros((1, lens[b]), bool)
                    row[0] = sight[t]
                    k, v, _ = ref.read(b, lens[b]) if t == 0 else (k, v, None)
                    for h in range(H):
                        kk, vv = k[row[0], h // 2], v[row[0], h // 2]
                        sc = kk @ qs[t, h] * 0.125
                        p = np.exp(sc - sc.max())
                        p /= p.sum()
                        size = p @ np.abs(vv)
                        lost = 2.0 ** -24 * ((hd + 4) * np.max(np.abs(kk) @ np.abs(qs[t, h])) * 0.125 + 4 * np.abs(sc).max())
                        lim = kvref.bound((p @ vv)[None], size[None], np.array([lost]), lens[b], "f32")[0]
                        assert (np.abs(got[b, t, h] - p @ vv) <= lim).all(), (view, b, t, h)


def test_refusals(dev):
    from goneuron_amd._lib import KVCache
    L, _ = _lib()
    ref = kvref.Cache(4, 16, 2, 32, np.arange(4).reshape(1, 4), np.random.default_rng(6))
    on = OnDevice(dev, ref)
    x, i = DBuf(dev, np.zeros(4096, np.float32)), DBuf(dev, np.zeros(8, np.int32))
    fields = {n: getattr(on.kv, n) for n, _ in KVCache._fields_}

    def win(q=x.p, out=x.p, qs=64, os=64, st=i.p, ln=i.p, B=1, N=1, mn=1, ml=64, heads=2, scale=1.0, sinks=1, window=1, dtype=0,
            work=x.p, **kv):
        return L.gn_kv_attention_window(dev.h, C.byref(KVCache(**{**fields, **kv})), q, out, qs, os, st, ln, B, N, mn, ml, heads,
                                        scale, sinks, window, dtype, work, None)

    def tre(q=x.p, out=x.p, qs=64, os=64, mask=i.p, ms=1, st=i.p, ln=i.p, B=1, N=1, mn=1, ml=64, heads=2, scale=1.0, dtype=0,
            work=x.p, **kv):
        return L.gn_kv_attention_tree(dev.h, C.byref(KVCache(**{**fields, **kv})), q, out, qs, os, mask, ms, st, ln, B, N, mn, ml,
                                      heads, scale, dtype, work, None)

    assert win() == 0 and tre() == 0
    odd = C.c_void_p(x.p.value + 2)
    for f in (win, tre):
        for kw in (dict(page_size=48), dict(pages=0), dict(kv_heads=0), dict(max_pages=0), dict(heads=3), dict(heads=0), dict(k=None),
                   dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(table=None), dict(st=None), dict(ln=None), dict(B=-1),
                   dict(N=-1), dict(mn=-1), dict(ml=-1), dict(dtype=2), dict(q=odd), dict(q=None), dict(out=None), dict(qs=63),
                   dict(os=63), dict(head_dim=0), dict(scale=math.inf), dict(scale=math.nan), dict(work=odd)):
            assert f(**kw) < 0, (f.__name__, kw)
        assert f(head_dim=257) == -4 and f(B=70000) == -4 and f(mn=1 << 27) == -4
        assert f(B=0) == 0 and f(N=0) == 0 and f(mn=0) == 0
    assert win(sinks=-1) == -1 and win(window=-1) == -1
    assert win(ml=60, work=None) == 0 and win(ml=8192, work=None) == 0      # a window of few keys is not split
    assert win(ml=8192, window=8192, work=None) == -1 and tre(ml=8192, work=None) == -1
    assert tre(mask=None) == -1 and tre(mask=C.c_void_p(i.p.value + 1)) == -1
    assert tre(ms=0) == -1 and tre(N=40, mn=33, ms=1) == -1 and tre(N=40, mn=33, ms=2) == 0 and tre(N=4, mn=33, ms=1) == 0
    on.same()
