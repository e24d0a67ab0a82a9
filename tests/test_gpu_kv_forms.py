"""GPU tests of the paged cache's operators in the forms and at the bounds that
test_gpu_kv_cache.py does not reach."""
import ctypes as C
import math

import numpy as np
import pytest

import kvref
from gpuutil import DBuf, log
from test_gpu_kv_cache import BF16, F32, OnDevice, as_dtype, attention_case, spread, starts_of, values

pytestmark = pytest.mark.gpu


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


def filled(rng, page, kvh, hd, lens):
    """A cache of B sequences of `lens` tokens each."""
    max_pages = max(-(-n // page) for n in lens) + 1
    pages, table = spread(rng, len(lens), max_pages)
    ref = kvref.Cache(pages, page, kvh, hd, table, rng)
    for b, n in enumerate(lens):
        x = rng.normal(size=(2, n, kvh, hd))
        ref.append(b, 0, x[0] * 1.5, x[1])
    return ref


def attention_floats(B, max_new, max_len, heads, kvh, hd):
    L, check = _lib()
    n = C.c_int64()
    check(None, L.gn_kv_attention_workspace(B, max_new, max_len, heads, kvh, hd, C.byref(n)))
    return n.value


@pytest.mark.parametrize("hd,G,past,new", [(128, 4, 300, 64), (64, 2, 0, 257), (96, 1, 120, 40), (256, 1, 70, 30)])
def test_bf16_prompts_are_as_good_as_their_rounding(dev, hd, G, past, new):
    """An output of bfloat16 queries is off by its own rounding (2^-8 of itself at most),
    by float32's errors, and by weights that keep 16 bits: each less than 2^-15 off, the
    sum over them as much, so 2^-14 of sum |w v|.  A weight of 8 bits would not do: its
    2^-9 of |w v| shows where an output is small against its terms."""
    L, check = _lib()
    log(f"bf16 prompt hd={hd} G={G} past={past} new={new}")
    rng = np.random.default_rng(hd + new)
    kvh = 2
    heads = kvh * G
    ref = filled(rng, 32, kvh, hd, [past + new])
    on = OnDevice(dev, ref)
    q, q64 = as_dtype(rng.normal(size=(new, heads * hd)), "bf16")
    work = DBuf(dev, np.full(max(1, attention_floats(1, new, past + new, heads, kvh, hd)), np.nan, np.float32))
    dq, do, st, ln = DBuf(dev, q), DBuf(dev, q * 0), DBuf(dev, starts_of([new])), DBuf(dev, np.array([past], np.int32))
    scale = float(np.float32(1 / math.sqrt(hd)))
    check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, heads * hd, heads * hd, st.p, ln.p, 1, new, new, past + new,
                                   heads, scale, 1, BF16, work.p, None))
    got = values(do.get(), "bf16").reshape(new, heads, hd)
    want, size, lost = kvref.attend(ref, 0, past, q64.reshape(new, heads, hd), scale, 1)
    lim = kvref.bound(want, size, lost, past + new, "f32") + 2.0 ** -14 * size + 2.0 ** -8 * np.abs(want)
    over = np.abs(got - want) / lim
    log(f"{over.max():.3f} of the bound")
    assert over.max() <= 1


def test_one_workspace_for_every_smaller_call(dev):
    """The workspace of the largest sizes, with a border of marks behind it, and calls of
    fewer sequences, new tokens and tokens in it."""
    L, check = _lib()
    rng = np.random.default_rng(21)
    kvh, G, hd = 2, 2, 64
    heads, scale = kvh * G, 0.125
    ref = filled(rng, 64, kvh, hd, [8300, 700, 4200, 40])
    on = OnDevice(dev, ref)
    floats = attention_floats(4, 70, 8300, heads, kvh, hd)
    assert floats > 0
    work = DBuf(dev, np.full(floats + 4096, 3.25, np.float32))
    for B, new, bound in ((4, 1, 8300), (4, 1, 8192), (3, 1, 4400), (1, 1, 8300), (1, 1, 8192), (1, 8, 8200), (2, 9, 8300),
                          (1, 32, 8300), (1, 33, 8192), (2, 64, 8300), (4, 70, 8300), (1, 70, 8300)):
        log(f"attention in a larger workspace: B={B} new={new} max_len={bound}")
        total = [min(n, bound) for n in (8300, 700, 4200, 40)][:B]
        if new > min(total):
            total[total.index(min(total))] = new
        past = [t - new for t in total]
        q, q64 = as_dtype(rng.normal(size=(B * new, heads * hd)), "f32")
        dq, do, st = DBuf(dev, q), DBuf(dev, q * 0), DBuf(dev, starts_of([new] * B))
        ln = DBuf(dev, np.asarray(past, np.int32))
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, heads * hd, heads * hd, st.p, ln.p, B, B * new, new, bound,
                                       heads, scale, 1, F32, work.p, None))
        assert (work.get()[floats:] == 3.25).all()
        got = do.get().astype(np.float64).reshape(B, new, heads, hd)
        for b in range(B):  # the first and the last of the new tokens
            for t in {0, new - 1}:
                want, size, lost = kvref.attend(ref, b, past[b] + t, q64.reshape(B, new, heads, hd)[b, t:t + 1], scale, 1)
                near = np.abs(got[b, t] - want[0]) <= kvref.bound(want, size, lost, total[b], "f32")[0]
                # where a call looks behind what was appended, to pages without a scale: NaN on both sides
                assert (near | (np.isnan(got[b, t]) & np.isnan(want[0]))).all(), (b, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_splits_that_the_scratch_does_not_hold(dev, dtype):
    """512 sequences of one key head of 256 with 16 query heads, told to be up to 4096 long:
    their splits would take more than the context's scratch, so they are not split."""
    L, check = _lib()
    rng = np.random.default_rng(22)
    B, G, hd = 512, 16, 256
    lens = [1 + b % 5 for b in range(B)]
    lens[7] = 300
    ref = filled(rng, 16, 1, hd, lens)
    on = OnDevice(dev, ref)
    assert attention_floats(B, 1, 4096, G, 1, hd) == 0
    q, q64 = as_dtype(rng.normal(size=(B, G * hd)), dtype)
    dq, do, st = DBuf(dev, q), DBuf(dev, q * 0), DBuf(dev, np.arange(B + 1, dtype=np.int32))
    ln = DBuf(dev, np.asarray(lens, np.int32) - 1)
    for bound in (4096, 4000, 3000):
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, G * hd, G * hd, st.p, ln.p, B, B, 1, bound, G, 0.0625, 1,
                                       F32 if dtype == "f32" else BF16, None, None))
        got = values(do.get(), dtype).reshape(B, G, hd)
        for b in list(range(0, B, 37)) + [7, B - 1]:
            want, size, lost = kvref.attend(ref, b, lens[b] - 1, q64.reshape(B, 1, G, hd)[b], 0.0625, 1)
            assert (np.abs(got[b] - want[0]) <= kvref.bound(want, size, lost, lens[b], dtype)[0]).all(), (bound, b)


def test_layer_skips_a_sequence_whole(dev):
    """gn_mha_cached_forward beside a good sequence with one whose positions end behind the
    rotation tables but within max_len, one behind max_len but within the tables, and one
    with negative length: flagged, nothing of theirs stored, their rows wOut's bias, and
    the good sequence's rows as if it were alone."""
    L, check = _lib()
    rng = np.random.default_rng(31)
    heads, hd, page = 2, 32, 16
    D = heads * hd
    nd = D * D + D
    params = (rng.normal(size=4 * nd) / math.sqrt(D)).astype(np.float32)
    cos, sin = kvref.tables(64, hd)
    x = rng.normal(size=(11, D)).astype(np.float32)
    new, past = [3, 3, 3, 2], [9, 30, 46, -1]

    def run(which, rope_len, max_len):
        r = np.random.default_rng(32)
        ref = filled(r, page, heads, hd, [9, 30, 46, 1])
        on = OnDevice(dev, ref)
        before = [a.get() for a in (on.k, on.v, on.ks, on.vs)]
        n = C.c_int64()
        B, N = len(which), sum(new[b] for b in which)
        check(None, L.gn_mha_cached_workspace(B, N, 3, max_len, D, heads, C.byref(n)))
        rows = np.concatenate([x[sum(new[:b]):sum(new[:b + 1])] for b in which])
        dx, dp, do = DBuf(dev, rows), DBuf(dev, params), DBuf(dev, rows * 0 + 5)
        dc, ds, work = DBuf(dev, cos), DBuf(dev, sin), DBuf(dev, np.full(n.value, np.nan, np.float32))
        st, ln, bad = DBuf(dev, starts_of([new[b] for b in which])), DBuf(dev, np.array([past[b] for b in which], np.int32)), \
            DBuf(dev, np.zeros(B, np.int32))
        check(dev.h, L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, do.p, dc.p, ds.p, rope_len, st.p, ln.p, B, N, 3,
                                             max_len, D, work.p, bad.p))
        return ref, before, [a.get() for a in (on.k, on.v, on.ks, on.vs)], do.get(), bad.get().tolist()

    bias = params[3 * nd + D * D:]
    for rope_len, max_len, flags in ((32, 64, [0, 1, 1, 1]), (64, 40, [0, 0, 1, 1]), (64, 12, [0, 1, 1, 1]), (33, 48, [0, 0, 1, 1])):
        ref, before, after, out, bad = run([0, 1, 2, 3], rope_len, max_len)
        assert bad == flags
        alone = run([0], rope_len, max_len)
        assert np.array_equal(out[:3], alone[3][:3])
        s = starts_of(new)
        for b in range(1, 4):
            if flags[b]:
                assert np.array_equal(out[s[b]:s[b + 1]], np.broadcast_to(bias, (new[b], D))), (rope_len, max_len, b)
                for was, now in zip(before, after):
                    assert np.array_equal(was[ref.table[b]], now[ref.table[b]], equal_nan=True), (rope_len, max_len, b)
            else:
                assert not np.array_equal(out[s[b]:s[b + 1]], np.broadcast_to(bias, (new[b], D)))


def test_calls_without_rows_flag_their_sequences(dev):
    """N = 0 or max_new = 0: nothing is stored or written, but what would be skipped is
    flagged as in any other call."""
    L, check = _lib()
    rng = np.random.default_rng(41)
    ref = filled(rng, 16, 1, 32, [20, 20, 20])
    on = OnDevice(dev, ref)
    x = DBuf(dev, np.full(4096, 7, np.float32))
    ln = DBuf(dev, np.array([20, 1000, -1], np.int32))
    for N, max_new, starts, flags in ((0, 5, [0, 0, 0, 0], [0, 1, 1]), (0, 0, [0, 0, 0, 0], [0, 1, 1]), (9, 0, [0, 2, 2, 2], [1, 1, 1]),
                                      (9, 0, [0, 0, 0, 0], [0, 1, 1]), (0, 1, [0, 1, 1, 1], [1, 1, 1])):
        st = DBuf(dev, np.array(starts, np.int32))
        for call in ("append", "attention"):
            bad = DBuf(dev, np.zeros(3, np.int32))
            if call == "append":
                check(dev.h, L.gn_kv_append(dev.h, C.byref(on.kv), x.p, x.p, x.p, x.p, 32, 32, 32, 32, None, None, 0, st.p, ln.p, 3, N,
                                            max_new, 1, F32, bad.p))
            else:
                check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), x.p, x.p, 32, 32, st.p, ln.p, 3, N, max_new, 64, 1, 1.0, 1, F32,
                                               None, bad.p))
            assert bad.get().tolist() == flags, (call, N, max_new, starts)
            on.same()
            assert (x.get() == 7).all()


def test_layer_rows_of_no_sequence(dev):
    """Rows outside every sequence get wOut's bias, where there is no sequence and where
    none may have a token too."""
    L, check = _lib()
    rng = np.random.default_rng(42)
    D, heads, N = 64, 2, 5
    nd = D * D + D
    params = rng.normal(size=4 * nd).astype(np.float32)
    ref = filled(rng, 16, heads, 32, [20, 3])
    on = OnDevice(dev, ref)
    n = C.c_int64()
    dx, dp, x = DBuf(dev, rng.normal(size=(N, D)).astype(np.float32)), DBuf(dev, params), np.full((N, D), 9, np.float32)
    for B, max_new, starts, flags in ((0, 4, [0, 0, 0], [0, 0]), (2, 0, [0, 0, 0], [0, 0]), (2, 0, [0, 3, 3], [1, 0]),
                                      (2, 4, [2, 2, 2], [0, 0])):
        check(None, L.gn_mha_cached_workspace(B, N, max_new, 64, D, heads, C.byref(n)))
        do, work = DBuf(dev, x), DBuf(dev, np.full(n.value, np.nan, np.float32))
        st, ln, bad = DBuf(dev, np.array(starts, np.int32)), DBuf(dev, np.array([20, 3], np.int32)), DBuf(dev, np.zeros(2, np.int32))
        check(dev.h, L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, do.p, None, None, 0, st.p, ln.p, B, N, max_new, 64, D,
                                             work.p, bad.p))
        assert bad.get().tolist() == flags
        assert np.array_equal(do.get(), np.broadcast_to(params[3 * nd + D * D:], (N, D))), (B, max_new)
        on.same()
    assert L.gn_mha_cached_forward(dev.h, C.byref(on.kv), dx.p, dp.p, None, None, None, 0, st.p, ln.p, 0, N, 4, 64, D, work.p, None) == -1
    assert L.gn_mha_cached_forward(dev.h, C.byref(on.kv), None, None, None, None, None, 0, st.p, ln.p, 2, 0, 4, 64, D, None, None) == 0


@pytest.mark.parametrize("dtype,hd,new", [("f32", 64, 1), ("bf16", 128, 1), ("bf16", 256, 1), ("f32", 192, 1), ("bf16", 64, 40),
                                          ("f32", 32, 20)])
def test_score_scales_of_any_size(dev, dtype, hd, new):
    """Score scales down to the smallest number, over keys of 0 (whose block scale is 2^-100)
    and ordinary ones; 0 and negative scales."""
    L, check = _lib()
    rng = np.random.default_rng(hd + new)
    ref = kvref.Cache(20, 16, 2, hd, rng.permutation(20).reshape(2, 10).astype(np.int32), rng)
    lens = [75 + new, 5 + new]
    for b, n in enumerate(lens):
        x = rng.normal(size=(2, n, 2, hd))
        x[0, :40] = 0
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    q, q64 = as_dtype(rng.normal(size=(2 * new, 2 * hd)), dtype)
    work = DBuf(dev, np.zeros(max(1, attention_floats(2, new, 160, 2, 2, hd)), np.float32))
    dq, do, st = DBuf(dev, q), DBuf(dev, q * 0), DBuf(dev, starts_of([new, new]))
    ln = DBuf(dev, np.asarray(lens, np.int32) - new)
    for scale in (1e-20, 1e-36, 1e-45, 0.0, -0.25, 4.0):
        scale = float(np.float32(scale))
        check(dev.h, L.gn_kv_attention(dev.h, C.byref(on.kv), dq.p, do.p, 2 * hd, 2 * hd, st.p, ln.p, 2, 2 * new, new, 160, 2, scale, 1,
                                       F32 if dtype == "f32" else BF16, work.p, None))
        got = values(do.get(), dtype).reshape(2, new, 2, hd)
        for b in range(2):
            want, size, lost = kvref.attend(ref, b, lens[b] - new, q64.reshape(2, new, 2, hd)[b], scale, 1)
            assert (np.abs(got[b] - want) <= kvref.bound(want, size, lost, lens[b], dtype)).all(), (scale, b)


# up to 16 rows a key head: dtype, hd, page, kvh, group, past, new
FEW = [
    ("f32", 72, 16, 2, 2, [333, 0, 701], 1),
    ("bf16", 96, 32, 2, 4, [300, 63], 1),
    ("bf16", 72, 64, 1, 3, [517, 90], 5),
    ("f32", 128, 128, 2, 1, [450, 6], 3),
    ("f32", 160, 64, 1, 2, [619, 127, 0], 1),
    ("bf16", 192, 16, 2, 1, [411, 255], 2),
    ("bf16", 136, 32, 1, 16, [290], 1),
    ("f32", 256, 32, 2, 1, [555, 3], 1),
    ("bf16", 256, 128, 1, 4, [777, 256], 4),
    ("f32", 200, 16, 1, 8, [365], 2),
]


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new", FEW)
def test_few_rows_of_every_head(dev, dtype, hd, page, kvh, G, past, new):
    """Heads of every padded size in the single-token kernel, several steps a wave, lengths
    that end inside a step; told the true length and one that splits the keys."""
    B = len(past)
    for max_len in (None, 20000):
        assert attention_case(dev, dtype, hd, page, kvh, G, past, [new] * B, 1, max_len=max_len).tolist() == [0] * B


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new", FEW)
def test_few_rows_with_missing_pages_and_nan(dev, dtype, hd, page, kvh, G, past, new):
    B = len(past)

    def missing(ref):
        ref.table[0, 1], ref.table[0, past[0] // page // 2] = -1, ref.pages + 7

    def nan(ref):
        for p, h, d, code in ((past[0] // 2, 0, hd - 1, 0x7f), (past[0] + new - 1, kvh - 1, 0, 0xff), (3, 0, hd // 2, 0x7f)):
            ref.v[ref.table[0, p // page], h, d, p % page] = code
        p = past[0] + new - 1  # a key that only the last new token sees
        ref.k[ref.table[0, p // page], 0, p % page, hd - 1] = 0x7f

    for max_len in (None, 9000):
        assert attention_case(dev, dtype, hd, page, kvh, G, past, [new] * B, 1, max_len=max_len, spoil=missing)[0] == 1
        attention_case(dev, dtype, hd, page, kvh, G, past, [new] * B, 1, max_len=max_len, spoil=nan)


@pytest.mark.parametrize("dtype,hd,page,kvh,G,past,new", [
    ("f32", 128, 32, 2, 2, [70, 0, 129], [90, 33, 1]), ("f32", 104, 16, 1, 3, [5], [140]), ("bf16", 192, 64, 1, 2, [100, 0], [65, 130]),
    ("bf16", 136, 32, 2, 1, [40], [77]), ("f32", 256, 64, 1, 1, [200], [70]), ("f32", 160, 128, 1, 5, [9, 300], [40, 17])])
def test_prompts_of_every_head(dev, dtype, hd, page, kvh, G, past, new):
    """Heads of every padded size in the prompts' kernel, whole and split along the keys,
    with missing pages and NaN."""
    def missing(ref):
        ref.table[0, 0] = -3

    def nan(ref):
        p = past[0] + new[0] // 2
        ref.v[ref.table[0, p // page], 0, hd - 1, p % page] = 0x7f
        ref.k[ref.table[0, (p + 3) // page], kvh - 1, (p + 3) % page, 1] = 0xff

    for max_len in (None, 3000):
        for spoil in (None, missing, nan):
            bad = attention_case(dev, dtype, hd, page, kvh, G, past, new, 1, max_len=max_len, spoil=spoil)
            assert bad.tolist() == [int(spoil is missing)] + [0] * (len(past) - 1)
    attention_case(dev, dtype, hd, page, kvh, G, past, new, 0)
