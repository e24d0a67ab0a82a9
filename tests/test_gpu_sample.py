"""GPU tests of gn_sample, gn_model_sample and Sequential.Sample against a
float64 restatement (kvref.sample): the same index, whatever the filters, ties
and numbers that are not finite.  A draw within the integer weights' resolution
(2^-43 a weight) of a border could differ; none of these lies there."""
import ctypes as C

import numpy as np
import pytest

import kvref
from gpuutil import DBuf, log

pytestmark = pytest.mark.gpu


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


def draw(dev, z, u, dtype="f32", temperature=None, top_k=None, top_p=None, min_p=None, gap=0, off=0):
    L, check = _lib()
    B, V = z.shape
    a = np.asarray(z, np.float32) if dtype == "f32" else kvref.bf16_bits(z)
    full = np.zeros(off + B * (V + gap), a.dtype)
    full[off:].reshape(B, V + gap)[:, :V] = a
    dz = DBuf(dev, full)
    n = C.c_int64()
    check(None, L.gn_sample_workspace(B, V, C.byref(n)))
    work = DBuf(dev, np.frombuffer(np.random.default_rng(1).bytes(4 * n.value), np.float32))
    settings = [None if s is None else DBuf(dev, np.asarray(s, t)) for s, t in
                ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    du, ids = DBuf(dev, np.asarray(u, np.float32)), DBuf(dev, np.full(B, -7, np.int32))
    for _ in range(2):
        check(dev.h, L.gn_sample(dev.h, C.c_void_p(dz.p.value + off * a.itemsize), V + gap, 0 if dtype == "f32" else 1,
                                 *[s.p if s else None for s in settings], du.p, ids.p, B, V, work.p))
    got = ids.get()
    held = a.astype(np.float64) if dtype == "f32" else kvref.bf16_value(a).astype(np.float64)

    def at(s, b):
        return None if s is None else np.float64(s[b])

    want = [kvref.sample(held[b], np.float32(u[b]), *(None if s is None else np.asarray(s, t)[b] for s, t in
                         ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))))
            for b in range(B)]
    assert got.tolist() == want, [(b, int(got[b]), want[b]) for b in range(B) if got[b] != want[b]][:5]
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 63), (4, 1000), (2, 8000), (7, 50257), (3, 131072), (130, 20001)])
def test_every_filter(dev, B, V, dtype):
    log(f"sample B={B} V={V} {dtype}")
    rng = np.random.default_rng(V)
    z = rng.normal(size=(B, V)) * 2 + 6 * (rng.random((B, V)) < 20 / V)
    u = rng.random(B).astype(np.float32)
    T = rng.uniform(0.5, 1.5, B).astype(np.float32)
    k = rng.integers(0, min(V, 1000) + 2, B).astype(np.int32)
    p = rng.uniform(0.3, 1.05, B).astype(np.float32)
    m = rng.uniform(0, 0.2, B).astype(np.float32)
    for kw in (dict(), dict(temperature=T), dict(top_k=k), dict(top_p=p), dict(min_p=m),
               dict(temperature=T, top_k=k, top_p=p, min_p=m), dict(temperature=T, top_k=k, top_p=p)):
        draw(dev, z, u, dtype, **kw)


def test_settings_at_their_ends(dev):
    rng = np.random.default_rng(2)
    V = 777
    z = np.repeat(rng.normal(size=(1, V)), 14, 0)
    T = np.array([1, 1, 1, 1, 1, 1, 0, -1, np.nan, np.inf, 1e-30, 1e-40, 1, 1], np.float32)
    k = np.array([0, -3, 1, V, V + 9, V - 1, 9, 9, 9, 9, 9, 9, 2, 2 ** 31 - 1], np.int32)
    p = np.array([1, 2, 1, 0, -1, 1e-9, .5, .5, .5, .5, .5, .5, 1, np.nan], np.float32)
    m = np.array([0, -1, 0, 0, 0, 0, .5, .5, .5, .5, .5, .5, 1, 2], np.float32)
    for u in (0.0, 0.5, np.float32(1 - 2.0 ** -24), 1.0, -1.0):
        draw(dev, z, np.full(14, u, np.float32), temperature=T, top_k=k, top_p=p, min_p=m)


def test_equal_logits_go_by_the_lowest_index(dev):
    rng = np.random.default_rng(3)
    B, V = 6, 30000
    z = np.zeros((B, V))
    z[1] = rng.integers(0, 3, V)
    z[2] = rng.integers(-2, 2, V)
    z[3, ::2] = -0.0
    z[4] = -5.0
    z[5, :] = np.where(np.arange(V) % 3 == 0, 1.0, 0.0)
    u = rng.random(B)
    for k, p in ((1, 1), (7, 1), (9000, 1), (V, 0.5), (12000, 0.77), (0, 0.1)):
        draw(dev, z, u, top_k=[k] * B, top_p=[p] * B)
        draw(dev, z, u, "bf16", top_k=[k] * B, top_p=[p] * B, min_p=[0.3] * B)


def test_numbers_that_are_not_finite(dev):
    rng = np.random.default_rng(4)
    B, V = 9, 5000
    z = rng.normal(size=(B, V)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, :] = -np.inf
    z[2, 4321] = -3.0e38
    z[3, 17] = np.inf
    z[4, [9, 4000, 4999]] = np.inf
    z[5, rng.random(V) < 0.5] = np.nan
    z[6, rng.random(V) < 0.5] = -np.inf
    z[7] = np.finfo(np.float32).min
    z[8, :] = np.where(np.arange(V) % 2 == 0, np.finfo(np.float32).min, np.finfo(np.float32).max)
    u = rng.random(B)
    got = draw(dev, z, u)
    assert got[0] == got[1] == -1 and got[2] == 4321 and got[3] == 17
    for kw in (dict(top_k=[3] * B), dict(top_p=[0.9] * B), dict(top_k=[2000] * B, top_p=[0.6] * B, min_p=[0.1] * B),
               dict(temperature=[0.0] * B), dict(temperature=[0.7] * B, min_p=[0.01] * B)):
        draw(dev, z, u, **kw)
        draw(dev, z, u, "bf16", **kw)


def test_rows_with_a_stride_and_at_odd_addresses(dev):
    rng = np.random.default_rng(5)
    z, u = rng.normal(size=(5, 9001)) * 3, rng.random(5)
    for dtype in ("f32", "bf16"):
        for gap, off in ((0, 0), (7, 0), (3, 1), (15, 16)):
            draw(dev, z, u, dtype, top_k=[50] * 5, top_p=[0.8] * 5, gap=gap, off=off)


def test_largest_vocabulary(dev):
    rng = np.random.default_rng(6)
    V = 1 << 20
    draw(dev, rng.normal(size=(2, V)), rng.random(2), top_k=[900000, 5], top_p=[0.99, 0.5])
    draw(dev, np.zeros((1, V)), [0.999], top_p=[0.7])


@pytest.mark.parametrize("V", [2048, 2049, 8192, 8193, 16384, 16385, 262143, 262145])
def test_sizes_at_which_the_way_changes(dev, V):
    log(f"sample V={V}")
    rng = np.random.default_rng(V)
    B = 6
    z, u = rng.normal(size=(B, V)) * 3, rng.random(B)
    k = [1, 2047, 2048, 2049, min(V, 9000), 0]
    for dtype in ("f32", "bf16"):
        for kw in (dict(), dict(top_k=k), dict(top_p=[0.85] * B), dict(top_k=k, top_p=[0.85, 0.3, 0.99, 0.6, 0.9, 0.4]),
                   dict(top_k=k, top_p=[0.9] * B, min_p=[0.05] * B), dict(top_k=k, min_p=[0.02] * B)):
            draw(dev, z, u, dtype, **kw)


@pytest.mark.parametrize("V", [5000, 20011, 70001])
def test_more_equal_logits_than_a_list_of_candidates(dev, V):
    log(f"sample ties V={V}")
    rng = np.random.default_rng(V + 1)
    z = np.zeros((6, V))
    z[1] = rng.integers(0, 2, V)
    z[2, V // 3] = 4.0
    z[3] = np.where(np.arange(V) < V - 100, -1.0, -1.0 - 2.0 ** -20)
    z[4] = -np.inf
    z[4, ::2] = 2.5
    z[5, :40] = np.linspace(1, 2, 40)
    u = rng.random(6)
    for k in (50, 2048, 4096):
        for kw in (dict(), dict(min_p=[0.2] * 6)):
            for q in (0.61, 0.999):
                draw(dev, z, u, top_k=[k] * 6, top_p=[q] * 6, **kw)
                draw(dev, z, u, "bf16", top_k=[k] * 6, top_p=[q] * 6, **kw)


@pytest.mark.parametrize("V", [3001, 33333])
def test_large_numbers_and_temperatures(dev, V):
    """Grid lines far from zero, where float32 holds no single one of them."""
    log(f"sample large V={V}")
    rng = np.random.default_rng(V + 2)
    z = rng.normal(size=(8, V)).astype(np.float32) * np.float32(3)
    z[1] += np.float32(1e6)
    z[2] -= np.float32(3e7)
    z[3] *= np.float32(1e30)
    z[4] *= np.float32(1e-30)
    z[5] *= np.float32(1e-42)                     # denormal
    z[6, rng.random(V) < 0.4] = -np.inf
    z[6, 11] = np.nan
    z[7, rng.integers(0, V, 3)] = np.inf
    u = rng.random(8)
    for T in (1.0, 0.01, 300.0, 1e-30, 1e-40, 1e30, np.inf):
        for kw in (dict(), dict(top_k=[700] * 8), dict(top_p=[0.8] * 8), dict(min_p=[0.3] * 8),
                   dict(top_k=[1500] * 8, top_p=[0.8] * 8, min_p=[1e-3] * 8), dict(top_k=[2500] * 8, top_p=[0.7] * 8)):
            draw(dev, z, u, temperature=[T] * 8, **kw)


def test_draws_follow_the_weights(dev):
    """One row drawn at many equally spaced u: each index as often as its weight says, to one draw."""
    z = np.log(np.array([0.1, 0.2, 0.05, 0.4, 0.25]))
    n = 4000
    u = (np.arange(n) + 0.5) / n
    got = draw(dev, np.repeat(z[None], n, 0), u)
    w = np.exp(z.astype(np.float32).astype(np.float64))
    assert np.abs(np.bincount(got, minlength=5) - n * w / w.sum()).max() <= 1


def test_refusals(dev):
    L, _ = _lib()
    n = C.c_int64()
    f, i = DBuf(dev, np.zeros(4096, np.float32)), DBuf(dev, np.zeros(8, np.int32))
    assert L.gn_sample_workspace(1, 0, C.byref(n)) == -1 and L.gn_sample_workspace(1, (1 << 20) + 1, C.byref(n)) == -1
    assert L.gn_sample_workspace(-1, 8, C.byref(n)) == -1 and L.gn_sample_workspace(1, 8, None) == -1

    def call(z=f.p, stride=8, dtype=0, u=f.p, ids=i.p, B=1, V=8, work=f.p):
        return L.gn_sample(dev.h, z, stride, dtype, None, None, None, None, u, ids, B, V, work)

    assert call(B=0) == 0
    for kw in (dict(z=None), dict(u=None), dict(ids=None), dict(work=None), dict(stride=7), dict(dtype=2), dict(V=0), dict(B=-1),
               dict(z=C.c_void_p(f.p.value + 2)), dict(work=C.c_void_p(f.p.value + 4))):
        assert call(**kw) == -1, kw
    assert call(V=(1 << 20) + 1, stride=1 << 21) == -4 and call(B=70000) == -4


def test_model_sample(gn, dev):
    rng = np.random.default_rng(7)
    m = gn.NewSequential(gn.Dense(12, 40, gn.Tanh), gn.Dense(40, 97, gn.Ref(gn.LogSoftmax)))
    m.Compile(gn.Adam(1e-3), gn.CrossEntropy, max_batch=8)
    x = rng.normal(size=(19, 12)).astype(np.float32)      # more rows than the model was compiled for
    z = m.PredictBatch(x).astype(np.float64)
    u = rng.random(19).astype(np.float32)
    for kw in (dict(), dict(temperature=0.5), dict(top_k=5, top_p=0.9), dict(temperature=0.0), dict(min_p=0.2),
               dict(top_k=np.arange(19))):
        got = m.Sample(x, u, **kw)
        rows = {n: np.broadcast_to(np.asarray(v), (19,)) for n, v in kw.items()}
        want = [kvref.sample(z[b], u[b], *(None if n not in rows else np.asarray(rows[n][b], t) for n, t in
                             (("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32))))
                for b in range(19)]
        assert got.tolist() == want, kw
    assert m.Sample(x[:0], u[:0]).size == 0
    with pytest.raises(gn.GNError):
        m.Sample(x, None)
    p = gn.NewSequential(gn.Dense(4, 5, gn.Ref(gn.Softmax)))
    p.Compile(gn.Adam(1e-3), gn.CrossEntropy, max_batch=8)
    with pytest.raises(gn.GNError, match="UNSUPPORTED"):
        p.Sample(rng.normal(size=(2, 4)), [0.1, 0.2])
    e = gn.NewSequential(gn.Embedding(10, 4), gn.Flatten(), gn.Dense(8, 10, gn.Ref(gn.LogSoftmax)))
    try:
        e.Compile(gn.Adam(1e-3), gn.CrossEntropy, max_batch=8)
    except gn.GNError:
        return
    with pytest.raises(gn.GNError):
        e.Sample(np.array([[1.0, 99.0]]), [0.5])
