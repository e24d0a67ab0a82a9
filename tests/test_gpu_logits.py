"""GPU tests of gn_logits_adjust against a float64 restatement (viewref.adjust): each step
rounds once to float32, and a bfloat16 result once more (2^-8 of itself)."""
import ctypes as C

import numpy as np
import pytest

import kvref
import viewref
from gpuutil import DBuf, log
from test_gpu_drafts import bits, rules
from test_gpu_kv_cache import BF16, F32, as_dtype, values

pytestmark = pytest.mark.gpu


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


def case(dev, dtype, B, V, H=0, nb=0, grammar=0, prompt=True, seed=0, gap=0, off=0, in_place=False, zs=None, tokens=None, ids=None,
         settings=None, rows=None):
    L, check = _lib()
    rng = np.random.default_rng(V * 3 + B + seed)
    z, z64 = as_dtype(rng.normal(size=(B, V)) * 3 if zs is None else zs, dtype)
    w = V + gap
    full, mark = np.zeros(off + B * w, z.dtype), as_dtype(np.full(off + B * w, 77.0), dtype)[0]
    full[off:].reshape(B, w)[:, :V] = z
    if in_place:
        mark[off:].reshape(B, w)[:, :V] = z
    R, want = {}, []
    if H:
        R["tokens"] = tokens if tokens is not None else (rng.random((B, H)) ** 2 * V).astype(np.int32)
        R["token_lens"] = rng.integers(0, H + 1, B).astype(np.int32)
        R["token_lens"][0] = H
        if prompt:
            R["prompt_lens"] = (R["token_lens"] * rng.random(B)).astype(np.int32)
        s = settings or dict(repetition=rng.uniform(0.8, 1.4, B), frequency=rng.uniform(-0.2, 0.5, B), presence=rng.uniform(-0.2, 0.5, B))
        R.update({k: np.asarray(v, np.float32) for k, v in s.items()})
    if nb:
        R["bias_ids"] = ids if ids is not None else rng.integers(-2, V + 2, (B, nb)).astype(np.int32)
        R["bias"] = (rng.normal(size=(B, nb)) * 4).astype(np.float32)
        R["bias_lens"] = rng.integers(0, nb + 1, B).astype(np.int32)
        R["bias_lens"][0] = nb
    ok = None
    if grammar:
        ok = rng.random((grammar, V)) < rng.random((grammar, 1))
        ok[0] = False
        R["allowed"] = bits(ok)
        R["allowed"][:, -1] |= -1 << (V % 32) if V % 32 else 0   # bits behind V are nothing
        R["allowed_row"] = (rng.integers(-1, grammar + 1, B) if rows is None else np.asarray(rows)).astype(np.int32)
    rule, held = rules(dev, **R)
    dz, do = DBuf(dev, full), DBuf(dev, mark)
    src = do if in_place else dz
    p = [C.c_void_p(d.p.value + off * z.itemsize) for d in (src, do)]
    check(dev.h, L.gn_logits_adjust(dev.h, p[0], w, p[1], w, F32 if dtype == "f32" else BF16, C.byref(rule), B, V))
    assert dz.get().tobytes() == full.tobytes()
    got = values(do.get(), dtype)
    assert (got[:off] == 77).all() and (got[off:].reshape(B, w)[:, V:] == 77).all()
    got = got[off:].reshape(B, w)[:, :V]
    worst = 0.0
    for b in range(B):
        kw = {}
        if H:
            n = R["token_lens"][b]
            kw = dict(tokens=R["tokens"][b, :n], prompt=R["prompt_lens"][b] if prompt else 0,
                      **{k: R[k][b] for k in ("repetition", "frequency", "presence") if k in R})
        if nb:
            n = R["bias_lens"][b]
            kw.update(ids=R["bias_ids"][b, :n], bias=R["bias"][b, :n])
        if grammar and 0 <= R["allowed_row"][b] < grammar:
            kw.update(allowed=ok[R["allowed_row"][b]])
        y, lim = viewref.adjust(z64[b], **kw)
        if dtype == "bf16":
            lim = lim * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(np.where(np.isfinite(y), y, 0))
            lim[y == z64[b]] = 0       # what no rule touches stays as it is
        fine = np.isfinite(y)
        assert np.array_equal(got[b][~fine], y[~fine], equal_nan=True), b
        assert np.isfinite(got[b][fine]).all()
        d = np.abs(got[b][fine] - y[fine])
        assert (d <= lim[fine]).all(), (b, np.flatnonzero(d > lim[fine])[:5], d.max())
        worst = max(worst, float((d / np.maximum(lim[fine], 1e-300)).max(initial=0)))
    log(f"adjust {dtype} B={B} V={V} history={H} biases={nb} grammars={grammar}: {worst:.3f} of the bound")


SIZES = [
    # dtype, B, V, history, biases, grammars
    ("f32", 4, 8000, 128, 20, 2),
    ("bf16", 5, 50257, 300, 64, 3),
    ("f32", 3, 1, 5, 2, 1),
    ("bf16", 2, 31, 100, 9, 1),
    ("f32", 7, 33, 1, 1, 7),
    ("f32", 2, 131072, 5000, 300, 1),
    ("bf16", 1, 131071, 1, 0, 1),
    ("f32", 1, 1 << 20, 40000, 10, 1),
    ("bf16", 65, 1001, 70, 3, 4),
    ("f32", 3, 4099, 0, 7, 0),
    ("bf16", 3, 4100, 0, 0, 3),
    ("f32", 3, 40961, 70000, 0, 0),       # a history whose counts pass 16 bits
]


@pytest.mark.parametrize("dtype,B,V,H,nb,grammar", SIZES)
def test_all_rules(dev, dtype, B, V, H, nb, grammar):
    case(dev, dtype, B, V, H, nb, grammar)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap,off", [(0, 0), (3, 1), (8, 0), (5, 4), (0, 3)])
def test_rows_of_any_stride_and_start(dev, dtype, gap, off):
    case(dev, dtype, 5, 3001, 200, 20, 2, gap=gap, off=off)
    case(dev, dtype, 5, 3001, 200, 20, 2, gap=gap, off=off, in_place=True)
    case(dev, dtype, 3, 6, 3, 2, 2, gap=gap, off=off)


def test_rows_of_unlike_starts(dev):
    """logits and out that lie differently in their 16 bytes."""
    L, check = _lib()
    rng = np.random.default_rng(4)
    B, V = 3, 2500
    for dtype in ("f32", "bf16"):
        for a, b, wa, wb in ((1, 2, V, V), (0, 3, V + 1, V + 4), (3, 0, V + 5, V)):
            z, z64 = as_dtype(rng.normal(size=a + B * wa), dtype)
            out = as_dtype(np.full(b + B * wb, 77.0), dtype)[0]
            ok = rng.random((1, V)) < 0.5
            R, held = rules(dev, allowed=bits(ok), allowed_row=np.zeros(B, np.int32))
            dz, do = DBuf(dev, z), DBuf(dev, out)
            e = z.itemsize
            check(dev.h, L.gn_logits_adjust(dev.h, C.c_void_p(dz.p.value + a * e), wa, C.c_void_p(do.p.value + b * e), wb,
                                            F32 if dtype == "f32" else BF16, C.byref(R), B, V))
            want = values(out, dtype)
            for r in range(B):
                want[b + r * wb:b + r * wb + V] = np.where(ok[0], z64[a + r * wa:a + r * wa + V], -np.inf)
            assert np.array_equal(values(do.get(), dtype), want)


def test_no_rule_copies(dev):
    L, check = _lib()
    from goneuron_amd._lib import LogitRules
    z = np.random.default_rng(1).normal(size=(3, 777)).astype(np.float32)
    z[0, :4] = [np.nan, np.inf, -np.inf, -0.0]
    dz, do = DBuf(dev, z), DBuf(dev, np.zeros_like(z))
    R = LogitRules()
    check(dev.h, L.gn_logits_adjust(dev.h, dz.p, 777, do.p, 777, F32, C.byref(R), 3, 777))
    assert np.array_equal(do.get().view(np.int32), z.view(np.int32))
    # an id list without values, or a text without penalties, is no rule
    i = DBuf(dev, np.zeros((3, 5), np.int32))
    R = LogitRules(tokens=i.p, tokens_stride=5)
    check(dev.h, L.gn_logits_adjust(dev.h, dz.p, 777, do.p, 777, F32, C.byref(R), 3, 777))
    assert np.array_equal(do.get().view(np.int32), z.view(np.int32))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_that_are_not_finite(dev, dtype):
    z = np.random.default_rng(2).normal(size=(4, 500)).astype(np.float32)
    z[:, ::7], z[:, 1::7], z[:, 2::7], z[:, 3::7], z[:, 4::7] = np.nan, np.inf, -np.inf, 0.0, np.finfo(np.float32).max * 0.9
    case(dev, dtype, 4, 500, 900, 300, 3, zs=z, rows=[-1, 1, 2, 0])


def test_settings_of_any_kind(dev):
    B, V = 8, 300
    s = dict(repetition=[0.0, -1.0, np.nan, np.inf, 1e-30, 1.0, 3e38, 1.5], frequency=[0, 1, 1, 0, 0, np.inf, 1e30, -1e30],
             presence=[0, 0, 1, 0, 0, 1, -np.inf, 1e-40])
    case(dev, "f32", B, V, 400, settings=s)
    for k in s:
        case(dev, "f32", B, V, 400, settings={k: s[k]}, prompt=False)


def test_ids_lengths_and_rows_out_of_range(dev):
    rng = np.random.default_rng(3)
    B, V, H, nb = 6, 200, 50, 12
    tokens = rng.integers(0, V, (B, H)).astype(np.int32)
    tokens[:, ::3] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31, V + 4096], (B, 17))
    ids = rng.integers(0, V, (B, nb)).astype(np.int32)
    ids[:, ::4] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31], (B, 3))
    case(dev, "f32", B, V, H, nb, 2, tokens=tokens, ids=ids, rows=[0, 1, 2, -1, 2 ** 31 - 1, -2 ** 31])
    # lengths beyond the rows and below 0
    L, check = _lib()
    z = rng.normal(size=(3, V)).astype(np.float32)
    lens = np.array([1000, -5, 2 ** 31 - 1], np.int32)
    R, held = rules(dev, tokens=tokens[:3], token_lens=lens, prompt_lens=np.array([-3, 5, 2 ** 31 - 1], np.int32),
                    repetition=np.full(3, 2, np.float32), presence=np.full(3, 1, np.float32), bias_ids=ids[:3],
                    bias=np.ones((3, nb), np.float32), bias_lens=lens)
    dz, do = DBuf(dev, z), DBuf(dev, z * 0)
    check(dev.h, L.gn_logits_adjust(dev.h, dz.p, V, do.p, V, F32, C.byref(R), 3, V))
    got = do.get()
    for b, (n, prompt, m) in enumerate(((H, 0, nb), (0, 0, 0), (H, H, nb))):
        y, lim = viewref.adjust(z[b], tokens[b, :n], prompt, 2.0, None, 1.0, ids[b, :m], np.ones(m))
        assert (np.abs(got[b] - y) <= lim).all()


def test_the_same_id_many_times(dev):
    """Every thread counts the same token; the last of many biases of one id counts."""
    V = 100
    tokens = np.full((2, 20000), 42, np.int32)
    tokens[1, ::2] = 7
    ids = np.full((2, 3000), 5, np.int32)
    ids[1, 1500:] = 6
    case(dev, "f32", 2, V, 20000, 3000, tokens=tokens, ids=ids)


def test_in_front_of_a_draw(dev):
    """A grammar that leaves one token, none, and a bias that bans the rest."""
    L, check = _lib()
    V = 3000
    z = np.random.default_rng(5).normal(size=(3, V)).astype(np.float32)
    ok = np.zeros((2, V), bool)
    ok[0, 1234] = True
    R, held = rules(dev, allowed=bits(ok), allowed_row=np.array([0, 1, -1], np.int32), bias_ids=np.arange(V, dtype=np.int32)[None].repeat(3, 0),
                    bias=np.where(np.arange(V) == 77, 0, -np.inf).astype(np.float32)[None].repeat(3, 0),
                    bias_lens=np.array([0, 0, V], np.int32))
    n = C.c_int64()
    check(None, L.gn_sample_workspace(3, V, C.byref(n)))
    dz, u, ids, work = DBuf(dev, z), DBuf(dev, np.full(3, 0.9, np.float32)), DBuf(dev, np.zeros(3, np.int32)), DBuf(dev, np.zeros(n.value, np.float32))
    check(dev.h, L.gn_logits_adjust(dev.h, dz.p, V, dz.p, V, F32, C.byref(R), 3, V))
    check(dev.h, L.gn_sample(dev.h, dz.p, V, F32, None, None, None, None, u.p, ids.p, 3, V, work.p))
    assert ids.get().tolist() == [1234, -1, 77]


def test_refusals(dev):
    from goneuron_amd._lib import LogitRules
    L, _ = _lib()
    z, i = DBuf(dev, np.ones(4096, np.float32)), DBuf(dev, np.zeros(64, np.int32))
    o = DBuf(dev, np.ones(4096, np.float32))

    def adj(logits=z.p, stride=100, out=o.p, os=100, dtype=0, B=2, V=100, rules=True, **kw):
        return L.gn_logits_adjust(dev.h, logits, stride, out, os, dtype, C.byref(LogitRules(**kw)) if rules else None, B, V)

    odd = C.c_void_p(z.p.value + 2)
    assert adj() == 0 and adj(B=0) == 0 and adj(dtype=1, logits=odd) == 0
    for kw in (dict(logits=None), dict(out=None), dict(stride=99), dict(os=99), dict(dtype=2), dict(B=-1), dict(V=0), dict(rules=False),
               dict(logits=odd), dict(out=odd), dict(out=z.p, os=101), dict(repetition=z.p, tokens_stride=5), dict(tokens_stride=-1),
               dict(bias=z.p, bias_stride=3), dict(bias_ids=i.p, bias_stride=3), dict(bias_stride=-1), dict(presence=odd),
               dict(allowed=i.p, allowed_stride=3, allowed_rows=2), dict(allowed=i.p, allowed_stride=4, allowed_rows=1),
               dict(allowed=i.p, allowed_stride=4, allowed_rows=0, allowed_row=i.p)):
        assert adj(**kw) == -1, kw
    assert adj(V=(1 << 20) + 1, stride=1 << 21, os=1 << 21) == -4 and adj(B=65536) == -4
    assert adj(repetition=z.p, tokens=i.p, tokens_stride=(1 << 30) + 1) == -4
    assert adj(allowed=i.p, allowed_stride=4, allowed_rows=1, allowed_row=i.p) == 0
    assert adj(repetition=z.p) == 0        # no text at all
    assert L.gn_logits_adjust(None, z.p, 100, o.p, 100, 0, C.byref(LogitRules()), 1, 100) == -1
