"""CPU checks that what gn_kv_attention_workspace grants holds what each of the cached
attentions takes: the plan of a call (gn_kv_attention_need, not of the public interface)
against the grant for its sizes and for larger ones."""
import ctypes as C
import os
import random

import pytest

PREFIX, WINDOW, TREE = range(3)
HEADS = [(8, 1, 128), (16, 2, 128), (24, 3, 64), (1, 1, 32), (2, 2, 256), (12, 3, 80), (32, 8, 128), (8, 8, 96), (40, 2, 192), (300, 1, 16)]
ALL = 2 ** 31 - 1


@pytest.fixture(scope="module")
def L():
    from goneuron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from goneuron_amd import build
        build.build()
    L = _lib.lib()
    L.gn_kv_attention_need.restype, L.gn_kv_attention_need.argtypes = C.c_int64, [C.c_int32] * 10
    return L


def grant(L, B, new, length, heads):
    n = C.c_int64()
    assert L.gn_kv_attention_workspace(B, new, length, *heads, C.byref(n)) == 0
    return n.value


def needs(L, B, new, length, heads, windows):
    """(need, view, dtype, window) of every view and type."""
    for dtype in (0, 1):
        yield L.gn_kv_attention_need(PREFIX, B, new, length, *heads, 0, 0, dtype), "prefix", dtype, None
        yield L.gn_kv_attention_need(TREE, B, new, length, *heads, 0, 0, dtype), "tree", dtype, None
        for sinks, window in windows:
            yield L.gn_kv_attention_need(WINDOW, B, new, length, *heads, sinks, window, dtype), "window", dtype, (sinks, window)


@pytest.mark.parametrize("B,heads,length,window", [
    (1, (8, 1, 128), 131072, 65536), (1, (16, 2, 128), 131072, 65536), (3, (8, 1, 128), 131072, 131072), (1, (8, 1, 128), 200000, ALL),
    (1, (8, 1, 128), 131072, 131072), (1, (8, 1, 128), 131072, 40000), (3, (8, 1, 128), 131072, 65536)])
def test_long_windows_of_few_sequences(L, B, heads, length, window):
    need = L.gn_kv_attention_need(WINDOW, B, 1, length, *heads, 4, window, 0)
    assert 0 < need <= grant(L, B, 1, length, heads)


def test_sizes_that_no_call_has(L):
    good = dict(view=WINDOW, B=1, new=1, length=9000, heads=8, kvh=1, hd=64, sinks=0, window=9000, dtype=0)
    assert L.gn_kv_attention_need(*good.values()) > 0
    for kw in (dict(view=-1), dict(view=3), dict(B=0), dict(new=0), dict(length=-1), dict(heads=0), dict(kvh=0), dict(kvh=3), dict(hd=0),
               dict(hd=257), dict(sinks=-1), dict(window=-1), dict(B=ALL, new=ALL)):
        assert L.gn_kv_attention_need(*{**good, **kw}.values()) == -1, kw


@pytest.mark.parametrize("heads", HEADS)
def test_few_sequences_of_every_view(L, heads):
    windows = [(s, w) for s in (0, 4, 70000, ALL) for w in (1, 4096, 32768, 33333, 40000, 65536, 131072, ALL)]
    for B in (1, 2, 3, 5):
        for new in (1, 2, 5, 16, 17, 40, 128):
            for length in (4096, 4097, 33000, 70000, 131072, 262144, ALL):
                have = grant(L, B, new, length, heads)
                for need, *what in needs(L, B, new, length, heads, windows):
                    assert need <= have, (B, new, length, what)


@pytest.mark.parametrize("heads", HEADS)
def test_sizes_at_random(L, heads):
    """Also what a program asked for once, at larger sizes."""
    rng = random.Random(str(heads))

    def log(lo, hi):
        return min(hi, int(lo * (hi / lo) ** rng.random() + rng.random()))

    for _ in range(1500):
        B, new, length = log(1, 3000), log(1, 5000), log(1, 2 ** 31 - 1)
        if B * new * heads[0] > 2 ** 28:
            continue
        more = [(B, new, length), (B * rng.choice([1, 2, 3]) + rng.randrange(3), new * rng.choice([1, 2]) + rng.randrange(5),
                                   min(length + rng.randrange(9000), ALL))]
        have = [grant(L, *m, heads) for m in more]
        for need, *what in needs(L, B, new, length, heads, [(log(1, length) - 1, log(1, ALL)) for _ in range(3)]):
            assert need <= min(have), (more, have, need, what)


@pytest.mark.parametrize("B,new,length,heads,rows", [(8, 128, 8192, (32, 8, 64), 65536), (2, 2000, 4000, (8, 8, 96), 65536),
                                                     (1, 64, 32768, (16, 2, 32), 65536), (3, 300, 9000, (12, 3, 80), 65280)])
def test_heads_that_share_their_rows_take_no_more_than_prefixes(L, B, new, length, heads, rows):
    """As many (split, token, head) rows as prefixes are split into, each with a maximum and a sum."""
    R = next(r for r in (32, 64, 96) if r >= heads[2])
    assert grant(L, B, new, length, heads) == rows * (R + 2)


# ---------------------------------------------------------------- the layer, which sees prefixes alone
def layer(L, B, rows, new, length, D, heads):
    """Floats that it asks for beside its own rows."""
    n = C.c_int64()
    assert L.gn_mha_cached_workspace(B, rows, new, length, D, heads, C.byref(n)) == 0
    return n.value - 4 * ((rows * D + 63) // 64 * 64)


@pytest.mark.parametrize("B,new,length,D,heads,floats", [
    # 65536 (split, token, head) rows at most, of 128 floats and two
    (2, 2048, 4096, 4096, 32, 65536 * 130), (1, 8192, 8192, 512, 4, 65536 * 130), (4, 16, 8192, 256, 8, 278528)])
def test_the_layer_does_not_pay_for_trees(L, B, new, length, D, heads, floats):
    assert layer(L, B, B * new, new, length, D, heads) == floats


@pytest.mark.parametrize("D,heads", [(256, 8), (256, 1), (64, 4), (960, 12), (4096, 32), (1024, 8)])
def test_the_layer_at_random(L, D, heads):
    rng = random.Random(D + heads)
    for _ in range(3000):
        B, new = int(3000 ** rng.random()), int(5000 ** rng.random())
        length = int((2 ** 31 - 1) ** rng.random())
        if B * new * heads > 2 ** 28:
            continue
        need = L.gn_kv_attention_need(PREFIX, B, new, length, heads, heads, D // heads, 0, 0, 0)
        more = (B + rng.randrange(3), new * rng.choice([1, 2]) + rng.randrange(3), min(length + rng.randrange(5000), ALL))
        assert need <= layer(L, B, B, new, length, D, heads) and need <= layer(L, more[0], B, *more[1:], D, heads)
