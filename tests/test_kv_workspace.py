"""CPU checks of the cached attention's workspaces: what is asked for at the largest
sizes serves every smaller call, so it never falls as a size grows."""
import ctypes as C
import os

import pytest

HEADS = [(8, 8, 128), (32, 8, 128), (8, 8, 32), (1, 1, 256), (7, 1, 64), (16, 1, 192), (40, 2, 80), (300, 1, 16)]
B = list(range(1, 40)) + [63, 64, 65, 127, 128, 255, 256, 257, 511, 512, 513, 2047, 2048, 2049, 5000, 65535]
NEW = list(range(1, 36)) + [63, 64, 65, 128, 129, 512, 2048, 20000]  # 300 x 20000 x 300 heads stay below 2^31
LEN = sorted(list(range(1, 9000, 251)) + [4095, 4096, 4097, 8191, 8192, 8200, 16384, 16640, 100000, 2 ** 30, 2 ** 31 - 1])


@pytest.fixture(scope="module")
def L():
    from goneuron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from goneuron_amd import build
        build.build()
    return _lib.lib()


def rising(values, at):
    last = 0
    for x, v in zip(values, map(at, values)):
        assert v >= last, (x, v, last)
        last = v


@pytest.mark.parametrize("heads,kvh,hd", HEADS)
def test_attention_workspace_never_falls(L, heads, kvh, hd):
    n = C.c_int64()

    def floats(b, new, length):
        assert L.gn_kv_attention_workspace(b, new, length, heads, kvh, hd, C.byref(n)) == 0
        return n.value

    for new, length in ((1, 4096), (1, 8200), (1, 131072), (2, 20000), (17, 3000), (40, 100000)):
        rising(B, lambda b: floats(b, new, length))
    for b, length in ((1, 4096), (4, 8192), (64, 8200), (300, 100000)):
        rising(NEW, lambda new: floats(b, new, length))
    for b, new in ((1, 1), (64, 1), (3, 16), (8, 20), (5, 333)):
        rising(LEN, lambda length: floats(b, new, length))


@pytest.mark.parametrize("heads,D", [(8, 256), (4, 64), (1, 256), (12, 960)])
def test_layer_workspace_never_falls(L, heads, D):
    n = C.c_int64()

    def floats(b, rows, new, length):
        assert L.gn_mha_cached_workspace(b, rows, new, length, D, heads, C.byref(n)) == 0
        return n.value

    for new, length in ((1, 4096), (1, 100000), (30, 9000)):
        rising(B, lambda b: floats(b, b * new, new, length))
    for b, length in ((1, 5000), (64, 9000)):
        rising(NEW, lambda new: floats(b, b * new, new, length))
    for b, new in ((8, 1), (2, 40)):
        rising(LEN, lambda length: floats(b, b * new, new, length))
    rising(list(range(1, 600, 7)), lambda rows: floats(8, rows, 1, 4200))


def test_what_a_server_asks_for_once_is_enough_later(L):
    """Sizes between which a plan's own need falls."""
    n, m = C.c_int64(), C.c_int64()
    for large, small, heads in (((64, 1, 8200), (64, 1, 8192), (32, 8, 128)), ((1, 1, 16640), (1, 1, 16384), (32, 8, 128)),
                                ((8, 2048, 4096), (8, 32, 4096), (8, 8, 32)), ((4, 512, 8192), (4, 128, 8192), (32, 8, 128)),
                                ((512, 1, 4096), (256, 1, 4096), (32, 8, 128)), ((512, 1, 8192), (256, 1, 8192), (32, 8, 128))):
        assert L.gn_kv_attention_workspace(*large, *heads, C.byref(n)) == 0
        assert L.gn_kv_attention_workspace(*small, *heads, C.byref(m)) == 0
        assert n.value >= m.value, (large, small)
