"""CPU checks of the token-step entry points that need no device: sizes and
their refusals, and a null context."""
import ctypes as C
import os

import pytest


@pytest.fixture(scope="module")
def L():
    from goneuron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from goneuron_amd import build
        build.build()
    return _lib.lib()


@pytest.mark.parametrize("hd,row", [(1, 32), (32, 32), (33, 64), (65, 96), (97, 128), (128, 128), (129, 192), (193, 256), (256, 256)])
def test_cache_bytes(L, hd, row):
    n, r = C.c_int64(), C.c_int32()
    assert L.gn_kv_cache_bytes(100000, 128, 8, hd, C.byref(n), C.byref(r)) == 0
    assert r.value == row and n.value == 100000 * 128 * 8 * row
    assert L.gn_kv_cache_bytes(1, 16, 1, hd, C.byref(n), None) == 0


@pytest.mark.parametrize("args", [(0, 16, 1, 32), (1, 0, 1, 32), (1, 24, 1, 32), (1, 256, 1, 32), (1, 16, 0, 32), (1, 16, 1, 0),
                                  (1, 16, 1, 257)])
def test_cache_bytes_refuses(L, args):
    n = C.c_int64()
    assert L.gn_kv_cache_bytes(*args, C.byref(n), None) == -1
    assert L.gn_kv_cache_bytes(1, 16, 1, 32, None, None) == -1


def test_workspaces(L):
    n = C.c_int64()
    assert L.gn_kv_attention_workspace(0, 0, 0, 1, 1, 32, C.byref(n)) == 0 and n.value == 0
    # one long sequence is split, a batch that fills the card is not
    assert L.gn_kv_attention_workspace(1, 1, 100000, 8, 8, 128, C.byref(n)) == 0 and n.value > 0
    assert L.gn_kv_attention_workspace(512, 1, 4096, 8, 8, 128, C.byref(n)) == 0 and n.value == 0
    for bad in ((-1, 1, 1, 1, 1, 32), (1, -1, 1, 1, 1, 32), (1, 1, -1, 1, 1, 32), (1, 1, 1, 3, 2, 32), (1, 1, 1, 0, 1, 32),
                (1, 1, 1, 1, 0, 32), (1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 1, 257)):
        assert L.gn_kv_attention_workspace(*bad, C.byref(n)) == -1
    assert L.gn_kv_attention_workspace(1, 1, 1, 1, 1, 32, None) == -1
    assert L.gn_mha_cached_workspace(2, 10, 5, 5, 64, 4, C.byref(n)) == 0 and n.value >= 4 * 10 * 64
    for bad in ((1, 1, 1, 1, 63, 4), (1, 1, 1, 1, 0, 1), (1, -1, 1, 1, 64, 4), (1, 1, 1, 1, 1024, 2)):
        assert L.gn_mha_cached_workspace(*bad, C.byref(n)) == -1
    assert L.gn_sample_workspace(4, 8000, C.byref(n)) == 0 and n.value > 0


def test_null_context(L):
    assert L.gn_kv_append(None, None, *[None] * 4, 0, 0, 0, 0, None, None, 0, None, None, 1, 1, 1, 1, 0, None) == -1
    assert L.gn_kv_attention(None, None, None, None, 0, 0, None, None, 1, 1, 1, 1, 1, 1.0, 1, 0, None, None) == -1
    assert L.gn_sample(None, None, 0, 0, *[None] * 6, 1, 1, None) == -1
    assert L.gn_rope_tables(None, None, None, 1, 2) == -1
    assert L.gn_model_sample(None, None, 1, *[None] * 6) == -1


@pytest.mark.parametrize("V", [8000, 16385, 20001, 131072, 262145, 1 << 20])
def test_sampling_workspace_serves_fewer_rows(L, V):
    n, last = C.c_int64(), 0
    for B in list(range(1, 600)) + [1000, 2047, 2048, 2049, 5000, 65535]:
        assert L.gn_sample_workspace(B, V, C.byref(n)) == 0
        assert n.value >= last
        last = n.value
