"""GPU tests that windows and trees stay within the workspace that
gn_kv_attention_workspace grants, where few sequences see the most keys: marks behind it."""
import ctypes as C

import numpy as np
import pytest

import kvref
import viewref
from gpuutil import DBuf, log
from test_gpu_kv_cache import BF16, F32, OnDevice, as_dtype, spread, starts_of, values
from test_gpu_kv_views import floats, tree

pytestmark = pytest.mark.gpu
MARKS = 1 << 19  # floats: more than a split of every key head's rows takes


def _lib():
    from goneuron_amd._lib import check, lib
    return lib(), check


@pytest.mark.parametrize("dtype,kvh,G,past,new,window", [
    ("bf16", 1, 8, [69999], 1, 66000),
    ("f32", 1, 2, [69999], 1, 2 ** 31 - 1),
    ("f32", 2, 1, [50000], 2, 40000),
    ("bf16", 1, 3, [66001, 7, 40000], 1, 65536),
])
def test_long_windows_of_few_sequences(dev, dtype, kvh, G, past, new, window):
    L, check = _lib()
    rng = np.random.default_rng(past[0] + kvh)
    B, H, hd, P = len(past), kvh * G, 32, 128
    lens = [a + new for a in past]
    max_pages = -(-max(lens) // P)
    pages, table = spread(rng, B, max_pages)
    ref = kvref.Cache(pages, P, kvh, hd, table, rng)
    for b, n in enumerate(lens):
        x = rng.normal(size=(2, n, kvh, hd))
        ref.append(b, 0, x[0], x[1])
    on = OnDevice(dev, ref)
    q, q64 = as_dtype(rng.normal(size=(B * new, H * hd)), dtype)
    need = floats(B, new, max(lens), H, kvh, hd)
    work = DBuf(dev, np.full(need + MARKS, 3.25, np.float32))
    dq, st, ln = DBuf(dev, q), DBuf(dev, starts_of([new] * B)), DBuf(dev, np.asarray(past, np.int32))
    masks = [tree(rng, new) for _ in past]
    dm = DBuf(dev, viewref.words(masks, 1).view(np.int32))
    code, w = F32 if dtype == "f32" else BF16, H * hd
    for view in ("window", "tree"):
        log(f"{view} {dtype} kvh={kvh} G={G} past={past} new={new} window={window}")
        do = DBuf(dev, q * 0)
        if view == "window":
            check(dev.h, L.gn_kv_attention_window(dev.h, C.byref(on.kv), dq.p, do.p, w, w, st.p, ln.p, B, B * new, new, max(lens), H,
                                                  0.25, 4, window, code, work.p, None))
        else:
            check(dev.h, L.gn_kv_attention_tree(dev.h, C.byref(on.kv), dq.p, do.p, w, w, dm.p, 1, st.p, ln.p, B, B * new, new, max(lens),
                                                H, 0.25, code, work.p, None))
        assert (work.get()[need:] == 3.25).all()
        got = values(do.get(), dtype).reshape(B, new, H, hd)
        for b in range(B):
            sight = viewref.window_sight(past[b], new, 4, window) if view == "window" else viewref.tree_sight(past[b], masks[b])
            want, size, lost = viewref.attend(ref, b, past[b], q64.reshape(B, new, H, hd)[b], 0.25, sight)
            assert (np.abs(got[b] - want) <= kvref.bound(want, size, lost, lens[b], dtype)).all(), (view, b)
