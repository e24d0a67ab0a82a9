"""GPU tests of the paged cache's operators in the forms and at the bounds that
test_gpu_kv_cache.py does not reach."""
import ctypes as C
import math

import numpy as np
import pytest

import kvref
from gpuutil import DBuf, log
from test_gpu_kv_cache import BF16, F32, OnDevice, as_dtype, spread, starts_of, values

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
