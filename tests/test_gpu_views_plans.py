"""GPU tests of windows and trees on both sides of what decides whether the waves of a
workgroup share their rows: heads of 128 and more, few and many sequences, short and long
histories."""
import numpy as np
import pytest

from test_gpu_kv_views import case, tree

pytestmark = pytest.mark.gpu
SIZES = [
    # dtype, hd, kvh, group, past, new: rows that the waves share ...
    ("bf16", 128, 1, 4, [100], [60]),
    ("bf16", 112, 2, 1, [700, 3], [200, 170]),
    ("bf16", 128, 1, 8, [40, 9, 300], [64, 1, 22]),
    # ... and rows of their own: a long history, many sequences
    ("bf16", 128, 1, 4, [4100], [45]),
    ("bf16", 128, 1, 1, [4200, 17], [161, 3]),
]


def spoiled(ref, past, new, rng):
    """NaN in keys and values, in sight and out of it, and a page that is not there."""
    for b in range(len(past)):
        for p in {0, past[b] // 2, past[b], past[b] + new[b] - 1}:
            if not 0 <= p < past[b] + new[b]:
                continue
            page, t = ref.table[b, p // ref.P], p % ref.P
            ref.v[page, 0, (p * 5) % ref.hd, t] = 0x7f
            if p % 2:
                ref.k[page, ref.kvh - 1, t, 5] = 0x7f
    ref.table[0, 2] = ref.pages


def views(rng, past, new, view):
    return dict(masks=[tree(rng, n) for n in new]) if view == "tree" else dict(sinks=5, window=max(past) // 2 + 7)


@pytest.mark.parametrize("dtype,hd,kvh,G,past,new", SIZES)
@pytest.mark.parametrize("view", ["window", "tree"])
@pytest.mark.parametrize("kind", ["plain", "spoiled"])
def test_few_sequences(dev, kind, view, dtype, hd, kvh, G, past, new):
    rng = np.random.default_rng(hd + sum(past) + sum(new))
    spoil = (lambda ref: spoiled(ref, past, new, rng)) if kind == "spoiled" else None
    case(dev, dtype, hd, 16, kvh, G, past, new, spoil=spoil, **views(rng, past, new, view))


@pytest.mark.parametrize("dtype,hd,B,most", [("f32", 128, 150, 32), ("bf16", 192, 140, 32), ("f32", 256, 150, 30), ("bf16", 128, 120, 96)])
@pytest.mark.parametrize("past_to", [20, 300])
@pytest.mark.parametrize("view", ["window", "tree"])
@pytest.mark.parametrize("kind", ["plain", "spoiled"])
def test_many_sequences(dev, kind, view, past_to, dtype, hd, B, most):
    """Mostly of a token or none, a few of the most."""
    rng = np.random.default_rng(hd + B + past_to)
    past, new = [int(x) for x in rng.integers(0, 20, B)], [int(x) for x in rng.integers(0, 3, B)]
    for b, n in ((0, most), (5, most - 1), (B - 1, 17)):
        past[b], new[b] = past_to, n
    spoil = (lambda ref: spoiled(ref, past, new, rng)) if kind == "spoiled" else None
    case(dev, dtype, hd, 16, 2, 2, past, new, spoil=spoil, **views(rng, past, new, view))
