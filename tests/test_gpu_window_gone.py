"""GPU tests that pages which no query of a windowed call sees may be gone without a flag,
windows of nothing among them, and that those which some query sees are missed."""
import numpy as np
import pytest

from test_gpu_kv_views import case

pytestmark = pytest.mark.gpu
NEW = [("f32", [1, 1, 1]), ("bf16", [1, 1, 1]), ("f32", [50, 3, 1]), ("bf16", [130, 66, 2])]


@pytest.mark.parametrize("dtype,new", NEW)
@pytest.mark.parametrize("sinks", [0, 1, 4, 17, 64, 100, 2 ** 31 - 1])
def test_without_a_window_only_the_first_tokens_count(dev, dtype, new, sinks):
    for past in ([100, 0, 15], [260, 33, 7], [96, 1, 200]):
        bad = case(dev, dtype, 64, 16, 2, 2, past, new, sinks, 0, gone=True, seed=sinks % 97)
        assert not bad.any()


@pytest.mark.parametrize("dtype,new", NEW)
@pytest.mark.parametrize("sinks,window", [(0, 1), (1, 1), (4, 15), (16, 16), (0, 17), (63, 65)])
def test_pages_outside_every_window(dev, dtype, new, sinks, window):
    for past in ([100, 0, 15], [260, 33, 7]):
        bad = case(dev, dtype, 32, 16, 2, 2, past, new, sinks, window, gone=True)
        assert not bad.any()


@pytest.mark.parametrize("dtype,new", NEW)
def test_first_tokens_that_are_not_there(dev, dtype, new):
    """Their page is missed with no window too; the one behind it is not."""

    def spoil(ref):
        ref.table[0, 0] = -1
        ref.table[1, 1] = ref.pages

    bad = case(dev, dtype, 64, 16, 2, 2, [100, 70, 50], new, 5, 0, spoil=spoil)
    assert bad.tolist() == [1, 0, 0]
