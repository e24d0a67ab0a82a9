"""GPU tests of gn_sample on long rows without a cut, and of gn_model_sample at other
widths and on its error path."""
import numpy as np
import pytest

import kvref
from gpuutil import log
from test_gpu_sample import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [16385, 20000, 131072, 300000])
def test_greedy_on_long_rows(dev, V, dtype):
    """Temperatures that take the largest logit, over several workgroups: equal largest
    logits in different ones, infinities and NaN beside them, rows with and without a cut in
    one call."""
    log(f"greedy V={V} {dtype}")
    rng = np.random.default_rng(V)
    z = np.round(rng.normal(size=(9, V)) * 4) / 4  # bfloat16 numbers, many equal
    top = z.max() + 1
    z[0, [V - 1, V // 2, V // 3]] = top
    z[1, V - 1] = top
    z[2, [5000, V - 7]] = np.inf
    z[3, rng.random(V) < 0.5] = np.nan
    z[4] = -np.inf
    z[5] = np.nan
    z[6, 17] = z[6, 16384] = top
    z[7] = -1.5
    z[8, :9000] = -np.inf
    u = np.array([0.999, 0, 0.7, 0.5, 0.5, 0.5, 1, 0.9, 0.3], np.float32)
    greedy = np.array([0, -1, np.nan, 0, 0, -np.inf, 0, 0, 0], np.float32)
    mixed = np.where(np.arange(9) % 2 == 0, greedy, np.float32(0.8)).astype(np.float32)
    got = draw(dev, z, u, dtype, temperature=greedy)
    assert got[:3].tolist() == [V // 3, V - 1, 5000] and got[4] == got[5] == -1 and got[6] == 17 and got[7] == 0
    k = np.array([0, 3, 5000, 0, 7, 0, 2, 9000, 40], np.int32)
    p = np.array([1, 0.5, 0.9, 0.3, 1, 1, 0.2, 0.6, 2], np.float32)
    for T in (greedy, mixed):
        for kw in (dict(), dict(top_k=k), dict(top_p=p), dict(top_k=k, top_p=p, min_p=[0.1] * 9), dict(min_p=[0.5] * 9)):
            draw(dev, z, u, dtype, temperature=T, **kw)


@pytest.mark.parametrize("V,rows", [(5, 3), (9000, 70), (20000, 33)])
def test_model_sample_of_other_widths(gn, dev, V, rows):
    rng = np.random.default_rng(V)
    m = gn.NewSequential(gn.Dense(6, 16, gn.Tanh), gn.Dense(16, V, gn.Linear))
    m.Compile(gn.Adam(1e-3), gn.MSE, max_batch=rows)
    x = rng.normal(size=(rows, 6)).astype(np.float32)
    z = m.PredictBatch(x).astype(np.float64)
    u = rng.random(rows).astype(np.float32)
    for kw in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5, temperature=0.3), dict(top_k=50, min_p=0.01)):
        got = m.Sample(x, u, **kw)
        cast = dict(temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
        want = [kvref.sample(z[b], u[b], **{n: cast[n](v) for n, v in kw.items()}) for b in range(rows)]
        assert got.tolist() == want, kw


def test_model_sample_reports_what_predict_reports(gn, dev):
    """An index outside the Embedding's table is an error of the draw as of the prediction,
    and the model goes on afterwards."""
    from goneuron_amd import configs
    cfg = configs.gpt(B=2, T=4, vocab=10, dim=8, heads=2, ff=8)
    m = configs.build(cfg)
    x, _ = configs.inputs(cfg)
    good = m.PredictBatch(x)
    x[1, 2] = 10
    for call in (lambda: m.PredictBatch(x), lambda: m.Sample(x, [0.5, 0.5])):
        with pytest.raises(gn.GNError) as e:
            call()
        assert e.value.code == -8
    x[1, 2] = 0
    x[1] = x[0]
    assert m.Sample(x, [0.5, 0.5], temperature=0.0).tolist() == [int(np.argmax(good[0]))] * 2
