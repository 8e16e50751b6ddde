"""Corners of row sampling on the GPU that its documentation allows."""
import numpy as np
import pytest

from test_gpu_sample_rows import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [2047, 2048, 2049, 2051, 3500, 4096, 4097])
def test_rows_around_the_length_of_a_list(qtts, V, dtype):
    rng = np.random.default_rng(V)
    n = 20
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    x[:4] = rng.integers(0, 4, (4, V))  # many ties
    x[5] = 0.25
    x[6, 1:] = -np.inf
    x[7, ::2] = np.nan
    check(qtts, x, rng.random(n).astype(np.float32), temperature=rng.choice([0.5, 1.0, 2.0], n),
          top_k=rng.choice([-3, 0, 1, 50, 600, 1100, V - 1], n), top_p=rng.choice([-1.0, 0.3, 0.95, 1.0, 7.0], n),
          min_p=rng.choice([-1.0, 0.0, 0.01], n), dtype=dtype, ld=V + 5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_longest_rows_of_equal_logits(qtts, dtype):
    V = 262144
    x = np.zeros((4, V), np.float32)
    x[1, ::3] = -1.0
    x[2, :100000] = 2.0
    u = np.array([0.0, 0.3, 0.999999, 0.5], np.float32)
    for kw in (dict(), dict(top_p=0.5), dict(top_k=70001), dict(top_k=200000, top_p=0.9, min_p=0.9), dict(temperature=0.0)):
        check(qtts, x, u, dtype=dtype, **kw)


def test_filters_that_are_not_numbers_are_off(qtts):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    check(qtts, x, u, top_p=np.nan)
    check(qtts, x, u, top_k=40, min_p=np.nan)
