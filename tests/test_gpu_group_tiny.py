"""GPU tests of products with stores of fewer than four scales, where rows of x are as large or as small as their type has them."""
import numpy as np
import pytest

from test_gpu_group import Store, check_product, lib, rows, torch, vectors  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("m", [4, 100])
@pytest.mark.parametrize("n,d,group", [(1, 30, 32), (3, 32, 32), (1, 96, 32), (1, 150, 64), (2, 61, 64), (3, 128, 128), (1, 384, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_of_very_different_sizes(lib, n, d, group, m, kind, zeros):  # noqa: F811
    """Sums before the scale would pass the largest number of 32 bits, the scores do not."""
    rng = np.random.default_rng(n + d + m)
    x = vectors(m, d, rng)
    with np.errstate(over="ignore", invalid="ignore"):
        x[0] *= np.float32(3e38) / np.abs(x[0]).max()     # or to infinity, where all are below 0.9
    x[1] = 3e38
    x[2] *= 1e-30
    x[3, ::3] *= 2.0 ** 18
    bad = np.repeat(~np.isfinite(x).all(1)[:, None], n, 1)
    store = Store.random(n, d, group, "f32", zeros, rng, size=2.0 ** -30)
    check_product(lib, rows(x, kind), kind, store, "f32", with_bias=False, bad=bad, statistic=False)
    store = Store.random(n, d, group, "f32", zeros, rng, size=2.0 ** 20)
    x[:2] *= 2.0 ** -60
    check_product(lib, rows(x, kind), kind, store, "f32", with_bias=False, bad=bad, statistic=False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,group", [(3, 32, 32), (1, 150, 64), (3, 100, 128)])
def test_infinities_and_nan_stay_in_their_rows(lib, n, d, group, kind):  # noqa: F811
    rng = np.random.default_rng(d)
    x = vectors(5, d, rng)
    x[1, 7], x[2, d - 1], x[3] = np.inf, np.nan, 0.0
    store = Store.random(n, d, group, "f16", True, rng)
    store.scales[0] = float("nan")
    bad = np.zeros((5, n), bool)
    bad[1:3] = True
    bad[:, 0] = True
    check_product(lib, rows(x, kind), kind, store, "f32", bad=bad, statistic=False)
