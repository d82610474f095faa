"""GPU tests of draws from rows with weights of less than 2^-960 of the best one's, which count as 0: a random number of 0 takes the
first column that counts."""
import numpy as np
import pytest

from test_gpu_sample import check, lib, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("filters", [dict(), dict(temperature=0.05), dict(temperature=30.0), dict(top_p=0.9), dict(top_k=100)], ids=str)
@pytest.mark.parametrize("rows,n", [(6, 1000), (6, 9001), (6, 40_000), (3, 100_003), (130, 70_001)])
def test_weights_that_count_as_nothing(lib, rows, n, kind, filters):  # noqa: F811
    rng = np.random.default_rng(n)
    x = np.stack([rng.uniform(-3000, 0, n), rng.standard_normal(n) * 300, np.sort(rng.uniform(-3000, 3000, n))])
    check(lib, np.tile(x, ((rows + 2) // 3, 1))[:rows], kind, draws=4, **filters)


@pytest.mark.parametrize("temperature", [1e-30, 1e-5, 0.01, 1.0, 1e30, np.inf])
def test_borders_next_to_the_best(lib, temperature):  # noqa: F811
    """Scores so large, or temperatures so small, that nothing but the best counts; and those with which all do."""
    rng = np.random.default_rng(1)
    x = np.stack([1e8 - 8.0 * rng.integers(0, 200, 20_000), -1e30 * rng.random(20_000), rng.standard_normal(20_000), -rng.random(20_000) * 3e38,
                  np.sort(rng.random(20_000))])
    check(lib, x, "f32", draws=4, temperature=temperature)
