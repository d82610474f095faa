"""GPU tests that the gradient at a label is rounded once: values within 2^-25 of themselves of the middle between two numbers of a 16-bit
type, which two roundings, to 32 bits and from there, put on the other side."""
import numpy as np
import pytest

from test_gpu_distil import gradient, lib, loss, rows_of, step, torch  # noqa: F401

pytestmark = pytest.mark.gpu
BITS = {"f16": 11, "bf16": 8}


def rounded(v, bits):
    m, e = np.frexp(v)
    return np.ldexp(np.rint(np.ldexp(m, bits)), e - bits)      # to nearest, halfway to even; nothing here is subnormal


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,times", [(2, 1), (16, 1), (16, 20), (9000, 1)])
def test_gradients_at_labels_are_rounded_once(lib, kind, n, times):  # noqa: F811
    """One label per row with a probability of 1, all scores equal: the gradient there is weight T (1 / m - 1) for m scores that are not
    masked, a power of two of them, which 64 bits hold."""
    bits, T = BITS[kind], float(np.float32(1.3713531))
    there = 2 if n == 2 else 16
    halfway = (2.0 ** bits + 2 * np.arange(2 ** (bits - 1)) + 1) / 2.0 ** bits
    weight = (halfway / (1 - 1 / there) / T).astype(np.float32)
    exact = -weight.astype(np.float64) * T * (1 - 1 / there)
    want = rounded(exact, bits)
    twice = rounded(exact.astype(np.float32).astype(np.float64), bits)
    assert (want != twice).sum() > len(want) // 10       # the rows are what the test is for
    rows = len(weight)
    x = np.full((rows, n), -np.inf)
    x[:, :there] = 0
    of = np.tile(np.arange(rows), times)
    dev = rows_of(x[of], kind)
    labels = torch.zeros(rows * times, 1, dtype=torch.int64, device="cuda")
    teacher = torch.zeros(rows * times, 1, device="cuda")
    w = torch.from_numpy(weight[of]).cuda()
    out = torch.empty(rows * times, n, dtype=dev.dtype, device="cuda")
    step(lib, dev, kind, labels, teacher, None, T, w, out)
    assert np.array_equal(out[:, 0].double().cpu().numpy(), want[of])
    _, stats = loss(lib, dev, kind, labels, teacher, None, T)
    out.fill_(5)
    gradient(lib, dev, kind, labels, teacher, None, T, stats, w, out)
    assert np.array_equal(out[:, 0].double().cpu().numpy(), want[of])
