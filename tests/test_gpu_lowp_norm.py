"""GPU tests of the root-mean-square norm into codes, as tight as its arithmetic is: only eight squares at a time are added in 32
bits, so that the error of a value does not grow with the row and a column left out of the mean shows at every length."""
import numpy as np
import pytest

import lowp_reference as ref
from test_gpu_lowp import INT8, MXFP4, MXFP8, TYPES, U, Codes, as64, at, lib, norm, rows, sample  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# Eight squares added in 32 bits: 8 U of the mean at most, 4 U of its root; all else up to the root's reciprocal is in 64 bits.
ROOT = 4 * U
# Before microscaled codes nothing else is lost but one rounding to odd, which leaves a value on its side of every halfway point.
MX = ROOT + U
# Before int8 codes the root's reciprocal and the products with it and with the weight are rounded to 32 bits each.
INT = ROOT + 3 * U

# one length of each of the kernel's shapes, with an end inside a block, a lane's eight elements or neither
LENGTHS = [33, 200, 520, 1000, 2056, 4100, 8200, 16384]


def check(y, got, fmt):
    codes, scales, sqr = got
    d = y.shape[1]
    if fmt == INT8:
        step = np.abs(y).max(-1) / 127
        assert (np.abs(scales - step) <= (INT + U) * 1.001 * step).all()     # and the division
        # in steps: the value's error, the largest value's, and 127 / max and the product with it rounded to 32 bits
        assert (np.abs(codes - y / step[:, None]) <= 0.5 + 127 * (2 * INT + 2 * U) * 1.001).all()
        v = codes * scales[:, None].astype(np.float64)
    else:
        v = ref.mx_values(codes, scales, fmt)[:, :d]

        def quantised(z):
            c, s = ref.mx_codes(z, fmt)
            return ref.mx_values(ref.pack(c, fmt), s, fmt)[:, :d]
        assert ref.between(v, y, MX * 1.001, quantised).all()
    s = (v ** 2).sum(-1)
    assert (np.abs(sqr - s) <= (d + 8) * U * s).all()


@pytest.mark.parametrize("d", LENGTHS)
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
@pytest.mark.parametrize("kind,residual,weight,pad", [("f32", False, False, 0), ("bf16", True, True, 3), ("f16", True, False, 8),
                                                      ("f32", True, True, 0)])
def test_values_are_off_by_a_few_roundings_at_any_length(lib, d, fmt, kind, residual, weight, pad):  # noqa: F811
    n = 37 if d <= 4100 else 11
    # the last columns are the largest: a mean without them is far off
    x = sample(n, d, d) * (1 + 3 * (np.arange(d) >= d - 4)).astype(np.float32)
    x = rows(x, kind, pad)
    res = rows(sample(n, d, d + 1), kind, pad) if residual else None
    w = rows(np.abs(sample(1, d, d + 2)) + np.float32(0.5), kind)[0] if weight else None
    got, total = norm(lib, x, res, w, kind, fmt)
    h = x.float() + (res.float() if residual else 0)
    assert torch.equal(total, h.to(x.dtype))
    check(ref.rms_norm(as64(h), None, None if w is None else as64(w), np.float32(1e-6)), got, fmt)


@pytest.mark.parametrize("left_out", [1, 4, 8])
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_a_mean_without_its_last_columns_would_be_seen(left_out, fmt):
    """The same check on values whose mean lacks a few of 16384 columns."""
    d, n = 16384, 11
    x = sample(n, d, d) * (1 + 3 * (np.arange(d) >= d - 4)).astype(np.float32)
    y = ref.rms_norm(x, None, None, np.float32(1e-6))
    z = x / np.sqrt((x[:, :d - left_out].astype(np.float64) ** 2).sum(-1, keepdims=True) / d + 1e-6)

    def got(v):
        if fmt == INT8:
            c, s = ref.int8_codes(v)
            q = c * s[:, None].astype(np.float64)
        else:
            c, s = ref.mx_codes(v, fmt)
            c = ref.pack(c, fmt)
            q = ref.mx_values(c, s, fmt)
        return c, s, (q ** 2).sum(-1)
    check(y, got(y), fmt)
    with pytest.raises(AssertionError):
        check(y, got(z), fmt)


@pytest.mark.parametrize("d", [40, 768, 5000])
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
@pytest.mark.parametrize("size,eps", [(2e-20, 1e-40), (3e-23, 1e-45), (1e-30, 1e-45), (1e-16, 1e-36), (5e-24, 1e-38)])
def test_squares_that_are_too_small_for_32_bits(lib, d, fmt, size, eps):  # noqa: F811
    """Rows and an epsilon whose squares are subnormal or nothing in 32 bits."""
    x = rows(sample(9, d, d) * np.float32(size), "f32")
    got, _ = norm(lib, x, None, None, "f32", fmt, eps=eps, keep_sum=False)
    y = ref.rms_norm(as64(x), None, None, float(np.float32(eps)))
    keep = np.abs(y).max() > 1e-6       # smaller results are still squared right, but their codes' squares may be nothing
    if keep:
        check(y, got, fmt)
    else:
        assert np.allclose(got[1] if fmt == INT8 else got[1].astype(float),
                           np.abs(y).max(-1) / 127 if fmt == INT8 else ref.mx_codes(y, fmt)[1], rtol=1e-6)


@pytest.mark.parametrize("d", [100, 768, 5000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_the_sum_over_an_input(lib, d, kind, over):  # noqa: F811
    """The sum in the place of x or of the residual, with and without gaps between rows."""
    for pad in (0, 8, 3):
        x, res = rows(sample(9, d, 3), kind, pad), rows(sample(9, d, 4), kind, pad)
        want = (x.float() + res.float()).to(x.dtype)
        (codes, scales, sqr), _ = norm(lib, x, res, None, kind, INT8)
        into, out = (x if over == "x" else res), Codes(9, d, INT8)
        lib[1](lib[0].ixa_op_rms_norm_quantise(at(x), d + pad, at(res), d + pad, None, TYPES[kind][0], 9, d, 1e-6, at(into), d + pad,
                                               INT8, 0.0, at(out.codes), at(out.scales), at(out.sqr), None))
        torch.cuda.synchronize()
        got = out.get()
        assert torch.equal(into, want)
        assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales) and np.array_equal(got[2], sqr)


def test_the_sum_beside_an_input(lib):  # noqa: F811
    """x and the sum are column ranges of one buffer."""
    d, n = 72, 50
    both = torch.full((n, 2 * d), 9.0, device="cuda")
    both[:, :d] = torch.from_numpy(sample(n, d, 6)).cuda()
    first, res = both[:, :d].clone(), rows(sample(n, d, 7), "f32")
    out = Codes(n, d, MXFP8)
    lib[1](lib[0].ixa_op_rms_norm_quantise(at(both), 2 * d, at(res), d, None, 0, n, d, 1e-6, at(both[:, d:]), 2 * d, MXFP8, 0.0,
                                           at(out.codes), at(out.scales), at(out.sqr), None))
    torch.cuda.synchronize()
    assert torch.equal(both[:, :d], first) and torch.equal(both[:, d:], first + res)
    check(ref.rms_norm(as64(first + res), None, None, np.float32(1e-6)), out.get(), MXFP8)
