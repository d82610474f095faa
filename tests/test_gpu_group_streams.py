"""GPU tests of products of few rows whose pieces fill most of a CU's LDS: every shape of the kernel that keeps them there, by eight
wavefronts and by four, against stores of few and of many rows.  The products in 64 bits are made on the GPU, from the values that the
definition gives (tests/group_reference.py)."""
import numpy as np
import pytest

import group_reference as ref
from test_gpu_group import GUARD, HALF_ULP, LEAST, TYPES, Store, lib, product, rows, torch, vectors  # noqa: F401

pytestmark = pytest.mark.gpu


def values_of(store):
    """The store's values in 64 bits, on the GPU."""
    n, ng, group = store.n, store.ng, store.group
    codes = store.codes[:n * ng * group // 2].view(n, -1)
    v = torch.empty(n, ng * group, dtype=torch.float64, device="cuda")
    v[:, 0::2] = (codes & 15).double()
    v[:, 1::2] = (codes >> 4).double()
    v = v.view(n, ng, group)
    v -= 8 if store.zeros is None else store.zeros[:n * ng].view(n, ng, 1).double()
    v *= store.scales[:n * ng].view(n, ng, 1).double()
    return v.view(n, -1)[:, :store.d]


def check(lib, x, kind, store, out_kind="f32"):  # noqa: F811
    """Every score within the worst that its sums in 32 bits can lose, and all of them within what they lose by chance."""
    m, d = x.shape
    n = store.n
    bias = torch.randn(n, device="cuda")
    out = torch.full((m + 1, n), 9.0, dtype=TYPES[out_kind][1], device="cuda")
    work = product(lib, x, kind, store, out, out_kind, -2.0, bias)
    torch.cuda.synchronize()
    assert (work[-64:] == GUARD).all() and (out[m] == 9).all()
    a, v = x.double(), values_of(store)
    pieces = 2 if kind == "f32" else 1
    lost, g, magnitude = (torch.empty(m, n, dtype=torch.float64, device="cuda") for _ in range(3))
    for i in range(0, n, 4096):
        part = v[i:i + 4096].t().contiguous()
        g[:, i:i + 4096] = a @ part
        part.abs_()
        magnitude[:, i:i + 4096] = a.abs() @ part
        # pieces: 2^-39 of the row's largest element, 2^-22 of each in fp32
        lost[:, i:i + 4096] = 2.0 ** -39 * a.abs().amax(1, keepdim=True) * part.sum(0) if kind != "f16" else 0.0
    if kind == "f32":
        lost += 2.0 ** -22 * magnitude
    # an addition, rounded or cut off, for each product, one multiply-add per group (two roundings of an intermediate with them), and
    # up to three additions of parts of a row
    adds = d * pieces + 2 * store.ng + 3
    want = -2.0 * g + bias.double()
    bound = 2.0 * (lost + adds * 2.0 ** -23 * magnitude) * 1.01 + 2.0 ** -23 * want.abs() + LEAST[out_kind] + HALF_ULP[out_kind] * want.abs()
    error = (out[:m].double() - want).abs()
    assert (error <= bound).all(), f"{int((error > bound).sum())} scores are off, by up to {(error / bound).max().item():.2f} of the bound"
    if out_kind == "f32":
        # by chance: sqrt(additions) roundings of partial sums that are 1 / sqrt(d) of the magnitude, and the pieces'
        per = ((error / (2.0 * magnitude + want.abs() + 1e-300)) ** 2).mean().sqrt().item()
        assert per <= 2.0 ** -23 * (np.sqrt(pieces) + 2) + (2.0 ** -22 if kind == "f32" else 0), f"{per * 2 ** 24:.1f} x 2^-24"


# Rows, dims: more than 72 KB of pieces, 256 bytes for every row and 128 dims, and twice that of fp32.
WIDE = [("f32", 3, 9000), ("f32", 4, 4700), ("f32", 1, 16_384), ("bf16", 4, 9300), ("f16", 3, 16_384), ("f32", 16, 2050), ("bf16", 12, 4096),
        ("f16", 16, 2300), ("bf16", 5, 8200), ("f32", 7, 2700), ("f32", 24, 1000), ("bf16", 24, 2000), ("f16", 17, 4000), ("f32", 32, 1024), ("f32", 40, 417),
        ("f32", 33, 600), ("bf16", 40, 1000), ("f16", 64, 1024), ("bf16", 63, 897), ("bf16", 48, 768), ("f16", 48, 700)]
# and less
FEW = [("f32", 16, 500), ("bf16", 5, 300), ("f16", 9, 1100), ("bf16", 16, 2050), ("f32", 8, 130), ("f32", 20, 300), ("bf16", 30, 700),
       ("f32", 50, 200), ("f16", 64, 500), ("bf16", 3, 1100), ("f32", 6, 1100)]


GROUPS = [(32, "f16", True), (64, "f32", False), (128, "bf16", True), (32, "f32", False), (64, "bf16", True), (128, "f32", True)]


def compare(lib, kind, m, d, n, group, scale, zeros):  # noqa: F811
    rng = np.random.default_rng(m * n + d)
    store = Store(n, d, group, scale, zeros)
    size = n * store.ng
    gen = torch.Generator(device="cuda").manual_seed(m + n + d)
    store.codes[:size * group // 2] = torch.randint(0, 256, (size * group // 2,), dtype=torch.uint8, device="cuda", generator=gen)
    store.scales[:size] = (torch.rand(size, device="cuda", generator=gen) * 1.5 + 0.5).to(TYPES[scale][1])
    if zeros:
        store.zeros[:size] = torch.randint(0, 16, (size,), dtype=torch.uint8, device="cuda", generator=gen)
    x = rows(vectors(m, d, rng), kind, pad=m % 3, shift=m % 2)
    check(lib, x, kind, store)
    if n < 1000:
        check(lib, x, kind, store, "bf16")


@pytest.mark.parametrize("group,scale,zeros", GROUPS)
@pytest.mark.parametrize("n", [300, 33_003])
@pytest.mark.parametrize("kind,m,d", WIDE + FEW)
def test_rows_that_stay(lib, kind, m, d, n, group, scale, zeros):  # noqa: F811
    compare(lib, kind, m, d, n, group, scale, zeros)


@pytest.mark.parametrize("group,scale,zeros", GROUPS)
@pytest.mark.parametrize("kind,m,n,d", [("f32", 64, 300, 2100), ("bf16", 50, 257, 5000), ("f16", 33, 513, 6001), ("f32", 130, 257, 200),
                                        ("bf16", 200, 70, 1100), ("f16", 65, 300, 129)])
def test_rows_in_tiles(lib, kind, m, n, d, group, scale, zeros):  # noqa: F811
    compare(lib, kind, m, d, n, group, scale, zeros)


def test_values_are_those_of_the_definition(lib):  # noqa: F811
    store = Store.random(20, 200, 64, "f16", True, np.random.default_rng(1))
    assert np.array_equal(values_of(store).cpu().numpy(), ref.values(*store.get(), 200))
