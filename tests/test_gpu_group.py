"""GPU tests of rows in 4 bits with group scales against their definitions in 64 bits (tests/group_reference.py): codes, scales
and zero points bit for bit, products within what sums in 32 bits can lose."""
import ctypes

import numpy as np
import pytest

import group_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
GUARD = 0x5a


@pytest.fixture(scope="module")
def lib():
    from indexsdk_amd import _capi
    return _capi.load(), _capi.check


def at(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def rows(x, kind, pad=0, shift=0):
    """A device tensor of x in rows of d + pad elements, `shift` elements behind an aligned address."""
    n, d = x.shape
    dtype = TYPES[kind][1]
    store = torch.full((shift + n * (d + pad),), 3.0, dtype=dtype, device="cuda")
    view = store[shift:].view(n, d + pad)[:, :d]
    view.copy_(torch.from_numpy(np.asarray(x)).to(dtype))
    return view


def as64(t):
    return t.detach().cpu().double().numpy()


class Store:
    """Codes, scales and zero points of n rows, with guards behind them."""

    def __init__(self, n, d, group, scale, zeros):
        self.n, self.d, self.group, self.kind = n, d, group, scale
        self.ng = ref.groups_of(d, group)
        self.codes = torch.full((n * self.ng * group // 2 + 64,), GUARD, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((n * self.ng + 16,), 7.0, dtype=TYPES[scale][1], device="cuda")
        self.zeros = torch.full((n * self.ng + 64,), GUARD, dtype=torch.uint8, device="cuda") if zeros else None

    @classmethod
    def random(cls, n, d, group, scale, zeros, rng, size=1.0):
        s = cls(n, d, group, scale, zeros)
        s.codes[:n * s.ng * group // 2] = torch.from_numpy(rng.integers(0, 256, n * s.ng * group // 2, dtype=np.uint8))
        s.scales[:n * s.ng] = torch.from_numpy(size * rng.uniform(0.5, 2.0, n * s.ng)).to(TYPES[scale][1])
        if zeros:
            s.zeros[:n * s.ng] = torch.from_numpy(rng.integers(0, 16, n * s.ng, dtype=np.uint8))
        return s

    def get(self):
        torch.cuda.synchronize()
        size = self.n * self.ng
        codes, scales = self.codes.cpu().numpy(), as64(self.scales)
        zeros = np.full(size + 64, 8, np.uint8) if self.zeros is None else self.zeros.cpu().numpy()
        assert (codes[size * self.group // 2:] == GUARD).all() and (scales[size:] == 7).all()
        assert self.zeros is None or (zeros[size:] == GUARD).all()
        shape = (self.n, self.ng)
        return (ref.unpack(codes[:size * self.group // 2].reshape(self.n, -1), self.group), scales[:size].reshape(shape),
                zeros[:size].reshape(shape))

    def values(self):
        return ref.values(*self.get(), self.d)


def quantise(lib, x, kind, group, scale, zeros, stream=None):
    n, d = x.shape
    s = Store(n, d, group, scale, zeros)
    lib[1](lib[0].ixa_op_group_quantise(at(x), x.stride(0), TYPES[kind][0], n, d, group, TYPES[scale][0], at(s.codes),
                                        at(s.scales), at(s.zeros), ctypes.c_void_p(stream)))
    return s


def workspace(lib, kind, m, d):
    size = ctypes.c_int64()
    lib[1](lib[0].ixa_group_product_workspace(TYPES[kind][0], m, d, ctypes.byref(size)))
    return torch.full((size.value + 64,), GUARD, dtype=torch.uint8, device="cuda"), size.value


def product(lib, x, kind, store, out, out_kind, alpha=1.0, bias=None, stream=None, work=None):
    m, d = x.shape
    work, size = workspace(lib, kind, m, d) if work is None else (work, work.numel())
    lib[1](lib[0].ixa_op_group_product(at(x), x.stride(0), TYPES[kind][0], m, at(store.codes), at(store.scales), at(store.zeros),
                                       store.group, TYPES[store.kind][0], store.n, d, alpha, at(bias), TYPES[out_kind][0],
                                       at(out), out.stride(0), at(work), size, ctypes.c_void_p(stream)))
    return work


# ----- codes ------------------------------------------------------------------------------------------------------------

def sample(n, d, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, d)) * np.exp2(rng.integers(-6, 7, (n, 1)))
    if n > 4:
        x[1] = 0
        x[2] = np.abs(x[2])                      # low is 0
        x[3] = -np.abs(x[3])                     # high is 0
        x[4] = np.rint(x[4] * 4)                 # many halfway points
        x[4, 0] = 7 * 2
    return x.astype(np.float32)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind,scale", [("f32", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,d,pad,shift", [(1, 1, 0, 0), (7, 31, 0, 1), (9, 200, 3, 0), (33, 128, 8, 0), (5, 2100, 1, 3), (300, 96, 0, 0)])
def test_codes_are_those_of_the_definition(lib, n, d, pad, shift, kind, group, scale, zeros):
    x = rows(sample(n, d, n + d), kind, pad, shift)
    s = quantise(lib, x, kind, group, scale, zeros)
    code, scales, zero = s.get()
    want = ref.quantise(as64(x), group, TYPES[scale][0], zeros)
    assert np.array_equal(scales, want[1]) and np.array_equal(zero, want[2])
    assert np.array_equal(code, want[0])
    for kind_out in TYPES:
        out = torch.full((n, d + 2), 9.0, dtype=TYPES[kind_out][1], device="cuda")
        lib[1](lib[0].ixa_op_group_dequantise(at(s.codes), at(s.scales), at(s.zeros), group, TYPES[scale][0], n, d,
                                              TYPES[kind_out][0], at(out), d + 2, None))
        torch.cuda.synchronize()
        v = ref.round_to_type(ref.values(code, scales, zero, d), TYPES[kind_out][0])
        assert np.array_equal(as64(out[:, :d]), v) and (out[:, d:] == 9).all()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", ["f16", "f32", "bf16"])
def test_codes_of_extreme_groups(lib, scale, zeros):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 128)).astype(np.float32)
    x[0] *= 1e-44                        # subnormal
    x[1] *= 1e38 / np.abs(x[1]).max()    # beyond what fp16 scales hold
    x[2, 5], x[3, 40], x[4, 100] = np.inf, np.nan, -np.inf
    x[5] = 3e38
    x[6] = -3e38
    x[7, ::2], x[7, 1::2] = 3.4e38, -3.4e38
    x[8] *= 2e-8                         # fp16 scales are subnormal or 0
    x[9] *= 1e-37
    x[10, 64:] = -0.0
    x[11, 3] = -np.nan
    s = quantise(lib, rows(x, "f32"), "f32", 64, scale, zeros)
    code, scales, zero = s.get()
    want = ref.quantise(x, 64, TYPES[scale][0], zeros)
    assert np.array_equal(scales, want[1], equal_nan=True) and np.array_equal(zero, want[2])
    assert np.array_equal(code, want[0])
    assert np.isnan(scales).sum() == 4
    out = torch.empty(12, 128, device="cuda")
    lib[1](lib[0].ixa_op_group_dequantise(at(s.codes), at(s.scales), at(s.zeros), 64, TYPES[scale][0], 12, 128, 0, at(out), 128,
                                          None))
    assert np.array_equal(as64(out), ref.values(code, scales, zero, 128).astype(np.float32), equal_nan=True)


def test_many_rows_take_several_launches(lib):
    """More rows than half a million workgroups of two long rows each hold."""
    n, d = 1_060_001, 2049
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda").normal_()
    s = quantise(lib, x, "bf16", 128, "bf16", False)
    pick = torch.cat((torch.arange(5), torch.arange(n - 5, n), torch.randint(0, n, (100,)), torch.arange(1048570, 1048580))).cuda()
    code, scale, _ = ref.quantise(as64(x[pick]), 128, 2, False)
    row = s.ng * 64
    assert np.array_equal(s.codes[:n * row].view(n, row)[pick].cpu().numpy(), ref.pack(code))
    assert np.array_equal(as64(s.scales[:n * s.ng].view(n, s.ng)[pick]), scale)
    out = torch.empty_like(x)
    lib[1](lib[0].ixa_op_group_dequantise(at(s.codes), at(s.scales), None, 128, 2, n, d, 2, at(out), d, None))
    v = ref.round_to_type(ref.values(code, scale, np.full(scale.shape, 8), d), 2)
    assert np.array_equal(as64(out[pick]), v)


# ----- products ---------------------------------------------------------------------------------------------------------

def check_product(lib, x, kind, store, out_kind, alpha=1.0, with_bias=True, pad=0, bad=None, statistic=True):
    """Every score within the worst that its sums in 32 bits can lose, and all of them within what they lose by chance."""
    m, d = x.shape
    n = store.n
    bias = torch.randn(n, device="cuda") if with_bias else None
    out = torch.full((m + 1, n + pad), 9.0, dtype=TYPES[out_kind][1], device="cuda")
    work = product(lib, x, kind, store, out, out_kind, alpha, bias)
    torch.cuda.synchronize()
    assert (work[-64:] == GUARD).all()
    assert (out[m] == 9).all() and (out[:, n:] == 9).all()
    got = as64(out[:m, :n])
    a, v = as64(x), store.values()
    with np.errstate(invalid="ignore", over="ignore"):
        g = a @ v.T
        magnitude = np.abs(a) @ np.abs(v).T
    if bad is not None:
        assert np.array_equal(~np.isfinite(got), bad | ~np.isfinite(g))
        g, magnitude = np.where(bad, 0, g), np.where(bad, 0, magnitude)
    # pieces: 2^-39 of the row's largest element, 2^-22 of each in fp32
    lost = np.zeros_like(g)
    if kind != "f16":
        finite = np.where(np.isfinite(a), np.abs(a), 0)
        lost = 2.0 ** -39 * finite.max(1)[:, None] * np.where(np.isfinite(v), np.abs(v), 0).sum(1)[None, :]
    if kind == "f32":
        lost = lost + 2.0 ** -22 * magnitude
    # an addition, rounded or cut off, for each product, one multiply-add per group (two roundings of an intermediate with them)
    pieces = 2 if kind == "f32" else 1
    adds = d * pieces + 2 * store.ng
    bound = lost + adds * 2.0 ** -23 * magnitude
    b = as64(bias)[None, :] if with_bias else 0.0
    want = alpha * g + b
    bound = abs(alpha) * bound * 1.01 + 2.0 ** -23 * np.abs(want) + LEAST[out_kind] + HALF_ULP[out_kind] * np.abs(want)
    with np.errstate(invalid="ignore"):
        error = np.abs(got - want)
        if out_kind == "f16":
            error = np.where((np.abs(want) > 65000) & (np.isinf(got) | (np.abs(got) > 65000)), 0, error)
    error = np.where(bad, 0, error) if bad is not None else error     # those have been compared
    assert (error <= bound).all(), f"{int((error > bound).sum())} scores are off, by up to {(error / bound).max():.2f} of the bound"
    if statistic and out_kind == "f32" and m * n >= 16:
        # by chance: sqrt(additions) roundings of partial sums that are 1 / sqrt(d) of the magnitude, and the pieces'
        per = np.sqrt(np.mean((error / (abs(alpha) * magnitude + np.abs(want) + 1e-300)) ** 2))
        assert per <= 2.0 ** -23 * (np.sqrt(pieces) + 2) + (2.0 ** -22 if kind == "f32" else 0), f"{per * 2 ** 24:.1f} x 2^-24"


def vectors(m, d, rng, spread=2):
    return (rng.standard_normal((m, d)) * np.exp2(rng.integers(-spread, spread + 1, (m, 1)))).astype(np.float32)


@pytest.mark.parametrize("group,scale,zeros", [(32, "f16", False), (64, "bf16", True), (128, "f32", True), (32, "f32", True),
                                               (64, "f16", True), (128, "bf16", False)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (1, 70, 128), (2, 15, 31), (3, 300, 200), (4, 33, 1100), (5, 1000, 129), (8, 17, 2050),
                                   (16, 65, 96), (17, 500, 320), (33, 130, 64), (64, 300, 200), (37, 33_003, 40),
                                   (3, 33_003, 200), (20, 32_801, 33), (2, 32_790, 100)])
def test_few_rows(lib, m, n, d, kind, group, scale, zeros):
    rng = np.random.default_rng(m * n + d)
    store = Store.random(n, d, group, scale, zeros, rng)
    x = rows(vectors(m, d, rng), kind, pad=m % 3, shift=m % 2)
    check_product(lib, x, kind, store, "f32")
    if n < 2000:
        check_product(lib, x, kind, store, "bf16", alpha=-2.0, pad=3)
        check_product(lib, x, kind, store, "f16", alpha=0.125, with_bias=False, pad=1)


@pytest.mark.parametrize("group,scale,zeros", [(32, "f16", True), (64, "bf16", False), (128, "f32", True)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,d", [(65, 1, 1), (65, 130, 33), (128, 128, 128), (130, 257, 200), (200, 300, 1100), (64, 300, 4096),
                                   (16, 200, 8200), (1, 100, 16384), (300, 1000, 64), (50, 257, 2000)])
def test_many_or_long_rows(lib, m, n, d, kind, group, scale, zeros):
    rng = np.random.default_rng(m * n + d)
    store = Store.random(n, d, group, scale, zeros, rng)
    x = rows(vectors(m, d, rng), kind, pad=m % 3, shift=m % 2)
    check_product(lib, x, kind, store, "f32")
    check_product(lib, x, kind, store, "bf16", alpha=-1.0, pad=5)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("m", [3, 70])
def test_rows_of_very_different_sizes(lib, m, kind):
    """Each row has a power of two of its own; within a row large elements meet codes that stand for zero."""
    rng = np.random.default_rng(7)
    x = vectors(m, 256, rng)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2, ::3] *= 2.0 ** 18
    store = Store.random(200, 256, 64, "f32", False, rng)
    check_product(lib, rows(x, kind), kind, store, "f32", with_bias=False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [4, 80])
def test_infinities_and_nan_stay_in_their_rows(lib, m, kind):
    rng = np.random.default_rng(11)
    n, d = 150, 320
    x = vectors(m, d, rng)
    x[1, 7], x[2, 319] = np.inf, np.nan
    store = Store.random(n, d, 64, "f16", True, rng)
    scales = store.scales[:n * store.ng].view(n, store.ng)
    scales[5, 0], scales[149, 4], scales[77, 2] = float("nan"), float("inf"), float("-inf")
    bad = np.zeros((m, n), bool)
    bad[1:3] = True
    bad[:, [5, 149, 77]] = True
    check_product(lib, rows(x, kind), kind, store, "f32", bad=bad, statistic=False)


def test_zero_points_of_a_whole_byte(lib):
    rng = np.random.default_rng(13)
    store = Store.random(90, 200, 32, "f16", True, rng)
    store.zeros[:90 * store.ng] = torch.from_numpy(rng.integers(0, 256, 90 * store.ng, dtype=np.uint8))
    for m in (2, 70):
        check_product(lib, rows(vectors(m, 200, rng), "f16"), "f16", store, "f32", statistic=False)


def test_last_scales_of_an_array_are_read_inside_it(lib):
    """Arrays that end on the last scale, whole groups of loads away from their end or less."""
    rng = np.random.default_rng(17)
    for n, d, group in ((1, 32, 32), (1, 96, 32), (2, 32, 32), (3, 160, 32), (5, 100, 64), (1, 500, 128), (2, 1, 128)):
        store = Store.random(n, d, group, "f16", True, rng)
        store.scales, store.zeros = store.scales[:n * store.ng].clone(), store.zeros[:n * store.ng].clone()
        x = rows(vectors(2, d, rng), "f16")
        out = torch.empty(2, n, device="cuda")
        product(lib, x, "f16", store, out, "f32")
        code = ref.unpack(store.codes[:n * store.ng * group // 2].view(n, -1).cpu().numpy(), group)
        v = ref.values(code, as64(store.scales).reshape(n, -1), store.zeros.cpu().numpy().reshape(n, -1), d)
        want = as64(x) @ v.T
        assert np.allclose(as64(out), want, rtol=1e-5, atol=(d + 8) * 2.0 ** -23 * (np.abs(as64(x)) @ np.abs(v).T).max())


def test_codes_past_32_bits(lib):
    """Rows whose codes lie more than 2^32 bytes behind the first."""
    n, d = 1_100_000, 8192
    store = Store(n, d, 128, "f16", False)
    store.codes.fill_(0x88)                       # zeros
    store.scales.fill_(1.0)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, d, device="cuda", generator=gen).half()
    pick = [0, 524_287, 524_288, 1_048_577, n - 1]
    byte = torch.randint(0, 256, (len(pick), d // 2), dtype=torch.uint8, device="cuda", generator=gen)
    store.codes[:n * d // 2].view(n, d // 2)[pick] = byte
    out = torch.empty(2, n, device="cuda")
    product(lib, x, "f16", store, out, "f32")
    v = ref.values(ref.unpack(byte.cpu().numpy(), 128), np.ones((5, d // 128)), np.full((5, d // 128), 8), d)
    want = as64(x) @ v.T
    assert np.abs(as64(out[:, pick]) - want).max() <= d * 2.0 ** -23 * (np.abs(as64(x)) @ np.abs(v).T).max()
    out[:, pick] = 0
    assert (out == 0).all()


@pytest.mark.parametrize("m", [3, 100])
def test_captured_products_give_what_eager_ones_do(lib, m):
    rng = np.random.default_rng(19)
    n, d = 400, 300
    store = Store.random(n, d, 64, "f16", True, rng)
    x = rows(vectors(m, d, rng), "f32")
    want, out = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    product(lib, x, "f32", store, want, "f32")
    work, _ = workspace(lib, "f32", m, d)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        product(lib, x, "f32", store, out, "f32", stream=torch.cuda.current_stream().cuda_stream, work=work)
    for round_ in range(3):
        out.zero_()
        x += 1
        product(lib, x, "f32", store, want, "f32")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_products_on_two_streams(lib):
    """Two calls at a time with workspaces of their own, and their results."""
    rng = np.random.default_rng(23)
    store = Store.random(3000, 512, 128, "f16", False, rng)
    xs = [rows(vectors(m, 512, rng), "bf16") for m in (2, 150)]
    want = [torch.empty(len(x), 3000, device="cuda") for x in xs]
    out = [torch.empty(len(x), 3000, device="cuda") for x in xs]
    works = [workspace(lib, "bf16", len(x), 512)[0] for x in xs]
    for x, w in zip(xs, want):
        product(lib, x, "bf16", store, w, "f32")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        for x, o, w, s in zip(xs, out, works, streams):
            product(lib, x, "bf16", store, o, "f32", stream=s.cuda_stream, work=w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(out, want))


def test_quantised_rows_score_as_their_values(lib):
    """The three operators together, as a store is filled and asked: codes of rows, the products of some with all, the best."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    n, m, d = 5000, 20, 200
    x = torch.randn(n, d, device="cuda", generator=gen)
    s = quantise(lib, x, "f32", 32, "f16", True)
    back = torch.empty(n, d, device="cuda")
    lib[1](lib[0].ixa_op_group_dequantise(at(s.codes), at(s.scales), at(s.zeros), 32, 1, n, d, 0, at(back), d, None))
    norms = (back.double() ** 2).sum(1).float()
    scores = torch.empty(m, n, device="cuda")
    product(lib, x[:m], "f32", s, scores, "f32", alpha=-2.0, bias=norms)
    dist, label = torch.empty(m, 3, device="cuda"), torch.empty(m, 3, dtype=torch.int64, device="cuda")
    lib[1](lib[0].ixa_op_topk_flat_fp32(at(scores), m, n, n, 3, 1, at(dist), at(label), None))
    exact = torch.cdist(x[:m].double(), back.double()).topk(3, largest=False).indices
    assert (label[:, 0] == torch.arange(m, device="cuda")).all() and (label == exact).float().mean() > 0.95


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_rows_read_back_are_those_of_few(lib, kind):
    n, d, group = 400_000 if kind == "bf16" else 200_000, 201, 32
    store = Store.random(n, d, group, "f16", True, np.random.default_rng(4))
    read = lambda codes, scales, zeros, rows_, out: lib[1](lib[0].ixa_op_group_dequantise(
        at(codes), at(scales), at(zeros), group, 1, rows_, d, TYPES[kind][0], at(out), d, None))
    out, part = torch.empty(n, d, dtype=TYPES[kind][1], device="cuda"), torch.empty(50_000, d, dtype=TYPES[kind][1], device="cuda")
    read(store.codes, store.scales, store.zeros, n, out)
    for first in range(0, n, 50_000):
        slot = first * store.ng
        read(store.codes[slot * group // 2:], store.scales[slot:], store.zeros[slot:], 50_000, part)
        assert torch.equal(out[first:first + 50_000], part)
