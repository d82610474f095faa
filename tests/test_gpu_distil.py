"""GPU tests of the loss against a teacher's top entries and of its gradient, against their definitions in 64 bits
(tests/scores_reference.py)."""
import ctypes

import numpy as np
import pytest

import scores_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -125, "f16": 2.0 ** -25, "bf16": 2.0 ** -125}
U = 2.0 ** -24
# Exponentials of t = (x - top) log2(e) / T: the difference of two numbers of 32 bits is rounded to within U of itself, which puts t off by
# U |t| and its exponential by ln 2 U |t| < 0.7 U |t|; with 16-bit scores the rounding of the product and that of log2(e) / T, U |t| each,
# come on top (1.4 U |t|); the instruction's own error and one product's are two units.
ARGUMENT = {"f32": 0.7 * U, "f16": 2.1 * U, "bf16": 2.1 * U}
# The logarithm of their sum: 32 additions in 32 bits, two units of each, and the arguments' with sum q |t| <= log2 n < 31.
LOG_SUM = {kind: 36 * U + 31 * a for kind, a in ARGUMENT.items()}


@pytest.fixture(scope="module")
def lib():
    from indexsdk_amd import _capi
    return _capi.load(), _capi.check


def at(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def rows_of(x, kind, pad=0, shift=0):
    rows, n = x.shape
    store = torch.full((shift + rows * (n + pad),), 3.0, dtype=TYPES[kind][1], device="cuda")
    view = store[shift:].view(rows, n + pad)[:, :n]
    view.copy_(torch.from_numpy(x).to(TYPES[kind][1]))
    return view


def workspace(lib, rows, n):
    size = ctypes.c_int64()
    lib[1](lib[0].ixa_distil_workspace(rows, n, ctypes.byref(size)))
    return torch.full((size.value + 64,), 0x5a, dtype=torch.uint8, device="cuda"), size.value


def given(x, kind, labels, teacher, whole, T):
    rows, n = x.shape
    return (at(x), x.stride(0), TYPES[kind][0], rows, n, at(labels), at(teacher), labels.shape[1], at(whole), T)


def loss(lib, x, kind, labels, teacher, whole, T, stream=None, out=None, work=None):
    rows, n = x.shape
    value, stats = out or (torch.full((rows + 1,), 9.0, device="cuda"), torch.full((rows + 1, 2), 9.0, device="cuda"))
    work, size = work or workspace(lib, rows, n)
    lib[1](lib[0].ixa_op_distil_loss(*given(x, kind, labels, teacher, whole, T), at(value), at(stats), at(work), size,
                                     ctypes.c_void_p(stream)))
    assert out or (work[-64:] == 0x5a).all()
    return value, stats


def gradient(lib, x, kind, labels, teacher, whole, T, stats, weight, out, stream=None):
    lib[1](lib[0].ixa_op_distil_gradient(*given(x, kind, labels, teacher, whole, T), at(stats), at(weight), at(out), out.stride(0),
                                         ctypes.c_void_p(stream)))
    return out


def step(lib, x, kind, labels, teacher, whole, T, weight, out, value=None, stream=None, work=None):
    rows, n = x.shape
    value = torch.full((rows + 1,), 9.0, device="cuda") if value is None else value
    work, size = work or workspace(lib, rows, n)
    lib[1](lib[0].ixa_op_distil_step(*given(x, kind, labels, teacher, whole, T), at(weight), at(value), at(out), out.stride(0),
                                     at(work), size, ctypes.c_void_p(stream)))
    return value


def compare(kind, T, x64, labels, teacher, whole, weight, value, grad):
    for r in range(len(x64)):
        l, g = ref.distil(x64[r], labels[r], teacher[r], T, None if whole is None else whole[r])
        w = 1.0 if weight is None else weight[r]
        there = (labels[r] >= 0) & (labels[r] < len(x64[r]))
        share = 1.0
        if whole is not None:
            share = np.exp(teacher[r][there] / T - whole[r]).sum()
        assert np.isfinite(l) or np.array_equal(np.float64(value[r]), l, equal_nan=True), (r, value[r], l)
        if np.isfinite(l):
            assert abs(value[r] - l) <= T * T * share * LOG_SUM[kind] + 2 * U * abs(l) + 1e-12, (r, value[r], l)
        if np.isnan(g).any():
            assert np.isnan(g).all() and np.isnan(grad[r]).all()
            continue
        g = g * w
        # q of its own: two units and its argument's; the sum's, and four more products
        some = x64[r] > -np.inf
        t = np.where(some, (np.where(some, x64[r], 0) - x64[r].max(initial=-1e30, where=some)) / T * 1.4427, 0.0)
        q = np.where(some, np.exp2(t), 0)
        q = q / max(q.sum(), 1e-300)
        off = LOG_SUM[kind] + 8 * U + ARGUMENT[kind] * np.abs(t)
        bound = abs(w) * T * share * q * off + (HALF_ULP[kind] + 4 * U) * np.abs(g) + LEAST[kind] + 2.0 ** -120
        bound += abs(w) * T * share * 2.0 ** -126          # exponentials below the least normal number are 0
        np.add.at(bound, labels[r][there], abs(w) * T * 2 * U * share)      # a probability that is added in fp32
        wrong = ~(np.abs(grad[r] - g) <= bound)
        assert not wrong.any(), f"row {r}: {wrong.sum()} gradients are off, first at {np.argmax(wrong)}: " \
                                f"{grad[r][np.argmax(wrong)]} instead of {g[np.argmax(wrong)]}"


def check(lib, x, kind, labels, teacher, T=1.0, whole=None, weight=None, pad=0, shift=0):
    rows, n = x.shape
    T = float(np.float32(T))        # as the entry points take it
    dev = rows_of(x, kind, pad, shift)
    dl, dt = torch.from_numpy(labels).cuda(), torch.from_numpy(teacher.astype(np.float32)).cuda()
    dw = None if whole is None else torch.from_numpy(whole.astype(np.float32)).cuda()
    rw = None if weight is None else torch.from_numpy(weight.astype(np.float32)).cuda()
    as64 = lambda t: None if t is None else t.double().cpu().numpy()
    dtype = TYPES[kind][1]
    value, stats = loss(lib, dev, kind, dl, dt, dw, T)
    out = torch.full((rows + 1, n + 3), 5.0, dtype=dtype, device="cuda")
    gradient(lib, dev, kind, dl, dt, dw, T, stats, rw, out)
    torch.cuda.synchronize()
    assert value[rows] == 9 and (stats[rows] == 9).all() and (out[rows] == 5).all() and (out[:, n:] == 5).all()
    args = (as64(dev), labels, as64(dt), as64(dw), as64(rw))
    compare(kind, T, *args, as64(value[:rows]), as64(out[:rows, :n]))
    # both at a time, and over the scores themselves
    out2 = torch.full((rows + 1, n + 3), 5.0, dtype=dtype, device="cuda")
    both = step(lib, dev, kind, dl, dt, dw, T, rw, out2)
    assert both[rows] == 9 and (out2[rows] == 5).all() and (out2[:, n:] == 5).all()
    compare(kind, T, *args, as64(both[:rows]), as64(out2[:rows, :n]))
    gradient(lib, dev, kind, dl, dt, dw, T, stats, rw, dev)
    assert torch.equal(dev.nan_to_num(7.0), out[:rows, :n].nan_to_num(7.0))
    again = rows_of(x, kind, pad, shift)
    both2 = step(lib, again, kind, dl, dt, dw, T, rw, again)
    assert torch.equal(both.nan_to_num(7.0), both2.nan_to_num(7.0)) and torch.equal(again.nan_to_num(7.0), out2[:rows, :n].nan_to_num(7.0))


def task(rows, n, k, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    x = -1.3 * np.log(rng.random((rows, n)) * n + 1) + rng.standard_normal((rows, n)) * spread + 6
    near = x + 0.7 * rng.standard_normal((rows, n))
    labels = np.argsort(-near, axis=1)[:, :k]
    teacher = np.take_along_axis(near, labels, 1)
    if labels.shape[1] < k:
        labels = np.pad(labels, ((0, 0), (0, k - labels.shape[1])), constant_values=-1)
        teacher = np.pad(teacher, ((0, 0), (0, k - teacher.shape[1])), constant_values=-3.4e38)
    labels[rng.random((rows, k)) < 0.1] = -1
    return x, np.ascontiguousarray(labels.astype(np.int64)), teacher


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,with_whole,weighted", [(1.0, False, False), (2.0, True, True), (0.3, False, True), (20.0, True, False)])
@pytest.mark.parametrize("rows,n,k,pad,shift", [(1, 1, 1, 0, 0), (3, 2, 5, 1, 1), (8, 1024, 10, 0, 0), (5, 63, 63, 3, 1), (4, 8192, 100, 0, 0),
                                                (3, 8193, 300, 5, 3), (2, 70_001, 2048, 0, 1), (2, 140_000, 64, 8, 0), (2500, 500, 7, 0, 0)])
def test_loss_and_gradient(lib, rows, n, k, pad, shift, T, with_whole, weighted, kind):
    x, labels, teacher = task(rows, n, k, rows + n + k)
    rng = np.random.default_rng(1)
    whole = rng.random(rows) + np.log(n) / 2 + np.where(labels >= 0, teacher, -1e30).max(1).clip(-50, None) / T if with_whole else None
    check(lib, x, kind, labels, teacher, T, whole, rng.standard_normal(rows) if weighted else None, pad, shift)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 20_000])
def test_labels_that_come_again_and_labels_that_are_none(lib, kind, n):
    rng = np.random.default_rng(5)
    x, labels, teacher = task(7, n, 40, 6)
    labels[0] = 3                                   # all the same
    labels[1] = rng.integers(0, 5, 40)
    labels[2] = -1
    labels[3] = [n, -5, 2 ** 40, n - 1, 0] * 8      # outside, and the ends
    labels[4, 1:] = -1
    labels[5] = labels[5, ::-1]
    teacher[6, ::3] = -np.inf
    check(lib, x, kind, labels, teacher, 1.5)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [50, 30_000])
def test_masked_scores_and_numbers_that_are_none(lib, kind, n):
    x, labels, teacher = task(9, n, 20, 8)
    labels[labels < 0] = 0
    x[0] = -np.inf                                  # no score
    x[1, 5], x[2, n - 1] = np.nan, np.inf
    keep = np.zeros(n, bool)
    keep[labels[3]] = True
    x[3, ~keep] = -np.inf                           # all but the labels are masked
    x[4, labels[4, 2]] = -np.inf                    # a label asks for a masked column
    x[5] = float(torch.finfo(TYPES[kind][1]).min)   # masked by the lowest number
    x[5, 7] = 1.0
    x[6, n // 2:] = -np.inf
    x[7] = 0.0
    teacher[8] = -np.inf                            # nothing of a teacher
    labels[6] = np.arange(20) % (n // 2)
    labels[5] = 7
    check(lib, x, kind, labels, teacher)


def test_large_scores_and_sharp_temperatures(lib):
    rng = np.random.default_rng(3)
    x, labels, teacher = task(4, 3000, 30, 9)
    for T in (0.01, 0.1):
        check(lib, x, "f32", labels, teacher, T)
    check(lib, x + 1e4, "f32", labels, teacher + 1e4)
    check(lib, x * 1e3, "f32", labels, teacher * 1e3, 100.0)


@pytest.mark.parametrize("weighted", [False, True])
def test_gradient_is_that_of_differences(lib, weighted):
    """Central differences of the loss itself: steps of 2^-5 leave third derivatives (at most T^2 * 2 / T^3 in size) * 2^-10 / 6, and
    two losses of a unit in 2^-20."""
    x, labels, teacher = task(1, 24, 6, 11)
    labels[0, 4] = labels[0, 1]
    h, T = 2.0 ** -5, 2.0
    x = np.round(x * 2 ** 10) / 2 ** 10
    dl, dt = torch.from_numpy(np.repeat(labels, 48, 0)).cuda(), torch.from_numpy(np.repeat(teacher, 48, 0).astype(np.float32)).cuda()
    moved = np.repeat(x, 48, 0)
    moved[np.arange(24), np.arange(24)] += h
    moved[24 + np.arange(24), np.arange(24)] -= h
    value, _ = loss(lib, rows_of(moved, "f32"), "f32", dl, dt, None, T)
    slope = (value[:24] - value[24:48]).double().cpu().numpy() / (2 * h)
    weight = torch.full((1,), 3.0 if weighted else 1.0, device="cuda")
    out = torch.empty(1, 24, device="cuda")
    step(lib, rows_of(x, "f32"), "f32", dl[:1], dt[:1], None, T, weight, out)
    top = value[:48].abs().max().item()
    bound = 2 / T * 2.0 ** -10 / 6 + 2 * (T * T * LOG_SUM["f32"] + U * top) / (2 * h)
    assert np.abs(out[0].double().cpu().numpy() / weight.item() - slope).max() <= bound


def test_rows_past_32_bits(lib):
    """The last rows lie more than 2^32 elements behind the first."""
    n, rows = 2 ** 21 + 1, 2100
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    labels = torch.full((rows, 2), 5, dtype=torch.int64, device="cuda")
    labels[:, 1] = n - 1
    teacher = torch.tensor([[1.0, 0.0]], device="cuda").repeat(rows, 1)
    x[:, 5] = 4.0
    out = torch.empty_like(x)
    value = step(lib, x, "bf16", labels, teacher, None, 1.0, None, out)
    row = np.zeros(n)
    row[5] = 4
    l, g = ref.distil(row, np.array([5, n - 1]), np.array([1.0, 0.0]), 1.0)
    for r in (0, 1, 2047, 2048, rows - 1):
        assert abs(value[r].item() - l) < 1e-4 * l
        got = out[r].double().cpu().numpy()
        assert np.abs(got - g).max() <= 2.0 ** -8 * np.abs(g).max() and abs(got.sum()) < 0.01 and got[5] < 0 and got[n - 1] < 0
    assert torch.equal(out[0], out[-1])


@pytest.mark.parametrize("rows,n", [(3, 500), (2, 100_000)])
def test_captured_steps_give_what_eager_ones_do(lib, rows, n):
    x, labels, teacher = task(rows, n, 30, 13)
    dev = rows_of(x, "bf16")
    dl, dt = torch.from_numpy(labels).cuda(), torch.from_numpy(teacher.astype(np.float32)).cuda()
    out, value, stats = torch.empty_like(dev), torch.zeros(rows + 1, device="cuda"), torch.zeros(rows + 1, 2, device="cuda")
    out2, value2 = torch.empty_like(dev), torch.zeros(rows + 1, device="cuda")
    work = workspace(lib, rows, n)
    step(lib, dev, "bf16", dl, dt, None, 2.0, None, out, value, work=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        step(lib, dev, "bf16", dl, dt, None, 2.0, None, out, value, stream=stream, work=work)
        loss(lib, dev, "bf16", dl, dt, None, 2.0, stream=stream, out=(value2, stats), work=work)
        gradient(lib, dev, "bf16", dl, dt, None, 2.0, stats, None, out2, stream=stream)
    for _ in range(3):
        dev.copy_(dev.roll(1, 1))
        want = torch.empty_like(dev)
        one = step(lib, dev, "bf16", dl, dt, None, 2.0, None, want)
        two, _ = loss(lib, dev, "bf16", dl, dt, None, 2.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(value[:rows], one[:rows]) and torch.equal(value2[:rows], two[:rows])
        assert (out2.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


# Rows that a workgroup keeps in its registers while it writes those before them: every size of a workgroup, and more rows than
# workgroups are resident, in an order in which all kinds of rows follow each other.
@pytest.mark.parametrize("T", [1.0, 1e-6])
@pytest.mark.parametrize("kind,rows,n,k", [("f32", 4400, 13, 3), ("bf16", 4400, 1003, 20), ("bf16", 5000, 260, 256), ("f16", 4200, 8192, 9),
                                           ("f32", 2200, 4100, 20), ("bf16", 2200, 16_384, 20), ("f16", 2300, 1000, 300),
                                           ("bf16", 1100, 17_001, 20), ("f32", 1100, 16_384, 300), ("f16", 600, 60_000, 20),
                                           ("bf16", 300, 131_072, 20), ("f32", 300, 65_533, 20), ("bf16", 300, 70_007, 300)])
def test_rows_in_registers(lib, kind, rows, n, k, T):
    x, labels, teacher = task(13, n, k, 21)
    x[1] = -np.inf
    x[3, n // 2] = np.nan
    x[4, n - 1] = np.inf
    x[5] = float(torch.finfo(TYPES[kind][1]).min)
    x[6] = float(torch.finfo(TYPES[kind][1]).min)
    x[6, n - 1] = 0.0
    x[7, 1:] = -np.inf
    x[8] = float(torch.finfo(TYPES[kind][1]).max)
    labels[9] = -1
    labels[10] = n // 3
    teacher[11] = -np.inf
    labels[7] = 0
    T = float(np.float32(T))
    first = rows_of(x, kind)
    of = torch.arange(rows, device="cuda") % 13
    dev = first[of]
    dl, dt = torch.from_numpy(labels).cuda()[of].contiguous(), torch.from_numpy(teacher.astype(np.float32)).cuda()[of].contiguous()
    out = torch.full((rows + 1, n), 5.0, dtype=dev.dtype, device="cuda")
    value = step(lib, dev, kind, dl, dt, None, T, None, out)
    as64 = lambda t: t.double().cpu().numpy()
    compare(kind, T, as64(first), labels, as64(dt[:13]), None, None, as64(value[:13]), as64(out[:13]))
    assert value[rows] == 9 and (out[rows] == 5).all()
    assert torch.equal(value[:rows].nan_to_num(7.0), value[:13][of].nan_to_num(7.0))
    assert torch.equal(out[:rows].nan_to_num(7.0), out[:13][of].nan_to_num(7.0))
    both = step(lib, dev, kind, dl, dt, None, T, None, dev)
    assert torch.equal(both.nan_to_num(7.0), value.nan_to_num(7.0)) and torch.equal(dev.nan_to_num(7.0), out[:rows].nan_to_num(7.0))
