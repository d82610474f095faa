"""GPU tests of draws from rows of scores against their definition in 64 bits (tests/scores_reference.py)."""
import ctypes

import numpy as np
import pytest

import scores_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
# sums of up to 2^20 weights in 64 bits, in another order (2^-53 each), of exponentials to 1e-14
SLACK = 2e-13


@pytest.fixture(scope="module")
def lib():
    from indexsdk_amd import _capi
    return _capi.load(), _capi.check


def at(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def workspace(lib, rows, n):
    size = ctypes.c_int64()
    lib[1](lib[0].ixa_sample_workspace(rows, n, ctypes.byref(size)))
    return torch.full((size.value + 64,), 0x5a, dtype=torch.uint8, device="cuda"), size.value


def as_setting(v, rows, dtype):
    if v is None:
        return None
    return torch.tensor(np.broadcast_to(np.asarray(v), (rows,)).copy(), device="cuda").to(dtype)


def call(lib, x, kind, uniform, temperature=None, top_k=None, top_p=None, min_p=None, probs=True, stream=None, out=None, work=None):
    rows, n = x.shape
    draws = uniform.shape[1]
    labels, p = out or (torch.full((rows + 1, draws), -7, dtype=torch.int64, device="cuda"),
                        torch.full((rows + 1, draws), 9.0, device="cuda"))
    work, size = workspace(lib, rows, n) if work is None else work
    lib[1](lib[0].ixa_op_sample(at(x), x.stride(0), TYPES[kind][0], rows, n, at(temperature), at(top_k), at(top_p), at(min_p),
                                at(uniform), draws, at(labels), at(p if probs else None), at(work), size,
                                ctypes.c_void_p(stream)))
    return labels, p, work


def check(lib, x, kind, draws=16, seed=0, pad=0, shift=0, **settings):
    """x (rows, n) in 64 bits -> its draws, all compared."""
    rows, n = x.shape
    store = torch.full((shift + rows * (n + pad),), 50.0, dtype=TYPES[kind][1], device="cuda")
    view = store[shift:].view(rows, n + pad)[:, :n]
    view.copy_(torch.from_numpy(x).to(TYPES[kind][1]))
    rng = np.random.default_rng(seed)
    u = rng.random((rows, draws)).astype(np.float32)
    u[:, :1] = 0
    if draws > 3:
        u[:, 1:4] = [1 - 2.0 ** -24, 0.5, 0.25]
    uniform = torch.from_numpy(u).cuda()
    s = {"temperature": (as_setting(settings.get("temperature"), rows, torch.float32), 1.0),
         "top_k": (as_setting(settings.get("top_k"), rows, torch.int32), 0),
         "top_p": (as_setting(settings.get("top_p"), rows, torch.float32), 1.0),
         "min_p": (as_setting(settings.get("min_p"), rows, torch.float32), 0.0)}
    labels, probs, work = call(lib, view, kind, uniform, **{k: v[0] for k, v in s.items()})
    torch.cuda.synchronize()
    labels, probs = labels.cpu().numpy(), probs.cpu().numpy().astype(np.float64)
    assert (labels[rows] == -7).all() and (probs[rows] == 9).all() and (work[-64:] == 0x5a).all()
    there = view.double().cpu().numpy()
    sizes = []
    for r in range(rows):
        w = ref.kept_weights(there[r], **{k: v[1] if v[0] is None else v[0][r].item() for k, v in s.items()})
        sizes.append(int((w > 0).sum()))
        for d in range(draws):
            assert ref.drawn(w, u[r, d], labels[r, d], probs[r, d], SLACK), \
                f"row {r}, draw {d} ({u[r, d]}): label {labels[r, d]}, probability {probs[r, d]}; {sizes[-1]} columns are left"
    return labels, sizes


def scores(rows, n, seed, flat=1.0):
    rng = np.random.default_rng(seed)
    return -1.3 * flat * np.log(rng.random((rows, n)) * n + 1) + flat * rng.standard_normal((rows, n)) + 6


SIZES = [(1, 1, 0, 0), (3, 2, 1, 1), (5, 63, 0, 0), (2, 500, 3, 1), (3, 513, 0, 0), (2, 1024, 0, 0), (3, 4099, 5, 3), (2, 8192, 0, 0),
         (2, 20_001, 0, 1), (3, 100_003, 0, 0), (300, 1000, 0, 0), (270, 9000, 1, 0)]
FILTERS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.0),
           dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.01), dict(temperature=1.5, top_p=0.8), dict(top_k=700),
           dict(top_k=3000, top_p=0.7), dict(temperature=0.05, top_p=0.99, min_p=0.3)]


@pytest.mark.parametrize("filters", FILTERS, ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()) or "none")
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,pad,shift", SIZES)
def test_draws(lib, rows, n, pad, shift, kind, filters):
    check(lib, scores(rows, n, rows * n), kind, pad=pad, shift=shift, **filters)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3000, 60_000])
@pytest.mark.parametrize("filters", [dict(top_p=0.9), dict(top_p=0.5, min_p=0.2), dict(top_k=2000), dict(top_k=2500, top_p=0.6),
                                     dict(min_p=0.5), dict(temperature=3.0, top_p=0.3), dict(top_p=0.999)], ids=str)
def test_flat_rows_keep_more_than_the_list_holds(lib, kind, n, filters):
    x = scores(4, n, n, flat=0.3)
    _, sizes = check(lib, x, kind, **filters)
    if n > 10_000 and filters in (dict(top_p=0.9), dict(top_p=0.999), dict(top_k=2000)):
        assert max(sizes) > 1024      # the rows are what the test is for


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=3), dict(top_k=1000), dict(top_k=2500), dict(top_p=0.25), dict(top_p=0.9),
                                     dict(min_p=1.0), dict(top_p=0.3, top_k=4000, min_p=0.5)], ids=str)
def test_ties_go_to_the_lower_columns(lib, kind, filters):
    rng = np.random.default_rng(3)
    n = 9001
    x = np.zeros((6, n))
    x[1] = rng.integers(0, 2, n)                   # two values
    x[2] = rng.integers(0, 7, n) * 0.5
    x[3, ::2] = -0.0                               # equal to 0
    x[4] = -5
    x[4, 8000:] = 2
    x[5, :] = -1e4
    check(lib, x, kind, **filters)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=600, top_p=0.5),
                                     dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("n", [77, 30_000])
def test_columns_that_are_not_there(lib, kind, n, filters):
    """Masks of -infinity, of the type's lowest number and of NaN, rows without a column, infinities."""
    x = scores(10, n, n)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 3:] = -np.inf
    x[3, ::2] = np.nan
    x[4, :-1] = -np.inf
    x[5, 1:] = float(torch.finfo(TYPES[kind][1]).min)
    x[6, [4, 70]] = np.inf
    x[7] = np.inf
    x[8, 10], x[8, 11], x[8, 12] = np.inf, np.nan, -np.inf
    x[9] = float(torch.finfo(TYPES[kind][1]).min)
    labels, sizes = check(lib, x, kind, **filters)
    assert (labels[:2] == -1).sum() == 2 * 16 and sizes[4] == 1 and sizes[6] <= 2


@pytest.mark.parametrize("order", ["rising", "falling", "first", "last"])
@pytest.mark.parametrize("filters", [dict(top_k=50), dict(top_p=0.9), dict(min_p=0.02), dict()], ids=str)
def test_rows_whose_best_lie_together(lib, order, filters):
    """A bound from the first columns that is far too high or far too low."""
    x = np.sort(scores(2, 50_000, 5), axis=1)
    if order == "falling":
        x = x[:, ::-1].copy()
    elif order != "rising":
        x -= 20
        x[:, slice(0, 30) if order == "first" else slice(49_970, 50_000)] += 25
    check(lib, x, "f32", **filters)


@pytest.mark.parametrize("setting,values", [
    ("temperature", [1e-30, 1e-3, 1e-45, 1e30, np.inf, -1.0, np.nan, 100.0]), ("top_k", [-1, 2 ** 31 - 1, 4000, 3999, 512, 513, 1, 0]),
    ("top_p", [0.0, -1.0, 1.0, 2.0, np.nan, 1e-30, 0.9999999, 0.5]), ("min_p", [0.0, -1.0, 1.0, 2.0, np.nan, 1e-30, 0.9999999, 0.5])])
@pytest.mark.parametrize("others", [dict(), dict(top_p=0.8), dict(top_k=100)], ids=str)
def test_settings_at_their_ends(lib, setting, values, others):
    check(lib, scores(8, 4000, 9), "f32", **{**others, setting: np.array(values)})


def test_rows_of_settings(lib):
    rng = np.random.default_rng(12)
    rows = 40
    check(lib, scores(rows, 30_001, 13), "bf16", temperature=rng.choice([0.0, 0.5, 1.0, 1.4], rows), top_k=rng.choice([0, 5, 60, 900], rows),
          top_p=rng.choice([0.5, 0.9, 1.0], rows), min_p=rng.choice([0.0, 0.01, 0.2], rows))


def test_many_draws_and_no_probabilities(lib):
    x = torch.from_numpy(scores(2, 5000, 21)).float().cuda()
    for filters in (dict(), dict(top_k=20), dict(top_p=0.9)):
        s = {k: as_setting(v, 2, torch.int32 if k == "top_k" else torch.float32) for k, v in filters.items()}
        uniform = ((torch.arange(20_000, device="cuda") + 0.5) / 20_000).repeat(2, 1).contiguous()
        a, p, _ = call(lib, x, "f32", uniform, **s)
        b, q, _ = call(lib, x, "f32", uniform, probs=False, **s)
        assert torch.equal(a, b) and (q == 9).all()
        w = ref.kept_weights(x[1].double().cpu().numpy(), **filters)
        freq = np.bincount(a[1].cpu().numpy(), minlength=5000) / 20_000
        assert np.abs(freq - w / w.sum()).max() <= 1.01 / 20_000      # evenly spaced numbers: one more or less


def test_columns_past_32_bits_of_bytes(lib):
    """A row of 1.2e9 columns: 4.8 GB."""
    n = 1_200_000_007
    x = torch.full((1, n), -30.0, device="cuda")
    x[0, [5, 600_000_000, 1_100_000_003, n - 1]] = torch.tensor([1.0, 2.0, 3.0, 2.5], device="cuda")
    u = torch.tensor([[0.0, 0.1, 0.5, 0.9, 0.999]], device="cuda")
    for filters in (dict(top_k=3), dict(top_p=0.95), dict()):
        s = {k: as_setting(v, 1, torch.int32 if k == "top_k" else torch.float32) for k, v in filters.items()}
        labels, probs, _ = call(lib, x, "f32", u, **s)
        e = np.exp(np.array([1.0, 2.0, 3.0, 2.5]) - 3)
        if filters == dict(top_k=3) or "top_p" in filters:
            e[0] = 0 if "top_k" in filters else e[0]
        if "top_p" in filters:
            flat = (n - 4) * np.exp(-33.0)
            order = np.argsort(-e)
            upto = np.cumsum(e[order])
            e[order[int((upto < 0.95 * (e.sum() + flat)).sum()) + 1:]] = 0
        where = np.array([5, 600_000_000, 1_100_000_003, n - 1])
        got = labels[0].cpu().numpy()
        run = np.cumsum(e) / e.sum()
        want = where[np.searchsorted(run, u[0].cpu().numpy(), side="right")]
        if filters:
            assert np.array_equal(got, want)
        else:
            assert (got >= 0).all() and (got < n).all() and got[2] == 1_100_000_003


def test_captured_draws_give_what_eager_ones_do(lib):
    x = torch.from_numpy(scores(5, 40_000, 31)).bfloat16().cuda()
    u = torch.rand(5, 8, device="cuda")
    s = dict(top_k=as_setting([0, 50, 0, 3000, 1], 5, torch.int32), top_p=as_setting([0.9, 0.9, 1.0, 0.5, 1.0], 5, torch.float32))
    labels, probs = torch.zeros(5, 8, dtype=torch.int64, device="cuda"), torch.zeros(5, 8, device="cuda")
    work = workspace(lib, 5, 40_000)
    call(lib, x, "bf16", u, out=(labels, probs), work=work, **s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(lib, x, "bf16", u, out=(labels, probs), work=work, stream=torch.cuda.current_stream().cuda_stream, **s)
    for round_ in range(4):
        u.copy_(torch.rand(5, 8, device="cuda"))
        x.copy_(x.roll(77, 1))
        want = call(lib, x, "bf16", u, **s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(labels, want[0][:5]) and torch.equal(probs, want[1][:5])


def test_the_same_draws_every_time(lib):
    """Lists and histograms are filled in any order: nothing of it shows."""
    x = torch.from_numpy(scores(64, 70_000, 41, flat=0.4)).bfloat16().cuda()
    u = torch.rand(64, 16, device="cuda")
    s = dict(top_p=as_setting(0.9, 64, torch.float32))
    first = call(lib, x, "bf16", u, **s)[:2]
    for _ in range(5):
        again = call(lib, x, "bf16", u, **s)[:2]
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# More equal scores than a list holds on both sides of a cut, which lies a few columns off the border between them or on it.
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("off", [-40, -1, 0, 1, 40])
@pytest.mark.parametrize("with_count", [False, True])
def test_cuts_next_to_many_equal_scores(lib, kind, off, with_count):
    n, many = 30_000, 5000
    rng = np.random.default_rng(7)
    x = np.full((4, n), -20.0) + rng.integers(0, 4, (4, n)) / 4
    at = rng.permutation(n)
    x[:, at[:many]] = 0.0
    x[:, at[many:2 * many]] = -1.0
    x[2:, at[2 * many:2 * many + 50]] = rng.integers(1, 9, 50) / 8      # a few larger ones
    x[1, at[many:2 * many]] = -0.0078125
    x[3, at[2 * many + 60:2 * many + 70]] = -0.25
    w = np.exp(x - x.max(1, keepdims=True))
    count = 2 * many + 1000
    if with_count:
        w = -np.sort(-w, 1)[:, :count]
    # in the middle of a column's weight
    weights = np.exp(x - x.max(1, keepdims=True))
    goal = np.where(x >= 0, weights, 0).sum(1) + (off + 0.5) * np.exp((-1.0 if off >= 0 else 0.0) - x.max(1))
    settings = {"top_p": np.float32(goal / w.sum(1))}
    if with_count:
        settings["top_k"] = count
    check(lib, x, kind, draws=8, **settings)


@pytest.mark.parametrize("temperature", [0.5, 4.0, 40.0, 1e4])
@pytest.mark.parametrize("filters", [{"top_p": 0.3}, {"top_p": 0.9}, {"top_p": 0.9999}, {"top_k": 7001}, {"top_k": 7001, "top_p": 0.7}])
def test_scores_a_few_steps_of_their_type_apart(lib, temperature, filters):
    """Bins of a histogram are finer than the scores here, or the scores finer than the type next to them."""
    rng = np.random.default_rng(17)
    n = 30_000
    x = np.empty((5, n))
    x[0] = 1e8 - 8.0 * rng.integers(0, 30, n)
    x[1] = -1e8 - 8.0 * rng.integers(0, 30, n)
    x[2] = 3e30 - 2.0 ** 78 * rng.integers(0, 5, n)
    x[3] = rng.choice([1e8, 5.0, 4.0, -3e30], n)
    x[4] = rng.standard_normal(n)
    x[4, 7] = 1e8
    check(lib, x, "f32", draws=8, temperature=temperature, **filters)
