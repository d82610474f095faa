"""GPU tests of 4-bit rows with group scales, draws and distillation as they are used together: a store in 4 bits scored against hidden
states, a teacher's lists from unrounded rows by the top-k operator, a training step of the hidden states, and draws from what
they then score; eagerly, on a stream of their own and as a captured graph."""
import ctypes

import numpy as np
import pytest

import group_reference as gref
import scores_reference as sref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

N, D, M, K, T, GROUP = 4099, 200, 37, 24, 2.0, 64
U = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    from indexsdk_amd import _capi
    return _capi.load(), _capi.check


def at(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def product_bound(x, values):
    """What a product in 32 bits is off by: 64 additions of a group's products, one multiply-add per group, and the last rounding, each
    of them U of a sum of magnitudes; and what lies 2^-39 below the largest element of x."""
    return 70 * U * (np.abs(x) @ np.abs(values.T)) + 2.0 ** -39 * np.abs(x).max(1, keepdims=True) * np.abs(values).sum(1)


class Run:
    """Everything between hidden states and drawn labels, in buffers of its own."""

    def __init__(self, lib, table, hidden, seed):
        self.lib, self.check = lib
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.table, self.hidden = table, hidden
        empty = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="cuda")
        per_row, groups = ctypes.c_int64(), ctypes.c_int64()
        self.check(self.lib.ixa_group_bytes(GROUP, D, ctypes.byref(per_row), ctypes.byref(groups)))
        self.codes, self.scales = empty(N, per_row.value, dtype=torch.uint8), empty(N, groups.value, dtype=torch.float16)
        self.zeros = empty(N, groups.value, dtype=torch.uint8)
        self.scores, self.exact = empty(M, N), empty(M, N)
        self.near, self.labels = empty(M, K), empty(M, K, dtype=torch.int64)
        self.teacher = empty(M, K)
        self.loss, self.gradient, self.drawn = empty(M), empty(M, N), empty(M, 3, dtype=torch.int64)
        self.probs, self.uniform = empty(M, 3), torch.rand(M, 3, device="cuda", generator=gen)
        self.top_p, self.top_k = torch.full((M,), 0.9, device="cuda"), torch.full((M,), 300, device="cuda", dtype=torch.int32)
        self.work = {}
        for name, args in (("ixa_group_product_workspace", (2, M, D)), ("ixa_distil_workspace", (M, N)), ("ixa_sample_workspace", (M, N))):
            size = ctypes.c_int64()
            self.check(getattr(self.lib, name)(*args, ctypes.byref(size)))
            self.work[name] = torch.empty(max(size.value, 16), dtype=torch.uint8, device="cuda"), size.value

    def fill(self, stream):
        self.check(self.lib.ixa_op_group_quantise(at(self.table), D, 0, N, D, GROUP, 1, at(self.codes), at(self.scales),
                                                  at(self.zeros), stream))

    def step(self, stream):
        """Scores, the teacher's list, loss and gradient, draws; nothing but the entry points."""
        work = lambda name: (at(self.work[name][0]), self.work[name][1])
        self.check(self.lib.ixa_op_group_product(at(self.hidden), D, 2, M, at(self.codes), at(self.scales), at(self.zeros), GROUP, 1,
                                                 N, D, 1.0, None, 0, at(self.scores), N, *work("ixa_group_product_workspace"), stream))
        # the teacher's best: the smallest of the negated scores
        self.check(self.lib.ixa_op_topk_flat_fp32(at(self.exact), M, N, N, K, 1, at(self.near), at(self.labels), stream))
        self.teacher.copy_(-self.near)
        self.check(self.lib.ixa_op_distil_step(at(self.scores), N, 0, M, N, at(self.labels), at(self.teacher), K, None, T, None,
                                               at(self.loss), at(self.gradient), N, *work("ixa_distil_workspace"), stream))
        self.check(self.lib.ixa_op_sample(at(self.scores), N, 0, M, N, None, at(self.top_k), at(self.top_p), None, at(self.uniform),
                                          3, at(self.drawn), at(self.probs), *work("ixa_sample_workspace"), stream))

    def results(self):
        return [t.clone() for t in (self.scores, self.labels, self.loss, self.gradient, self.drawn, self.probs)]


@pytest.fixture(scope="module")
def inputs():
    rng = np.random.default_rng(11)
    table = torch.from_numpy(rng.standard_normal((N, D)).astype(np.float32)).cuda()
    hidden = torch.from_numpy(rng.standard_normal((M, D)) * 0.2).cuda().to(torch.bfloat16)
    return table, hidden


def prepared(lib, inputs, seed=0):
    run = Run(lib, inputs[0], inputs[1].clone(), seed)
    run.exact.copy_(-(inputs[1].double() @ inputs[0].double().T).float())
    run.fill(None)
    torch.cuda.synchronize()
    return run


def test_from_rows_to_draws(lib, inputs):
    run = prepared(lib, inputs)
    run.step(None)
    torch.cuda.synchronize()
    as64 = lambda t: t.double().cpu().numpy()
    # the store and its scores
    values = gref.values(*gref.quantise(as64(run.table), GROUP, gref.F16, True), D)
    x, scores = as64(run.hidden), as64(run.scores)
    assert (np.abs(scores - x @ values.T) <= product_bound(x, values)).all()
    # the teacher's lists are the best of its scores
    order = np.argsort(as64(run.exact), axis=1, kind="stable")[:, :K]
    assert np.array_equal(order, run.labels.cpu().numpy())
    for r in range(M):
        loss, gradient = sref.distil(scores[r], order[r], as64(run.teacher)[r], T)
        # a logarithm of a sum of 32-bit exponentials: 36 units and those of the arguments (31 of 0.7), as for the loss by itself
        off = 60 * U
        assert abs(as64(run.loss)[r] - loss) <= T * T * off + 2 * U * abs(loss) + 1e-12
        q = np.exp((scores[r] - scores[r].max()) / T)
        q /= q.sum()
        t = np.abs(scores[r] - scores[r].max()) / T * 1.4427
        bound = T * q * (off + 8 * U + 0.7 * U * t) + 5 * U * np.abs(gradient) + 2.0 ** -120
        bound[order[r]] += T * 2 * U
        assert (np.abs(as64(run.gradient)[r] - gradient) <= bound).all()
        w = sref.kept_weights(scores[r], top_k=300, top_p=float(np.float32(0.9)))
        for d in range(3):
            assert sref.drawn(w, run.uniform[r, d].item(), run.drawn[r, d].item(), run.probs[r, d].item(), 2e-13)


def test_the_gradient_of_the_hidden_states(lib, inputs):
    """It is the scores' gradient times the store's values: a difference of the loss along it, over scores in 64 bits."""
    run = prepared(lib, inputs)
    run.step(None)
    torch.cuda.synchronize()
    as64 = lambda t: t.double().cpu().numpy()
    values, x = gref.values(*gref.quantise(as64(run.table), GROUP, gref.F16, True), D), as64(run.hidden)
    labels, teacher = run.labels.cpu().numpy(), as64(run.teacher)
    gradient = as64(run.gradient) @ values
    row = np.sqrt((values ** 2).sum(1)).max()
    h = 1e-5
    for r in range(0, M, 9):
        loss = lambda s: sref.distil((x[r] + s * gradient[r]) @ values.T, labels[r], teacher[r], T)[0]
        slope, square = (loss(h) - loss(-h)) / (2 * h), (gradient[r] ** 2).sum()
        # The third derivative along the step is T^2 times a third central moment of the scores' change over T, |change| <= move; the loss is
        # a number of 64 bits below 100.
        move = np.abs(values @ gradient[r]).max()
        bound = h * h / 6 * T * T * (2 * move / T) ** 3 + 1e-12 / h
        # The scores' gradient is that of scores off by `off`: q by 2 off / T of itself, by the bound of its own kernel, and the sum over the
        # columns, T in all, times no more than a row of the store.
        off = product_bound(x[r:r + 1], values).max()
        bound += np.sqrt(square) * row * T * (2 * off / T + 140 * U)
        assert abs(slope - square) <= bound, (r, slope, square, bound)


def test_on_another_stream_and_as_a_graph(lib, inputs):
    run, other = prepared(lib, inputs), prepared(lib, inputs)
    run.step(None)
    torch.cuda.synchronize()
    want = run.results()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other.step(ctypes.c_void_p(stream.cuda_stream))
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other.results()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    for turn in range(3):
        for r in (run, other):
            r.hidden.copy_(inputs[1].roll(turn, 0))
            r.uniform.copy_(run.uniform.roll(turn, 1) if r is run else run.uniform)
        run.step(None)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run.results(), other.results())), turn


def test_two_at_once(lib, inputs):
    """Two runs on two streams, with workspaces of their own, do not disturb each other."""
    runs = [prepared(lib, inputs, seed) for seed in (1, 2)]
    want = []
    for r in runs:
        r.step(None)
        torch.cuda.synchronize()
        want.append(r.results())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for r, s in zip(runs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                r.step(ctypes.c_void_p(s.cuda_stream))
    torch.cuda.synchronize()
    for r, w in zip(runs, want):
        assert all(torch.equal(a, b) for a, b in zip(r.results(), w))
