"""Draws from scores and the loss against a teacher without a GPU: the tests' own reference on hand-worked numbers, and what the
entry points refuse before they touch the device."""
import ctypes
import os

import numpy as np
import pytest

import scores_reference as ref


def test_reference_cuts_in_the_order_that_is_said():
    x = np.log([1.0, 4, 2, 4, 1, 0.5])
    w = lambda **f: (ref.kept_weights(x, **f) * 4).round(6).tolist()
    assert w() == [1, 4, 2, 4, 1, 0.5]
    assert w(top_k=1) == [0, 4, 0, 0, 0, 0] and w(top_k=4) == [1, 4, 2, 4, 0, 0]
    assert w(top_p=0.32) == [0, 4, 0, 0, 0, 0] and w(top_p=0.33) == [0, 4, 0, 4, 0, 0]
    assert w(top_p=0.8, top_k=3) == [0, 4, 0, 4, 0, 0] and w(top_p=0.81, top_k=3) == [0, 4, 2, 4, 0, 0]
    assert w(min_p=0.25) == [1, 4, 2, 4, 1, 0] and w(temperature=0) == [0, 4, 0, 0, 0, 0]
    assert w(temperature=0.5, min_p=0.25) == [0, 4, 1, 4, 0, 0]
    assert ref.kept_weights([-np.inf, np.nan]).tolist() == [0, 0]
    assert ref.kept_weights([0, np.inf, np.inf, np.nan]).tolist() == [0, 1, 1, 0]


def test_reference_of_draws():
    w = np.array([0, 1.0, 0, 3.0])
    assert ref.drawn(w, 0.0, 1, 0.25, 0) and ref.drawn(w, 0.25, 3, 0.75, 0) and ref.drawn(w, 0.2499, 1, 0.25, 0)
    assert not ref.drawn(w, 0.26, 1, 0.25, 1e-9) and not ref.drawn(w, 0.1, 0, 0, 1e-9) and ref.drawn(w, 1.0, 3, 0.75, 0)
    assert ref.drawn(np.zeros(3), 0.5, -1, 0.0, 0)


def test_reference_gradient_is_that_of_differences():
    rng = np.random.default_rng(2)
    x, labels, teacher = rng.standard_normal(12), np.array([3, 7, -1, 3, 20]), rng.standard_normal(5)
    for whole in (None, 2.0):
        _, g = ref.distil(x, labels, teacher, 1.7, whole)
        for i in range(12):
            up, down = x.copy(), x.copy()
            up[i] += 1e-5
            down[i] -= 1e-5
            slope = (ref.distil(up, labels, teacher, 1.7, whole)[0] - ref.distil(down, labels, teacher, 1.7, whole)[0]) / 2e-5
            assert abs(slope - g[i]) < 1e-8
    loss, g = ref.distil(np.log([0.5, 0.25, 0.25]), np.array([0, 1]), np.log([2.0, 1.0]), 1.0)
    assert abs(loss - (2 / 3 * np.log(4 / 3) + 1 / 3 * np.log(4 / 3))) < 1e-12 and np.allclose(g, [0.5 - 2 / 3, 0.25 - 1 / 3, 0.25])


@pytest.fixture(scope="module")
def capi():
    from indexsdk_amd import _capi
    if not os.path.exists(_capi.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    _capi.load()
    return _capi


@pytest.mark.parametrize("name", ["ixa_sample_workspace", "ixa_distil_workspace"])
def test_workspaces(capi, name):
    size, f = ctypes.c_int64(-1), getattr(capi.load(), name)
    for rows, n in ((0, 0), (0, 100), (1, 0), (1, 1), (1 << 22, 1000), (3, 0x7fffffff)):
        assert f(rows, n, ctypes.byref(size)) == 0 and 0 <= size.value < 1 << 32
    for rows, n in ((-1, 1), (1, -1), ((1 << 22) + 1, 1), (1, 1 << 31)):
        assert f(rows, n, ctypes.byref(size)) == 2001
    assert f(1, 1, None) == 2001


# Addresses are checked before anything is queued and are never read: these stand for buffers.
P, ODD, OFF, BIG = 1 << 30, (1 << 30) + 1, (1 << 30) + 8, 1 << 40


def _sample(**kw):
    a = dict(scores=P, ld=64, type=0, rows=4, n=64, temperature=P, top_k=P, top_p=P, min_p=P, uniform=P, draws=1, labels=P, probs=P,
             work=P, size=BIG)
    a.update(kw)
    return "ixa_op_sample", tuple(a.values()) + (None,)


_TASK = dict(scores=P, ld=64, type=0, rows=4, n=64, labels=P, teacher=P, k=5, whole=P, T=1.0)


def _loss(**kw):
    a = dict(_TASK, loss=P, stats=P, work=P, size=BIG)
    a.update(kw)
    return "ixa_op_distil_loss", tuple(a.values()) + (None,)


def _gradient(**kw):
    a = dict(_TASK, stats=P, weight=P, gradient=2 * P, ld_g=64)
    a.update(kw)
    return "ixa_op_distil_gradient", tuple(a.values()) + (None,)


def _step(**kw):
    a = dict(_TASK, weight=P, loss=P, gradient=2 * P, ld_g=64, work=P, size=BIG)
    a.update(kw)
    return "ixa_op_distil_step", tuple(a.values()) + (None,)


@pytest.mark.parametrize("call,needle", [
    (_sample(scores=None), "nullptr"), (_sample(uniform=None), "nullptr"), (_sample(labels=None), "nullptr"),
    (_sample(type=3), "element type"), (_sample(rows=-1), "rows"), (_sample(rows=(1 << 22) + 1), "rows"), (_sample(n=-1), "rows"),
    (_sample(n=1 << 31, ld=1 << 31), "columns"), (_sample(ld=63), "steps of"), (_sample(draws=-1), "draws"),
    (_sample(draws=(1 << 20) + 1), "draws"), (_sample(scores=ODD), "aligned"), (_sample(temperature=P + 2), "aligned"),
    (_sample(top_k=ODD), "aligned"), (_sample(top_p=ODD), "aligned"), (_sample(min_p=ODD), "aligned"), (_sample(uniform=ODD), "aligned"),
    (_sample(labels=P + 4), "aligned"), (_sample(probs=ODD), "aligned"),
    (_loss(scores=None), "nullptr"), (_loss(labels=None), "nullptr"), (_loss(teacher=None), "nullptr"), (_loss(loss=None), "nullptr"),
    (_loss(type=-1), "element type"), (_loss(rows=-1), "rows"), (_loss(n=1 << 31, ld=1 << 31), "columns"), (_loss(ld=63), "steps of"),
    (_loss(k=-1), "entries"), (_loss(k=2049), "entries"), (_loss(T=0.0), "temperature"), (_loss(T=float("nan")), "temperature"),
    (_loss(T=1e7), "temperature"), (_loss(T=-1.0), "temperature"), (_loss(labels=P + 4), "entries"), (_loss(teacher=ODD), "entries"),
    (_loss(whole=P + 2), "entries"), (_loss(loss=ODD), "aligned"), (_loss(stats=ODD), "aligned"), (_loss(scores=ODD), "aligned"),
    (_loss(work=None), "workspace"), (_loss(size=0), "workspace"), (_loss(work=OFF), "workspace"),
    (_gradient(stats=None), "nullptr"), (_gradient(gradient=None), "nullptr"), (_gradient(ld_g=63), "steps of"),
    (_gradient(stats=ODD), "aligned"), (_gradient(weight=ODD), "weights"), (_gradient(gradient=ODD), "aligned"),
    (_gradient(gradient=P, ld_g=65), "own"), (_gradient(gradient=P + 4), "own"), (_gradient(gradient=P + 256), "own"),
    (_gradient(ld=128, ld_g=128, gradient=P + 252), "own"), (_step(gradient=P + 512), "own"), (_step(gradient=P, ld_g=128), "own"),
    (_step(loss=None), "nullptr"), (_step(gradient=None), "nullptr"), (_step(T=float("inf")), "temperature"),
    (_step(work=None), "workspace"), (_step(size=16), "workspace"), (_step(k=5000), "entries"),
])
def test_entry_points_refuse(capi, call, needle):
    lib = capi.load()
    name, args = call
    assert getattr(lib, name)(*args) == 2001
    assert needle in lib.ixa_last_error().decode()


@pytest.mark.parametrize("call", [
    _sample(rows=0, scores=None, uniform=None, labels=None, probs=None, work=None, size=0), _sample(draws=0, uniform=None, labels=None),
    _loss(rows=0, scores=None, labels=None, teacher=None, loss=None, work=None, size=0),
    _gradient(rows=0, scores=None, labels=None, teacher=None, stats=None, gradient=None), _gradient(n=0, scores=None, gradient=None),
    _step(rows=0, scores=None, labels=None, teacher=None, loss=None, gradient=None, work=None, size=0),
])
def test_no_rows_need_no_buffers(capi, call):
    name, args = call
    assert getattr(capi.load(), name)(*args) == 0, capi.load().ixa_last_error().decode()


@pytest.mark.parametrize("call", [
    _sample(), _sample(temperature=None, top_k=None, top_p=None, min_p=None, probs=None), _sample(n=0, scores=None), _loss(),
    _loss(k=0, labels=None, teacher=None, whole=None, stats=None), _gradient(), _gradient(gradient=P, weight=None),
    _gradient(ld=128, ld_g=128, gradient=P + 256), _step(), _step(gradient=P), _loss(n=0, scores=None),
])
def test_no_device_is_an_error(capi, call):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these would be launched")
    name, args = call
    assert getattr(capi.load(), name)(*args) == 2016 and "no CPU path" in capi.load().ixa_last_error().decode()
