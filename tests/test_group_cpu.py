"""Rows in 4 bits with group scales without a GPU: the tests' own reference on hand-worked numbers, and what the entry points
refuse before they touch the device."""
import ctypes
import os

import numpy as np
import pytest

import group_reference as ref


def test_reference_on_worked_numbers():
    x = np.zeros((1, 64))
    x[0, :5] = [7, -7, 0.5, 1.5, 2.5]                 # scale 1: halfway points go to the even number
    x[0, 32:36] = [-3, 12, 0, 4]                       # low -3, high 12
    code, scale, zero = ref.quantise(x, 32, ref.F32, False)
    assert scale[0].tolist() == [1.0, float(np.float32(12 / 7))] and (zero == 8).all()
    assert code[0, 0, :6].tolist() == [15, 1, 8, 10, 10, 8]
    code, scale, zero = ref.quantise(x, 32, ref.F16, True)
    assert scale[0, 1] == 1 and zero[0, 1] == 3 and code[0, 1, :5].tolist() == [0, 15, 3, 7, 3]
    assert ref.values(code, scale, zero, 36)[0, 32:].tolist() == [-3, 12, 0, 4]


def test_reference_rounds_scales():
    assert ref.round_to_type(1 + 2.0 ** -8, ref.BF16) == 1 and ref.round_to_type(1 + 3 * 2.0 ** -8, ref.BF16) == 1 + 2.0 ** -6
    assert ref.round_to_type(2.0 ** -25, ref.F16) == 0 and ref.round_to_type(1 + 2.0 ** -11, ref.F16) == 1


def test_reference_of_bytes_is_its_own_inverse():
    raw = np.random.default_rng(3).integers(0, 256, (5, 48), dtype=np.uint8)
    assert np.array_equal(ref.pack(ref.unpack(raw, 32)), raw)


@pytest.fixture(scope="module")
def capi():
    from indexsdk_amd import _capi
    if not os.path.exists(_capi.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    _capi.load()
    return _capi


def test_group_bytes(capi):
    lib = capi.load()
    for group, d, want in ((32, 200, (112, 7)), (64, 200, (128, 4)), (128, 200, (128, 2)), (128, 1, (64, 1)), (32, 16384, (8192, 512))):
        a, b = ctypes.c_int64(), ctypes.c_int64()
        assert lib.ixa_group_bytes(group, d, ctypes.byref(a), ctypes.byref(b)) == 0 and (a.value, b.value) == want
    assert lib.ixa_group_bytes(32, 32, None, None) == 0
    for group, d in ((16, 32), (0, 32), (32, 0), (64, 16385)):
        assert lib.ixa_group_bytes(group, d, None, None) == 2001 and "group_bytes" in lib.ixa_last_error().decode()


def test_product_workspace(capi):
    lib, size = capi.load(), ctypes.c_int64(-1)
    for kind, m, d, least in ((0, 0, 100, 0), (1, 1, 128, 0), (0, 100, 200, 100 * 2 * 256 * 2), (2, 100, 200, 100 * 256 * 2),
                              (1, 64, 16384, 64 * 16384 * 2)):
        assert lib.ixa_group_product_workspace(kind, m, d, ctypes.byref(size)) == 0
        assert size.value >= least and (size.value > 0) == (least > 0)
    for kind, m, d in ((3, 1, 1), (0, -1, 1), (0, (1 << 23) + 1, 1), (0, 1, 0), (0, 1, 16385)):
        assert lib.ixa_group_product_workspace(kind, m, d, ctypes.byref(size)) == 2001
    assert lib.ixa_group_product_workspace(0, 1, 1, None) == 2001


# Addresses are checked before anything is queued and are never read: these stand for buffers.
P, ODD, OFF = 1 << 20, (1 << 20) + 1, (1 << 20) + 8


def _quantise(**kw):
    a = dict(x=P, ld=64, type=0, n=4, d=64, group=32, scale=1, codes=P, scales=P, zeros=None)
    a.update(kw)
    return "ixa_op_group_quantise", tuple(a.values()) + (None,)


def _dequantise(**kw):
    a = dict(codes=P, scales=P, zeros=None, group=32, scale=1, n=4, d=64, type=0, out=P, ld=64)
    a.update(kw)
    return "ixa_op_group_dequantise", tuple(a.values()) + (None,)


def _product(**kw):
    a = dict(x=P, ld_x=64, type=0, m=4, codes=P, scales=P, zeros=P, group=32, scale=1, n=4, d=64, alpha=1.0, bias=None, out_type=0,
             out=P, ld=4, work=None, size=0)
    a.update(kw)
    return "ixa_op_group_product", tuple(a.values()) + (None,)


@pytest.mark.parametrize("call,needle", [
    (_quantise(x=None), "nullptr"), (_quantise(codes=None), "nullptr"), (_quantise(scales=None), "nullptr"),
    (_quantise(type=3), "element type"), (_quantise(scale=-1), "element type"), (_quantise(group=48), "groups of"),
    (_quantise(d=0), "dims"), (_quantise(d=16385, ld=16385), "dims"), (_quantise(n=-1), "rows"), (_quantise(n=1 << 31), "rows"),
    (_quantise(ld=63), "steps of"), (_quantise(x=ODD), "aligned"), (_quantise(codes=OFF), "16 bytes"),
    (_quantise(scales=ODD), "scales on"), (_quantise(scale=0, scales=P + 2), "scales on"),
    (_dequantise(out=None), "nullptr"), (_dequantise(codes=None), "nullptr"), (_dequantise(type=9), "element type"),
    (_dequantise(group=256), "groups of"), (_dequantise(ld=63), "steps of"), (_dequantise(out=ODD), "aligned"),
    (_product(x=None), "nullptr"), (_product(codes=None), "nullptr"), (_product(out=None), "nullptr"),
    (_product(type=5), "element type"), (_product(out_type=5), "element type"), (_product(scale=5), "element type"),
    (_product(group=0), "groups of"), (_product(m=-1), "rows"), (_product(m=(1 << 23) + 1), "rows"), (_product(n=-1, ld=0), "rows"),
    (_product(n=1 << 31, ld=1 << 31), "rows"), (_product(d=16385, ld_x=16385), "dims"), (_product(ld_x=63), "steps of"),
    (_product(ld=3), "steps of"), (_product(alpha=float("inf")), "alpha"), (_product(alpha=float("nan")), "alpha"),
    (_product(bias=P + 2), "biases"), (_product(out=ODD), "aligned"), (_product(x=ODD), "aligned"),
    (_product(m=65), "workspace"), (_product(m=65, work=P, size=100), "workspace"), (_product(m=65, work=OFF, size=1 << 20), "workspace"),
])
def test_entry_points_refuse(capi, call, needle):
    lib = capi.load()
    name, args = call
    assert getattr(lib, name)(*args) == 2001
    assert needle in lib.ixa_last_error().decode()


@pytest.mark.parametrize("call", [
    _quantise(n=0, x=None, codes=None, scales=None), _dequantise(n=0, codes=None, scales=None, out=None),
    _product(m=0, x=None, codes=None, scales=None, zeros=None, out=None), _product(n=0, ld=0, codes=None, scales=None, out=None),
    _product(m=0), _product(n=0, m=100, ld=0),
])
def test_no_rows_need_no_buffers(capi, call):
    name, args = call
    assert getattr(capi.load(), name)(*args) == 0, capi.load().ixa_last_error().decode()


def test_no_device_is_an_error(capi):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for name, args in (_quantise(), _dequantise(), _product(), _product(m=65, work=P, size=1 << 20)):
        assert getattr(capi.load(), name)(*args) == 2016 and "no CPU path" in capi.load().ixa_last_error().decode()
