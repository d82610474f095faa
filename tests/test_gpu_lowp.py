"""GPU tests of the low-precision operators against their definitions in 64 bits (tests/lowp_reference.py): codes and scales bit
for bit where the arithmetic is exact, the norm's within the error of its sums, products within that of 32-bit sums."""
import ctypes

import numpy as np
import pytest

import lowp_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
INT8, MXFP8, MXFP4 = ref.INT8, ref.MXFP8, ref.MXFP4
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
    view.copy_(torch.from_numpy(x).to(dtype))
    return view


def as64(t):
    return t.detach().cpu().double().numpy()


class Codes:
    """Buffers for n rows of codes with guard bytes behind them."""

    def __init__(self, n, d, fmt, sqr=True):
        self.n, self.d, self.fmt = n, d, fmt
        nb = ref.blocks_of(d)
        self.row = d if fmt == INT8 else nb * (32 if fmt == MXFP8 else 16)
        self.per = 4 if fmt == INT8 else nb
        self.codes = torch.full((n * self.row + 64,), GUARD, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((n * self.per + 64,), GUARD, dtype=torch.uint8, device="cuda")
        self.sqr = torch.full((n + 16,), 7.0, device="cuda") if sqr else None

    def get(self):
        torch.cuda.synchronize()
        c, s = self.codes.cpu().numpy(), self.scales.cpu().numpy()
        assert (c[self.n * self.row:] == GUARD).all() and (s[self.n * self.per:] == GUARD).all()
        if self.sqr is not None:
            assert (self.sqr[self.n:].cpu().numpy() == 7).all()
        c, s = c[:self.n * self.row].reshape(self.n, self.row), s[:self.n * self.per].reshape(self.n, self.per)
        if self.fmt == INT8:
            return c.view(np.int8), s.copy().view(np.float32)[:, 0], None if self.sqr is None else as64(self.sqr[:self.n])
        return c, s, None if self.sqr is None else as64(self.sqr[:self.n])


def quantise(lib, x, kind, fmt, fixed=0.0, sqr=True, stream=None):
    n, d = x.shape
    out = Codes(n, d, fmt, sqr)
    lib[1](lib[0].ixa_op_quantise(at(x), x.stride(0), TYPES[kind][0], n, d, fmt, fixed, at(out.codes), at(out.scales),
                                  at(out.sqr), ctypes.c_void_p(stream)))
    return out


def sample(n, d, seed, spread=0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, d)).astype(np.float32)
    return x * np.exp2(rng.integers(-spread, spread + 1, (n, 1))).astype(np.float32) if spread else x


def check_codes(x64, x32, fmt, got, fixed=0.0):
    """codes, scales and squared norms of quantised rows: the first two bit for bit"""
    codes, scales, sqr = got
    n, d = x64.shape
    if fmt == INT8:
        want, want_s = ref.int8_codes(x32, fixed)
        assert np.array_equal(scales.view(np.uint32) | (np.isnan(scales) * 0xffffffff).astype(np.uint32),
                              want_s.view(np.uint32) | (np.isnan(want_s) * 0xffffffff).astype(np.uint32))
        assert np.array_equal(codes, want)
        v = want.astype(np.float64) * want_s.astype(np.float64)[:, None]
    else:
        code, want_s = ref.mx_codes(x64, fmt)
        assert np.array_equal(scales, want_s)
        assert np.array_equal(codes, ref.pack(code, fmt))
        v = ref.mx_values(codes, scales, fmt)
    if sqr is not None:
        with np.errstate(invalid="ignore", over="ignore"):
            s = (v ** 2).sum(-1)
        ok = np.isfinite(s) & (s < 3e38) & (s > 1e-30)
        assert np.isnan(sqr[np.isnan(s)]).all()
        assert (np.abs(sqr[ok] - s[ok]) <= (d + 8) * U * s[ok]).all()


# ----- codes of rows ----------------------------------------------------------------------------------------------------

# both sides of every line between the kernels' shapes (128, 256, 512, 1024, 2048, 4096, 8192), blocks that end early, one element
DIMS = [1, 8, 31, 32, 33, 96, 128, 129, 200, 256, 257, 512, 520, 768, 1000, 1024, 1030, 2048, 2056, 4096, 4100, 8192, 8200, 16384]


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_quantise(lib, d, fmt):
    for k, (kind, n, pad, shift) in enumerate([("f32", 37, 0, 0), ("f16", 5, 3, 0), ("bf16", 18, 8, 0), ("f32", 1, 0, 1),
                                               ("bf16", 3, 0, 3)]):
        x = rows(sample(n, d, d * 7 + k, spread=12 if kind != "f16" else 3), kind, pad, shift)
        check_codes(as64(x), x.float().cpu().numpy(), fmt, quantise(lib, x, kind, fmt).get())


@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_quantise_of_one_and_of_many_rows(lib, fmt):
    for n in (1, 2, 15, 16, 17, 1000):
        x = rows(sample(n, 40, n), "f32")
        check_codes(as64(x), x.cpu().numpy(), fmt, quantise(lib, x, "f32", fmt).get())


def special_rows():
    """Zeros, negative zeros, subnormals, the largest numbers, powers of two and their neighbours, halfway numbers, infinities and
    NaN, each in a block of its own and one to a row."""
    f = np.float32
    half = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 0.2499, 0.2501] * 3)[:32]
    out = [np.zeros(96), -np.zeros(96), np.full(96, 1e-45), np.full(96, 3.4028234e38), np.full(96, 2.0 ** -126),
           np.full(96, 2.0 ** -125), np.full(96, 1.1754942e-38), np.tile(half, 3), -np.tile(half, 3) * 2.0 ** 100,
           np.tile(half, 3) * 2.0 ** -124]
    for p in (-3, 0, 5):
        v = np.full(96, 0.1 * 2.0 ** p)
        v[0], v[32], v[64] = 2.0 ** p, np.nextafter(f(2.0 ** p), f(0)), np.nextafter(f(2.0 ** p), f(1e9))
        out.append(v)
    for bad in (np.inf, -np.inf, np.nan):
        v = np.linspace(-1, 1, 96)
        v[40] = bad
        out.append(v)
    tiny = np.linspace(-1, 1, 96) * 1e-37
    return np.array(out + [tiny, tiny * 1e-4], dtype=np.float32)


@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_quantise_of_special_numbers(lib, fmt):
    x = special_rows()
    with np.errstate(over="ignore"):
        for kind in ("f32", "bf16"):
            t = rows(x, kind)
            check_codes(as64(t), t.float().cpu().numpy(), fmt, quantise(lib, t, kind, fmt).get())


def test_quantise_every_16_bit_number(lib):
    """Every finite float16 number next to a 1.0 that fixes the block's scale, and every bfloat16 number in blocks by exponent."""
    h = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.float16)
    h = h[torch.isfinite(h) & (h.abs() <= 6)]
    h = h[:h.numel() // 31 * 31].view(-1, 31)
    x = torch.cat([torch.ones(len(h), 1, dtype=torch.float16), h], 1).cuda()
    b = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 32).cuda()
    for fmt in (MXFP4, MXFP8):
        check_codes(as64(x), None, fmt, quantise(lib, x, "f16", fmt, sqr=False).get())
        check_codes(as64(b), None, fmt, quantise(lib, b, "bf16", fmt, sqr=False).get())


@pytest.mark.parametrize("d", [7, 8, 128, 1000])
def test_quantise_with_a_fixed_scale(lib, d):
    x = sample(21, d, d) * 3
    x[3, 0], x[4, d // 2], x[5, d - 1] = np.inf, -np.inf, np.nan
    t = rows(x, "f32", 5)
    for scale in (0.02, 1.0, 1e-30):
        got = quantise(lib, t, "f32", INT8, fixed=scale)
        check_codes(as64(t), t.cpu().numpy(), INT8, got.get(), np.float32(scale))
    # the scales may be left out
    out = Codes(21, d, INT8, sqr=False)
    lib[1](lib[0].ixa_op_quantise(at(t), t.stride(0), 0, 21, d, INT8, 0.02, at(out.codes), None, None, None))
    torch.cuda.synchronize()
    assert np.array_equal(out.codes[:21 * d].cpu().numpy().view(np.int8).reshape(21, d), ref.int8_codes(t.cpu().numpy(), 0.02)[0])


# ----- codes back into values ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [1, 15, 16, 17, 32, 48, 64, 100, 200, 768, 1000, 4096, 5000])
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_dequantise(lib, d, fmt):
    rng = np.random.default_rng(d)
    for n, kind, pad in ((1, "f32", 0), (29, "bf16", 0), (13, "f16", 5), (300, "f32", 8)):
        c = Codes(n, d, fmt, sqr=False)
        raw = torch.from_numpy(rng.integers(0, 256, c.codes.numel(), dtype=np.uint8))
        c.codes.copy_(raw)
        if fmt == INT8:
            s = rng.standard_normal(n).astype(np.float32)
            s[0] = np.nan if n > 1 else s[0]
            scales = torch.from_numpy(s).cuda()
            v = raw[:n * d].numpy().view(np.int8).reshape(n, d).astype(np.float32) * s[:, None]
        else:
            nb = ref.blocks_of(d)
            s = rng.integers(0 if kind == "f32" else 110, 250 if kind == "f32" else 136, (n, nb)).astype(np.uint8)
            if n > 1:
                s[1, nb - 1] = 255
            scales = torch.from_numpy(s).cuda()
            v = ref.mx_values(raw[:n * c.row].numpy().reshape(n, c.row), s, fmt)[:, :d]
        want = torch.from_numpy(v).to(torch.float32).to(TYPES[kind][1])
        store = torch.full((n, d + pad), 9.0, dtype=TYPES[kind][1], device="cuda")
        lib[1](lib[0].ixa_op_dequantise(at(c.codes), at(scales), fmt, n, d, TYPES[kind][0], at(store), d + pad, None))
        torch.cuda.synchronize()
        got = store.cpu()
        assert (got[:, d:] == 9).all()
        got = got[:, :d].float().numpy()
        w = want.float().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(got[~np.isnan(w)], w[~np.isnan(w)])


# ----- root-mean-square norm ----------------------------------------------------------------------------------------------

def norm(lib, x, res, w, kind, fmt, eps=1e-6, fixed=0.0, keep_sum=True, sqr=True):
    n, d = x.shape
    out = Codes(n, d, fmt, sqr)
    total = torch.full((n, d + 5), 9.0, dtype=x.dtype, device="cuda") if keep_sum else None
    lib[1](lib[0].ixa_op_rms_norm_quantise(at(x), x.stride(0), at(res), res.stride(0) if res is not None else 0, at(w),
                                           TYPES[kind][0], n, d, eps, at(total), d + 5 if keep_sum else 0, fmt, fixed,
                                           at(out.codes), at(out.scales), at(out.sqr), None))
    torch.cuda.synchronize()
    if keep_sum:
        assert (total[:, d:] == 9).all()
    return out.get(), None if total is None else total[:, :d]


def check_norm(y, got, fmt):
    """The codes are those of y to within the error of a sum of d squares and four roundings in 32 bits."""
    codes, scales, sqr = got
    n, d = y.shape
    delta = (d + 16) * U
    if fmt == INT8:
        top = np.abs(y).max(-1)
        assert (np.abs(scales - top / 127) <= 2 * delta * top / 127).all()
        # in steps of the row's scale: off by half a step and what the sums lose of up to 127 steps
        assert (np.abs(codes - y / np.where(top > 0, top / 127, 1)[:, None]) <= 0.5 + 127 * 3 * delta).all()
        v = codes * scales[:, None]
    else:
        v = ref.mx_values(codes, scales, fmt)[:, :d]

        def quantised(z):
            c, s = ref.mx_codes(z, fmt)
            return ref.mx_values(ref.pack(c, fmt), s, fmt)[:, :d]
        assert ref.between(v, y, delta, quantised).all()
    if sqr is not None:
        s = (v ** 2).sum(-1)
        assert (np.abs(sqr - s) <= (d + 8) * U * s).all()


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_rms_norm(lib, d, fmt):
    for k, (kind, n, pad, residual, weight) in enumerate([("bf16", 19, 0, True, True), ("f16", 4, 3, False, True),
                                                          ("f32", 33, 8, True, False), ("f32", 1, 0, True, True)]):
        x = sample(n, d, d + k) * (1 + 20 * (np.arange(d) % 97 == 5)).astype(np.float32)
        x = rows(x, kind, pad)
        res = rows(sample(n, d, d + k + 50), kind, 1) if residual else None
        w = rows(np.abs(sample(1, d, d + k + 99)) + np.float32(0.5), kind)[0] if weight else None
        got, total = norm(lib, x, res, w, kind, fmt)
        h = x.float() + (res.float() if residual else 0)
        assert torch.equal(total, h.to(x.dtype))        # one rounding of the 32-bit sum
        check_norm(ref.rms_norm(as64(h), None, None if w is None else as64(w), np.float32(1e-6)), got, fmt)


@pytest.mark.parametrize("fmt", [MXFP8, MXFP4])
def test_rms_norm_gives_the_codes_of_the_result_in_64_bits(lib, fmt):
    """1.5 million values whose only error before the last rounding is that of eight squares added in 32 bits, 2^-29 of a value
    over a row's 96 sums: with halfway points 2^-3 of a value apart, one in 2^25 may fall to the other side, here none or one."""
    n, d = 2000, 768
    x, res = rows(sample(n, d, 1) * np.float32(3), "bf16"), rows(sample(n, d, 2), "bf16")
    w = rows(np.abs(sample(1, d, 3)) + np.float32(0.5), "bf16")[0]
    (codes, scales, _), _ = norm(lib, x, res, w, "bf16", fmt)
    want, s = ref.mx_codes(ref.rms_norm(as64(x), as64(res), as64(w), 1e-6), fmt)
    got = ref.mx_values(codes, scales, fmt)[:, :d]
    assert (got != ref.mx_values(ref.pack(want, fmt), s, fmt)[:, :d]).sum() <= 1


@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_rms_norm_of_rows_at_the_ends(lib, fmt):
    """A row of zeros, rows whose squares overflow or vanish in 32 bits, one element that dwarfs the others."""
    d = 200
    x = sample(6, d, 1)
    x[0] = 0
    x[1] *= np.float32(1e25)
    x[2] *= np.float32(1e-30)
    x[3, 7] = 1e15
    x[4] = np.float32(3e38)
    t = rows(x, "f32")
    got, _ = norm(lib, t, None, None, "f32", fmt, keep_sum=False)
    codes, scales, sqr = got
    assert not codes[0].any() and sqr[0] == 0
    y = ref.rms_norm(x, None, None, np.float32(1e-6))
    keep = [1, 3, 4, 5]
    check_norm(y[keep], (codes[keep], scales[keep], sqr[keep]), fmt)
    tiny = codes[2:3] * scales[2:3, None] if fmt == INT8 else ref.mx_values(codes[2:3], scales[2:3], fmt)[:, :d]
    assert np.allclose(tiny, y[2:3], rtol=0.13 if fmt == MXFP8 else 0.6, atol=np.abs(y[2]).max() / (200 if fmt != MXFP4 else 6))


@pytest.mark.parametrize("fmt", [INT8, MXFP8, MXFP4])
def test_rms_norm_of_rows_that_are_not_finite(lib, fmt):
    d = 96
    x = sample(4, d, 2)
    x[0, 3], x[1, 50] = np.inf, np.nan
    got, _ = norm(lib, rows(x, "f32"), None, None, "f32", fmt, keep_sum=False)
    codes, scales, sqr = got
    if fmt == INT8:
        assert np.isnan(scales[:2]).all() and not codes[:2].any() and np.isfinite(scales[2:]).all()
    else:
        assert scales[0, 0] == 255 and (scales[0, 1:] == 0).all()      # finite elements over an infinite norm are 0
        assert (scales[1] == 255).all() and (scales[2:] < 255).all()
        zeros = 0x77 if fmt == MXFP4 else 0x7f                          # of either sign
        assert not (codes[0] & zeros).any() and not codes[1].any()
    assert np.isnan(sqr[:2]).all() and np.isfinite(sqr[2:]).all()


def test_rms_norm_writes_its_sum_over_an_input(lib):
    for d in (100, 768, 5000):
        x = rows(sample(9, d, 3), "bf16")
        res = rows(sample(9, d, 4), "bf16")
        want = (x.float() + res.float()).bfloat16()
        first, _ = norm(lib, x, res, None, "bf16", INT8)
        out = Codes(9, d, INT8, sqr=False)
        lib[1](lib[0].ixa_op_rms_norm_quantise(at(x), d, at(res), d, None, 2, 9, d, 1e-6, at(res), d, INT8, 0.0, at(out.codes),
                                               at(out.scales), None, None))
        torch.cuda.synchronize()
        assert torch.equal(res, want) and np.array_equal(out.get()[0], first[0])


def test_rms_norm_with_a_fixed_scale_fills_the_int8_index(lib):
    """Normalised rows under one scale are comparable: the exact int8 index finds the nearest of them."""
    import indexsdk_amd as ix
    n, d = 500, 64
    x, w = sample(n, d, 8), None
    t = rows(x, "f32")
    (codes, scales, _), _ = norm(lib, t, None, w, "f32", INT8, fixed=0.03, keep_sum=False)
    assert (scales == np.float32(0.03)).all()
    y = ref.rms_norm(x, None, None, np.float32(1e-6))
    step = (d + 16) * U * np.abs(y) / 0.03
    assert (np.abs(codes - np.clip(y / np.float32(0.03), -127, 127)) <= 0.5 + step).all()
    index = ix.AscendIndexInt8Flat(d)
    index.add(codes)
    _, labels = index.search_int32(codes[:20], 1)
    assert np.array_equal(labels[:, 0], np.arange(20))


# ----- product ------------------------------------------------------------------------------------------------------------

def random_codes(n, d, fmt, rng, wild):
    """Packed codes and scales: quantised Gaussians, or (wild) every number and scales of many sizes."""
    nb = ref.blocks_of(d)
    if not wild:
        return (lambda c, s: (ref.pack(c, fmt), s))(*ref.mx_codes(rng.standard_normal((n, d)), fmt))
    raw = rng.integers(0, 256, (n, nb * (32 if fmt == MXFP8 else 16)), dtype=np.uint8)
    if fmt == MXFP8:
        raw[(raw & 127) == 127] ^= 1
    per = unpacked = ref.unpack(raw, fmt).reshape(n, -1)
    per[:, d:] = 0                      # what lies behind the last column is zero, as the quantiser writes it
    return ref.pack(unpacked.reshape(n, nb, 32), fmt), rng.integers(115, 140, (n, nb)).astype(np.uint8)


def product(lib, a, a_fmt, b, d, metric, norms, out, ld, stream=None):
    lib[1](lib[0].ixa_op_mx_product(at(a[0]), at(a[1]), a_fmt, a[0].shape[0], at(b[0]), at(b[1]), b[0].shape[0], d, metric,
                                    at(norms[0]), at(norms[1]), {v[1]: v[0] for v in TYPES.values()}[out.dtype], at(out), ld,
                                    ctypes.c_void_p(stream)))


def check_product(lib, m, n, d, a_fmt, metric, kind, wild, pad=0, seed=0):
    rng = np.random.default_rng(seed + m * 31 + n * 7 + d)
    ac, asc = random_codes(m, d, a_fmt, rng, wild)
    bc, bs = random_codes(n, d, MXFP4, rng, wild)
    va, vb = ref.mx_values(ac, asc, a_fmt), ref.mx_values(bc, bs, MXFP4)
    if kind == "f16" and wild:      # scores that the type holds
        asc = (asc - 18).astype(np.uint8)
        va = ref.mx_values(ac, asc, a_fmt)
    norms = ((va ** 2).sum(-1).astype(np.float32), (vb ** 2).sum(-1).astype(np.float32))
    a, b = [torch.from_numpy(t).cuda() for t in (ac, asc)], [torch.from_numpy(t).cuda() for t in (bc, bs)]
    dn = [torch.from_numpy(t).cuda() for t in norms] if metric else (None, None)
    dtype = TYPES[kind][1]
    out = torch.full((m + 1, n + pad), 9.0, dtype=dtype, device="cuda")
    product(lib, a, a_fmt, b, d, metric, dn, out, n + pad)
    torch.cuda.synchronize()
    got = as64(out)
    assert (got[m] == 9).all() and (got[:, n:] == 9).all()
    got = got[:m, :n]
    g, mag = va @ vb.T, np.abs(va) @ np.abs(vb).T
    # each addition to the 32-bit sum may lose a unit of its last place: one or two of them per 64 columns, and the joining of
    # eight partial sums at most
    adds = 2 * ((ref.blocks_of(d) + 1) // 2) + 8
    bound = adds * 2 * U * mag
    if metric:
        s = norms[0].astype(np.float64)[:, None] + norms[1].astype(np.float64)[None, :]
        g = s - 2 * g
        bound = 2 * bound + 3 * U * (s + 2 * mag)
    least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[kind]
    bound = bound * 1.01 + {"f32": 0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind] * np.abs(g) + least
    if kind == "f16":
        beyond = np.abs(g) - bound > 65520       # rounds to infinity
        assert (got[beyond] == np.sign(g[beyond]) * np.inf).all()
        fits = np.abs(g) + bound < 65520
        g, got, bound = g[fits], got[fits], bound[fits]
    assert (np.abs(got - g) <= bound).all()


SHAPES = [(1, 1, 1), (1, 33, 32), (2, 31, 33), (31, 64, 64), (32, 32, 65), (33, 100, 96), (7, 1000, 128), (64, 257, 200),
          (65, 300, 256), (100, 129, 257), (127, 513, 288), (128, 256, 300), (129, 1025, 512), (200, 255, 520), (16, 4097, 768),
          (256, 512, 1000), (257, 700, 1030), (300, 1300, 64), (40, 600, 4096), (130, 300, 2080), (5, 70, 16384),
          (520, 770, 16), (1000, 1024, 160),
          # whole groups of 512 columns, tiles of 256 by 256 and their edges
          (256, 256, 512), (256, 1, 500), (300, 700, 2048), (513, 260, 1024), (1030, 2100, 1536), (257, 515, 4096),
          (1000, 16400, 512), (1024, 16384, 500), (250, 65600, 510), (2000, 4096, 2048), (490, 16640, 4096)]


@pytest.mark.parametrize("m,n,d", SHAPES)
@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
def test_product(lib, m, n, d, a_fmt):
    check_product(lib, m, n, d, a_fmt, 1, "f32", wild=False)
    check_product(lib, m, n, d, a_fmt, 0, "f32", wild=True, pad=3)
    check_product(lib, m, n, d, a_fmt, 0, "bf16", wild=False, pad=8)
    check_product(lib, m, n, d, a_fmt, 1, "f16", wild=True)


@pytest.mark.parametrize("m,n,d", [(1000, 16400, 384), (1024, 16384, 768), (760, 22016, 630), (512, 32832, 890), (2040, 4100, 2176)])
@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
def test_product_in_whole_steps_of_128_columns(lib, m, n, d, a_fmt):
    check_product(lib, m, n, d, a_fmt, 1, "f32", wild=True)
    check_product(lib, m, n, d, a_fmt, 0, "bf16", wild=False)
    # rows of scores that are longer than their scores and still start on 64 bytes
    check_product(lib, m, n - 12, d, a_fmt, 0, "f32", wild=False, pad=12 + 64 - n % 16)
    check_product(lib, m, n - 12, d, a_fmt, 1, "f16", wild=True, pad=12 + 64 - n % 32)


@pytest.mark.parametrize("m,n,d,kind", [(510, 65601, 520, "f32"), (1000, 33001, 700, "bf16")])
@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
def test_product_of_many_rows_of_any_length(lib, m, n, d, kind, a_fmt):
    check_product(lib, m, n, d, a_fmt, 1, kind, wild=True)
    check_product(lib, m, n, d, a_fmt, 0, kind, wild=False, pad=5)


@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
def test_product_of_one_large_and_many_small_numbers(lib, a_fmt):
    """What an instruction that aligns its products to the largest would drop: 448 * 6 next to 2^-9 * 0.5 in one block."""
    m, n, d = 33, 40, 320
    rng = np.random.default_rng(5)
    ac = rng.integers(1, 8, (m, d)).astype(np.uint8) if a_fmt == MXFP8 else np.full((m, d // 2), 0x11, np.uint8)
    for i in range(m):
        ac[i, rng.integers(0, ac.shape[1])] = 0x7e if a_fmt == MXFP8 else 0x17
    bc = np.full((n, d // 2), 0x11, np.uint8)
    bc[:, rng.integers(0, d // 2, 40)] = 0x77
    asc, bs = np.full((m, 10), 127, np.uint8), np.full((n, 10), 127, np.uint8)
    want = ref.mx_values(ac, asc, a_fmt) @ ref.mx_values(bc, bs, MXFP4).T
    out = torch.empty(m, n, device="cuda")
    product(lib, [torch.from_numpy(t).cuda() for t in (ac, asc)], a_fmt, [torch.from_numpy(t).cuda() for t in (bc, bs)], d, 0,
            (None, None), out, n)
    torch.cuda.synchronize()
    assert np.abs(as64(out) - want).max() <= 20 * U * np.abs(want).max()


@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
@pytest.mark.parametrize("m,n,d", [(3, 50, 40), (40, 300, 200), (300, 700, 300)])
def test_product_with_blocks_that_are_no_number(lib, m, n, d, a_fmt):
    """NaN scales make their rows NaN and no other; scales next to a row's last one belong to the next row and stay there."""
    rng = np.random.default_rng(m)
    ac, asc = random_codes(m, d, a_fmt, rng, False)
    bc, bs = random_codes(n, d, MXFP4, rng, False)
    asc[1, 0] = 255
    bs[7, 0] = 255
    bs[20, -1] = 255
    ac[2, :] = 0
    if a_fmt == MXFP8:
        ac[0, 1] = 0x7f
    out = torch.empty(m, n, device="cuda")
    product(lib, [torch.from_numpy(t).cuda() for t in (ac, asc)], a_fmt, [torch.from_numpy(t).cuda() for t in (bc, bs)], d, 0,
            (None, None), out, n)
    torch.cuda.synchronize()
    nan = np.zeros((m, n), bool)
    nan[1], nan[:, 7], nan[:, 20] = True, True, True
    nan[0] |= a_fmt == MXFP8
    got = as64(out)
    assert np.array_equal(np.isnan(got), nan)
    keep = [j for j in range(n) if j not in (7, 20)]
    assert (got[2, keep] == 0).all()


@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
@pytest.mark.parametrize("m", [2, 130])
def test_product_of_more_codes_than_32_bits_address(lib, m, a_fmt):
    """2.2M rows of 4096 dimensions: 4.5 GB of codes, scores in rows of more than 2^31 bytes."""
    n, d = 2_200_000, 4096
    rng = np.random.default_rng(1)
    ac, asc = random_codes(m, d, a_fmt, rng, False)
    some = rng.integers(0, 256, (1000, d // 2), dtype=np.uint8)
    codes = torch.zeros(n, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, d // 32), 127, dtype=torch.uint8, device="cuda")
    at_rows = np.concatenate([np.arange(500), n - 500 + np.arange(500)])
    codes[torch.from_numpy(at_rows).cuda()] = torch.from_numpy(some).cuda()
    wide = 1_100_000_000 if m == 2 else n
    out = torch.empty(m * wide, dtype=torch.float16, device="cuda")
    product(lib, [torch.from_numpy(t).cuda() for t in (ac, asc)], a_fmt, [codes, scales], d, 0, (None, None), out, wide)
    torch.cuda.synchronize()
    got = torch.stack([out[i * wide:i * wide + n] for i in range(m)])
    want = ref.mx_values(ac, asc, a_fmt) @ ref.mx_values(some, np.full((1000, d // 32), 127, np.uint8), MXFP4).T
    diff = np.abs(as64(got[:, torch.from_numpy(at_rows).cuda()]) - want)
    assert (diff <= 2.0 ** -10 * np.abs(want) + 1e-2).all()
    assert (got[:, 500:n - 500] == 0).all()


def test_rows_at_large_offsets(lib):
    """Row 2 of three starts more than 2^32 bytes behind row 0."""
    d, ld = 100, 1_200_000_000
    x = torch.empty(2 * ld + d, device="cuda")
    want = sample(3, d, 9)
    for i in range(3):
        x[i * ld:i * ld + d] = torch.from_numpy(want[i])
    out = Codes(3, d, MXFP4)
    lib[1](lib[0].ixa_op_quantise(at(x), ld, 0, 3, d, MXFP4, 0.0, at(out.codes), at(out.scales), at(out.sqr), None))
    check_codes(want.astype(np.float64), want, MXFP4, out.get())


def test_more_rows_than_one_launch_takes(lib):
    """1.3 million rows of 2056 elements, 64 different ones over and over: the codes and values of the 64."""
    d, n, some = 2056, 1_300_003, 64
    few = rows(sample(some, d, 5), "bf16")
    which = torch.arange(n, device="cuda") % some
    x = few[which]
    want, got = Codes(some, d, MXFP4), Codes(n, d, MXFP4)
    for t, c in ((few, want), (x, got)):
        lib[1](lib[0].ixa_op_rms_norm_quantise(at(t), d, None, 0, None, 2, c.n, d, 1e-6, None, 0, MXFP4, 0.0, at(c.codes),
                                               at(c.scales), at(c.sqr), None))
    values = [torch.full((c.n, d), 9.0, dtype=torch.bfloat16, device="cuda") for c in (want, got)]
    for v, c in zip(values, (want, got)):
        lib[1](lib[0].ixa_op_dequantise(at(c.codes), at(c.scales), MXFP4, c.n, d, 2, at(v), d, None))
    torch.cuda.synchronize()
    for name, size in (("codes", want.row), ("scales", want.per), ("sqr", 1)):
        small, large = getattr(want, name)[:some * size].view(some, size), getattr(got, name)
        assert all(torch.equal(large[i * size:j * size].view(-1, size), small[which[i:j]])
                   for i in range(0, n, 200_000) for j in [min(n, i + 200_000)])
        assert (large[n * size:] == (7 if name == "sqr" else GUARD)).all()
    assert all(torch.equal(values[1][i:i + 200_000], values[0][which[i:i + 200_000]]) for i in range(0, n, 200_000))


# ----- streams, graphs, the path as a whole ---------------------------------------------------------------------------------

def chain(lib, x, q, w, stream):
    """Hidden states -> norm -> stored 4-bit rows; queries -> 8-bit rows; squared distances; nearest rows."""
    n, m, d = x.shape[0], q.shape[0], x.shape[1]
    base, query = Codes(n, d, MXFP4), Codes(m, d, MXFP8)
    dist, near, label = torch.empty(m, n, device="cuda"), torch.empty(m, 5, device="cuda"), \
        torch.empty(m, 5, dtype=torch.int64, device="cuda")

    def go(s):
        for t, c in ((x, base), (q, query)):
            lib[1](lib[0].ixa_op_rms_norm_quantise(at(t), d, None, 0, at(w), 2, t.shape[0], d, 1e-6, None, 0, c.fmt, 0.0,
                                                   at(c.codes), at(c.scales), at(c.sqr), ctypes.c_void_p(s)))
        lib[1](lib[0].ixa_op_mx_product(at(query.codes), at(query.scales), MXFP8, m, at(base.codes), at(base.scales), n, d, 1,
                                        at(query.sqr), at(base.sqr), 0, at(dist), n, ctypes.c_void_p(s)))
        lib[1](lib[0].ixa_op_topk_flat_fp32(at(dist), m, n, n, 5, 1, at(near), at(label), ctypes.c_void_p(s)))
    return go, dist, label


def test_a_stream_of_its_own_and_a_graph(lib):
    d = 160
    x, q, w = rows(sample(900, d, 1), "bf16"), rows(sample(33, d, 2), "bf16"), rows(sample(1, d, 3) + 2, "bf16")[0]
    go, dist, label = chain(lib, x, q, w, None)
    go(None)
    torch.cuda.synchronize()
    want_d, want_l = dist.clone(), label.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    dist.zero_()
    torch.cuda.synchronize()
    go(s.cuda_stream)
    s.synchronize()
    assert torch.equal(dist, want_d) and torch.equal(label, want_l)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        x.copy_(rows(sample(900, d, 10 + k), "bf16"))
        dist.zero_()
        label.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got_d, got_l = dist.clone(), label.clone()
        go(None)
        torch.cuda.synchronize()
        assert torch.equal(got_d, dist) and torch.equal(got_l, label) and not torch.equal(got_d, want_d)


def test_the_same_call_gives_the_same_bits(lib):
    d = 520
    x, q, w = rows(sample(3000, d, 1), "bf16"), rows(sample(150, d, 2), "bf16"), rows(sample(1, d, 3) + 2, "bf16")[0]
    go, dist, _ = chain(lib, x, q, w, None)
    go(None)
    first = dist.clone()
    for _ in range(3):
        dist.zero_()
        go(None)
        assert torch.equal(dist, first)


def test_4_bit_rows_find_the_nearest(lib):
    """Queries that are stored rows with a little noise: the row itself comes first."""
    d = 128
    x = sample(5000, d, 1)
    q = x[:64] + 0.05 * sample(64, d, 2)
    go, _, label = chain(lib, rows(x, "bf16"), rows(q, "bf16"), None, None)
    go(None)
    torch.cuda.synchronize()
    assert (label[:, 0].cpu().numpy() == np.arange(64)).mean() > 0.95


def test_the_example(lib, capsys):
    """examples/low_precision_search.py: rows to 4 bits keep about a tenth of their norm as error, and the row that a query was
    made from, far nearer than any other, comes first."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "low_precision_search.py")
    spec = importlib.util.spec_from_file_location("low_precision_search", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(n=5003, m=300, d=200, k=10, page=128)
    assert got["bytes"] == 5003 * (7 * 16 + 7 + 4)
    assert got["itself"] == 1.0 and 0.05 < got["error"] < 0.2 and got["recall"] > 0.2
    assert "nearest" in capsys.readouterr().out
