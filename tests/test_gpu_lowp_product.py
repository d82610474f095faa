"""GPU tests of products of low-precision rows where a persistent workgroup takes many tiles, where few queries are in tiles made
for many, and where the blocks of a row differ by many powers of two.  The definition in 64 bits is worked out on the GPU."""
import pytest

import lowp_reference as ref
from test_gpu_lowp import MXFP4, MXFP8, TYPES, U, lib, product  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CHUNK = 4096    # stored rows at a time


def draw(n, d, fmt, gen, scales=(115, 140)):
    """Every number of the format under scales of many sizes; zeros behind the last column."""
    nb = ref.blocks_of(d)
    row = nb * (32 if fmt == MXFP8 else 16)
    codes = torch.randint(0, 256, (n, row), dtype=torch.uint8, device="cuda", generator=gen)
    if fmt == MXFP8:
        codes = torch.where((codes & 127) == 127, codes ^ 1, codes)
        codes[:, d:] = 0
    else:
        codes[:, (d + 1) // 2:] = 0
        if d % 2:
            codes[:, d // 2] &= 15
    return codes, torch.randint(scales[0], scales[1], (n, nb), dtype=torch.uint8, device="cuda", generator=gen)


def values(codes, scales, fmt):
    grid = torch.from_numpy(ref.grid(fmt)).cuda().double()
    half = 8 if fmt == MXFP4 else 128
    if fmt == MXFP8:
        grid = torch.cat((grid, torch.full((1,), float("nan"), device="cuda", dtype=torch.float64)))
        c = codes
    else:
        c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1)
    v = grid[(c % half).long()]
    v = torch.where(c >= half, -v, v)
    s = torch.pow(2.0, scales.double() - 127)
    s[scales == 255] = float("nan")
    return v * s.repeat_interleave(32, 1)


def check(lib, a, a_fmt, b, d, metric, kind, pad=0):  # noqa: F811
    """The product and the error of its sums in 32 bits: a unit of the last place for each of one or two additions per 64 columns."""
    m, n = a[0].shape[0], b[0].shape[0]
    va = values(*a, a_fmt)
    dtype = TYPES[kind][1]
    out = torch.full((m + 1, n + pad), 9.0, dtype=dtype, device="cuda")
    sq_a = torch.nan_to_num((va ** 2).sum(-1)).float()
    sq_b = torch.cat([torch.nan_to_num((values(b[0][i:i + CHUNK], b[1][i:i + CHUNK], MXFP4) ** 2).sum(-1)).float()
                      for i in range(0, n, CHUNK)])
    product(lib, a, a_fmt, b, d, metric, (sq_a, sq_b) if metric else (None, None), out, n + pad)
    torch.cuda.synchronize()
    assert (out[m] == 9).all() and (out[:, n:] == 9).all()
    adds = 2 * ((ref.blocks_of(d) + 1) // 2) + 8
    worst = 0.0
    for i in range(0, n, CHUNK):
        vb = values(b[0][i:i + CHUNK], b[1][i:i + CHUNK], MXFP4)
        # a NaN makes its row NaN and touches no other: rows without one are compared, the others have to be NaN
        g, mag = va @ vb.t(), va.abs() @ vb.abs().t()
        got = out[:m, i:i + CHUNK][:, :vb.shape[0]].double()
        bad = va.isnan().any(1)[:, None] | vb.isnan().any(1)[None, :]
        assert torch.equal(got.isnan(), bad)
        bound = adds * 2 * U * mag
        if metric:
            s = sq_a.double()[:, None] + sq_b.double()[None, i:i + CHUNK]
            g = s - 2 * g
            bound = 2 * bound + 3 * U * (s + 2 * mag)
        least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[kind]
        bound = bound * 1.01 + {"f32": 0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind] * g.abs() + least
        ok = ((got - g).abs() <= bound) | bad
        if kind == "f16":
            big = g.abs() - bound > 65520
            ok = torch.where(big, got == torch.sign(g) * float("inf"), ok | (g.abs() + bound >= 65520))
        worst = max(worst, ((got - g).abs() / bound)[~bad].nan_to_num().max().item()) if (~bad).any() else worst
        assert ok.all(), f"columns {i} ...: {int((~ok).sum())} scores are off, by up to {worst:.2f} of what sums in 32 bits lose"
    return worst


@pytest.mark.parametrize("d", [512, 640, 768, 896])
@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
@pytest.mark.parametrize("metric,kind", [(1, "f32"), (0, "bf16")])
def test_many_tiles_for_every_workgroup(lib, d, a_fmt, metric, kind):  # noqa: F811
    """1028 tiles of 256 x 256, four or five for each of 256 workgroups, in rows of four to seven steps of 128 columns: the places
    of codes and scales go round several times, with every phase at a tile's end."""
    gen = torch.Generator(device="cuda").manual_seed(d + a_fmt)
    check(lib, draw(1024, d, a_fmt, gen), a_fmt, draw(65600, d, MXFP4, gen), d, metric, kind)


@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
@pytest.mark.parametrize("metric,kind", [(0, "f32"), (1, "f16")])
def test_wide_tiles_with_blocks_that_are_no_number(lib, a_fmt, metric, kind):  # noqa: F811
    """514 tiles; NaN scales and an 8-bit NaN in first and later tiles, first and last rows and blocks."""
    m, n, d = 500, 65600, 640
    gen = torch.Generator(device="cuda").manual_seed(a_fmt)
    a = draw(m, d, a_fmt, gen, (108, 115) if kind == "f16" else (115, 140))
    b = draw(n, d, MXFP4, gen, (120, 128) if kind == "f16" else (115, 140))
    for row, block in ((0, 19), (130, 0), (257, 7), (499, 12)):
        a[1][row, block] = 255
    for row, block in ((0, 0), (7, 19), (300, 4), (33000, 11), (60001, 18), (65599, 19)):
        b[1][row, block] = 255
    if a_fmt == MXFP8:
        a[0][77, 333], a[0][444, 0] = 0x7f, 0xff
    check(lib, a, a_fmt, b, d, metric, kind)


@pytest.mark.parametrize("m,n,d,a_fmt", [(64, 98_050, 1024, MXFP8), (8, 98_100, 16384, MXFP8), (33, 98_311, 4100, MXFP4),
                                         (64, 98_048, 1024, MXFP8), (17, 20_001, 4096, MXFP8)])
def test_few_queries_whose_codes_do_not_stay_in_lds(lib, m, n, d, a_fmt):  # noqa: F811
    """Up to 64 queries in tiles made for 64 or for 128, on both sides of the line between them."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    a, b = draw(m, d, a_fmt, gen), draw(n, d, MXFP4, gen)
    check(lib, a, a_fmt, b, d, 0, "f32")
    check(lib, a, a_fmt, b, d, 1, "bf16", pad=3)


@pytest.mark.parametrize("a_fmt", [MXFP4, MXFP8])
@pytest.mark.parametrize("m,n,d", [(3, 700, 512), (40, 40_000, 128), (300, 700, 512), (1000, 16_400, 512)])
def test_blocks_that_differ_by_many_powers_of_two(lib, m, n, d, a_fmt):  # noqa: F811
    """One block of a row holds one large product, its neighbours 32 that are 2^8 to 2^24 times smaller each: together they count,
    and an instruction that aligns the products of several blocks to the largest would lose them."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    for shift in range(8, 25, 2):
        a, b = draw(m, d, a_fmt, gen, (127, 128)), draw(n, d, MXFP4, gen, (127, 128))
        # every number positive, so that nothing cancels
        a[0].bitwise_and_(0x7f if a_fmt == MXFP8 else 0x77)
        b[0].bitwise_and_(0x77)
        a[1].fill_(127 - shift)
        large = torch.randint(0, d // 32, (m,), device="cuda", generator=gen)
        a[1][torch.arange(m, device="cuda"), large] = 127
        per = 32 if a_fmt == MXFP8 else 16
        wide = a[0].view(m, -1, per)
        one = torch.zeros(m, per, dtype=torch.uint8, device="cuda")
        one[:, 3] = 0x38 if a_fmt == MXFP8 else 0x02
        wide[torch.arange(m, device="cuda"), large] = one
        check(lib, a, a_fmt, b, d, 0, "f32")
