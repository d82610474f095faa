"""The work that the low-precision operators are measured on: embeddings on their way into and through an 8-bit or 4-bit store.

Three kinds of pass, each through the public entry points on GPU memory:

* ``quantise`` -- float vectors become codes with scales and the squared norms of what the codes stand for
  (``ixa_op_quantise``), and the codes are read back as values (``ixa_op_dequantise``), as a store is filled and checked;
* ``norm``     -- an embedding model's last step: residual added, root-mean-square norm, weight, codes with scales
  (``ixa_op_rms_norm_quantise``), read back as above;
* ``product``  -- scores of query rows against stored 4-bit rows (``ixa_op_mx_product``): inner products or squared distances.

``listed`` holds the named cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes what a program has in
hand (the vectors, or the stored codes with their scales and norms, and the buffers it keeps for the results), ``run`` is one
pass.  Where ``own`` is false ``run`` works the definitions out in elementary torch operations in 32 bits.

The values of 8-bit and 4-bit codes are given in bfloat16: it holds an E2M1 or E4M3 number times a power of two exactly, and
an int8 code times its row's scale to half a unit of its last place.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
_FORMATS = {"int8": 0, "mxfp8": 1, "mxfp4": 2}
_METRICS = {"IP": 0, "L2": 1}
_BLOCK = 32
# exponent of the largest power of two that an element of the format holds, and its largest number
_TOP = {"mxfp8": (8, 448.0), "mxfp4": (2, 6.0)}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # One query vector of the headline dimension becomes 8-bit blocks: launches and latency count.
        {"name": "quantise_query", "kind": "quantise", "n": 1, "d": 128, "pad": 0, "type": "f32", "format": "mxfp8"},
        # A collection goes into the 4-bit store: 1.2M x 200, a size and a dimension off every tile (200 = 6 blocks and a
        # quarter), the float vectors with a stride of their own.
        {"name": "quantise_base", "kind": "quantise", "n": 1_234_567, "d": 200, "pad": 8, "type": "f32", "format": "mxfp4"},
        # The last step of an embedding model for one query of 768 dimensions, into int8 with the row's scale.
        {"name": "norm_query", "kind": "norm", "n": 1, "d": 768, "pad": 0, "type": "bf16", "format": "int8",
         "residual": True},
        # The same for the benchmark's batch of 4096 queries, into 8-bit blocks for the product.
        {"name": "norm_batch", "kind": "norm", "n": 4096, "d": 768, "pad": 0, "type": "bf16", "format": "mxfp8",
         "residual": True},
        # An odd batch of half-precision rows in a wider buffer, no residual.
        {"name": "norm_ragged", "kind": "norm", "n": 999, "d": 1000, "pad": 24, "type": "f16", "format": "int8",
         "residual": False},
        # A corpus's hidden states at the largest dimension an index takes, into int8.
        {"name": "norm_corpus", "kind": "norm", "n": 131_072, "d": 4096, "pad": 0, "type": "bf16", "format": "int8",
         "residual": True},
        # Eight queries against 1024 list centroids: the smallest product of a search.
        {"name": "product_lists", "kind": "product", "m": 8, "n": 1024, "d": 128, "a_format": "mxfp8", "metric": "L2",
         "out": "f32"},
        # One interactive query against a million stored rows.
        {"name": "product_query", "kind": "product", "m": 1, "n": 1_000_000, "d": 128, "a_format": "mxfp8", "metric": "L2",
         "out": "f32"},
        # Odd everything: 37 queries, 100003 rows, 200 dimensions, half-precision scores.
        {"name": "product_ragged", "kind": "product", "m": 37, "n": 100_003, "d": 200, "a_format": "mxfp4",
         "metric": "IP", "out": "f16"},
        # The largest small batch, 64 queries, against a million unit-norm embeddings of 768 dimensions.
        {"name": "product_64", "kind": "product", "m": 64, "n": 1_000_000, "d": 768, "a_format": "mxfp8", "metric": "IP",
         "out": "f32"},
        # A batch of 2048 queries against one stretch of a large base: the scores fill the default scratch of 1 GiB.
        {"name": "product_batch", "kind": "product", "m": 2048, "n": 131_072, "d": 768, "a_format": "mxfp4",
         "metric": "L2", "out": "f32"},
        # 4096 queries against 32768 list centroids at the largest dimension, scores in bfloat16: the matrix cores.
        {"name": "product_wide", "kind": "product", "m": 4096, "n": 32_768, "d": 4096, "a_format": "mxfp4",
         "metric": "IP", "out": "bf16"},
    ]


def _log_int(rng, lo, hi):
    """An integer between lo and hi, uniform over the logarithm; every second one of some size is a multiple of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v = v // 32 * 32
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quantise", "norm", "product", "product"])
    if kind == "product":
        d = _log_int(rng, 32, 4096)
        n = _log_int(rng, 1000, min(1_000_000, 500_000_000 // d))
        m = _log_int(rng, 1, max(1, min(4096, 250_000_000 // n, 500_000_000_000 // (n * d))))
        return {"kind": kind, "m": m, "n": n, "d": d, "a_format": rng.choice(["mxfp4", "mxfp8"]),
                "metric": rng.choice(["IP", "L2"]), "out": rng.choice(["f32", "f32", "f16", "bf16"])}
    d = _log_int(rng, 32, 4096)
    n = _log_int(rng, 1, 200_000_000 // d)
    case = {"kind": kind, "n": n, "d": d, "pad": rng.choice([0, 0, 8, 3]), "type": rng.choice(["f32", "f16", "bf16"])}
    if kind == "quantise":
        case["format"] = rng.choice(["mxfp4", "mxfp4", "mxfp8"])
    else:
        case["format"] = rng.choice(["int8", "mxfp8"])
        case["residual"] = rng.random() < 0.7
    return case


def _blocks(d):
    return (d + _BLOCK - 1) // _BLOCK


def _code_bytes(fmt, d):
    return d if fmt == "int8" else _blocks(d) * (_BLOCK if fmt == "mxfp8" else _BLOCK // 2)


def work(case):
    if case["kind"] == "product":
        m, n, d = case["m"], case["n"], case["d"]
        size = 4 if case["out"] == "f32" else 2
        moved = m * (_code_bytes(case["a_format"], d) + _blocks(d)) + n * (_code_bytes("mxfp4", d) + _blocks(d))
        moved += m * n * size + ((m + n) * 4 if case["metric"] == "L2" else 0)
        return {"bytes": moved, "flops": 2 * m * n * d}
    n, d = case["n"], case["d"]
    size = 4 if case["type"] == "f32" else 2
    coded = n * (_code_bytes(case["format"], d) + (4 if case["format"] == "int8" else _blocks(d)))
    moved = n * d * size + 2 * coded + n * d * 2        # vectors in, codes out and in again, bfloat16 values out
    if case["kind"] == "norm":
        moved += (2 * n * d * size if case["residual"] else 0) + d * size
        return {"bytes": moved, "flops": 8 * n * d}
    return {"bytes": moved + 4 * n, "flops": 5 * n * d}


def _rows(n, d, gen):
    """Embeddings: a mixture of directions with noise, rows of different lengths."""
    comp = torch.randn(256, d, device="cuda", generator=gen)
    which = torch.randint(0, 256, (n,), device="cuda", generator=gen)
    x = torch.randn(n, d, device="cuda", generator=gen).mul_(0.25).add_(comp[which])
    return x.mul_(torch.rand(n, 1, device="cuda", generator=gen).add_(0.5))


def _padded(x, pad, dtype):
    """x in rows of x.shape[1] + pad elements."""
    if not pad:
        return x.to(dtype)
    wide = torch.full((x.shape[0], x.shape[1] + pad), 7.0, device="cuda", dtype=dtype)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    d = case["d"]
    s = {"case": case}
    if case["kind"] == "product":
        m, n = case["m"], case["n"]
        s["a_codes"], s["a_scales"], s["a_sqr"] = _pack(_rows(m, d, gen).mul_(d ** -0.5), case["a_format"])
        s["b_codes"], s["b_scales"], s["b_sqr"] = _pack(_rows(n, d, gen).mul_(d ** -0.5), "mxfp4")
        s["out"] = torch.empty(m, n, device="cuda", dtype=_TYPES[case["out"]][1])
        return s
    n, dtype, fmt = case["n"], _TYPES[case["type"]][1], case["format"]
    x = _rows(n, d, gen)
    if case["kind"] == "norm":
        # hidden states have a few channels that are much larger than the rest
        x[:, torch.randint(0, d, (max(1, d // 200),), device="cuda", generator=gen)] *= 20
        s["weight"] = torch.rand(d, device="cuda", generator=gen).add_(0.5).to(dtype)
        if case["residual"]:
            s["residual"] = _padded(_rows(n, d, gen), case["pad"], dtype)
            s["sum"] = torch.empty(n, d, device="cuda", dtype=dtype)
    s["x"] = _padded(x, case["pad"], dtype)
    s["codes"] = torch.empty(n, _code_bytes(fmt, d), device="cuda", dtype=torch.uint8)
    s["scales"] = torch.empty(n, device="cuda") if fmt == "int8" else torch.empty(n, _blocks(d), device="cuda",
                                                                                  dtype=torch.uint8)
    s["sqr"] = torch.empty(n, device="cuda")
    s["values"] = torch.empty(n, d, device="cuda", dtype=torch.bfloat16)
    return s


# ----- plain forms -----------------------------------------------------------------------------------------------------

def _mx_scale(blocks, fmt):
    """Biased exponents of the blocks' scales [n][nb]: the power of two of the largest magnitude, less the format's own."""
    exponent = torch.frexp(blocks.abs().amax(-1))[1] - 1
    biased = (exponent - _TOP[fmt][0] + 127).clamp_(0, 254)
    return torch.where(blocks.abs().amax(-1) == 0, torch.zeros_like(biased), biased)


def _mx_round(v, fmt):
    """v (scaled, 32 bits) to the nearest number of the format, ties to even, the largest number where v is beyond it."""
    if fmt == "mxfp8":
        return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    a = v.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp_(max=6.0)
    return torch.copysign(r, v)


def _split(x):
    """x (n, d) in blocks of 32 (n, nb, 32), zeros behind the last column."""
    n, d = x.shape
    nb = _blocks(d)
    return torch.nn.functional.pad(x, (0, nb * _BLOCK - d)).view(n, nb, _BLOCK)


def _mx(x, fmt):
    """(numbers of the format [n][nb][32], biased scales [n][nb]) of 32-bit rows."""
    blocks = _split(x)
    biased = _mx_scale(blocks, fmt)
    return _mx_round(torch.ldexp(blocks, (127 - biased).unsqueeze(-1)), fmt), biased


def _pack(x, fmt):
    """Codes, scales and squared norms as a store keeps them."""
    q, biased = _mx(x, fmt)
    n = x.shape[0]
    sqr = torch.ldexp(q, (biased - 127).unsqueeze(-1)).square_().sum((1, 2))
    if fmt == "mxfp8":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8).view(n, -1)
    else:
        a = q.abs()
        code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
        code |= torch.signbit(q).to(torch.uint8) << 3
        code = code.view(n, -1, 2)
        codes = code[..., 0] | (code[..., 1] << 4)
    return codes.contiguous(), biased.to(torch.uint8).contiguous(), sqr


def _unpack(codes, scales, fmt):
    """The 32-bit values [n][nb * 32] that codes and scales stand for."""
    n, nb = scales.shape
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(_E2M1, device=codes.device)
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
    return torch.ldexp(v.view(n, nb, _BLOCK), (scales.int() - 127).unsqueeze(-1)).view(n, nb * _BLOCK)


def _plain(s):
    case = s["case"]
    if case["kind"] == "product":
        a, b = _unpack(s["a_codes"], s["a_scales"], case["a_format"]), _unpack(s["b_codes"], s["b_scales"], "mxfp4")
        g = a @ b.t()
        if case["metric"] == "L2":
            g = (s["a_sqr"][:, None] + s["b_sqr"][None, :]) - g - g
        return g.to(_TYPES[case["out"]][1])
    fmt, d = case["format"], case["d"]
    y, out = s["x"].float(), {}
    if case["kind"] == "norm":
        if case["residual"]:
            y = y + s["residual"].float()
            out["sum"] = y.to(s["x"].dtype)
        y = y * (1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)) * s["weight"].float()
    if fmt == "int8":
        top = y.abs().amax(-1, keepdim=True)
        scale = top / 127.0
        q = torch.round(y * torch.where(top > 0, 127.0 / top, torch.zeros_like(top)))
        out["values"] = (q * scale).to(torch.bfloat16)
        out["scales"] = scale.view(-1)
        return out
    q, biased = _mx(y, fmt)
    v = torch.ldexp(q, (biased - 127).unsqueeze(-1)).view(q.shape[0], -1)
    if case["kind"] == "quantise":
        out["sqr"] = (v * v).sum(-1)
    out["values"] = v[:, :d].to(torch.bfloat16)
    return out


# ----- the framework's operators ---------------------------------------------------------------------------------------

_bound = None


def _lib():
    global _bound
    if _bound is None:
        from indexsdk_amd import _capi
        _bound = (_capi.load(), _capi.check)
    return _bound


def _at(t):
    return ctypes.c_void_p(t.data_ptr() if t is not None else None)


def _kernels(s):
    lib, check = _lib()
    case = s["case"]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    if case["kind"] == "product":
        l2 = case["metric"] == "L2"
        check(lib.ixa_op_mx_product(_at(s["a_codes"]), _at(s["a_scales"]), _FORMATS[case["a_format"]], case["m"],
                                    _at(s["b_codes"]), _at(s["b_scales"]), case["n"], case["d"], _METRICS[case["metric"]],
                                    _at(s["a_sqr"] if l2 else None), _at(s["b_sqr"] if l2 else None),
                                    _TYPES[case["out"]][0], _at(s["out"]), case["n"], stream))
        return s["out"]
    n, d, fmt, kind, x = case["n"], case["d"], _FORMATS[case["format"]], _TYPES[case["type"]][0], s["x"]
    out = {"values": s["values"]}
    if case["kind"] == "norm":
        res, total = s.get("residual"), s.get("sum")
        check(lib.ixa_op_rms_norm_quantise(_at(x), x.stride(0), _at(res), res.stride(0) if res is not None else 0,
                                           _at(s["weight"]), kind, n, d, 1e-6, _at(total), d if total is not None else 0,
                                           fmt, 0.0, _at(s["codes"]), _at(s["scales"]), None, stream))
        if total is not None:
            out["sum"] = total
        if case["format"] == "int8":
            out["scales"] = s["scales"]
    else:
        check(lib.ixa_op_quantise(_at(x), x.stride(0), kind, n, d, fmt, 0.0, _at(s["codes"]), _at(s["scales"]),
                                  _at(s["sqr"]), stream))
        out["sqr"] = s["sqr"]
    check(lib.ixa_op_dequantise(_at(s["codes"]), _at(s["scales"]), fmt, n, d, _TYPES["bf16"][0], _at(s["values"]), d, stream))
    return out


def run(state):
    return _kernels(state) if own else _plain(state)


# ----- the definitions in 64 bits --------------------------------------------------------------------------------------

def _grid(fmt):
    """The non-negative numbers of the format, ascending."""
    if fmt == "mxfp4":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
    e, f = np.divmod(np.arange(127), 8)
    return np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))


def _nearest(v, grid):
    """The number of the grid nearest to each v >= 0; halfway the one with the even place; the last one beyond the end."""
    mid = (grid[:-1] + grid[1:]) / 2
    at = torch.bucketize(v, mid)                       # the lower of two neighbours halfway between them
    odd = (at % 2 == 1) & (at < len(mid)) & (v == mid[at.clamp(max=len(mid) - 1)])
    return grid[at + odd]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        def values(codes, scales, fmt):
            power = torch.pow(2.0, scales.double() - 127).repeat_interleave(_BLOCK, 1)
            grid = torch.from_numpy(_grid(fmt)).cuda()
            c = codes if fmt == "mxfp8" else torch.stack((codes % 16, codes // 16), -1).view(codes.shape[0], -1)
            half = 128 if fmt == "mxfp8" else 8
            return torch.where(c >= half, -1.0, 1.0).double() * grid[(c % half).long()] * power
        a, b = values(s["a_codes"], s["a_scales"], case["a_format"]), values(s["b_codes"], s["b_scales"], "mxfp4")
        g = a @ b.t()
        if case["metric"] == "L2":
            g = s["a_sqr"].double()[:, None] + s["b_sqr"].double()[None, :] - 2 * g
        return g
    d, fmt = case["d"], case["format"]
    y, out = s["x"].double(), {}
    if case["kind"] == "norm":
        if case["residual"]:
            y = y + s["residual"].double()
            out["sum"] = y
        y = y / torch.sqrt(torch.sum(y ** 2, -1, keepdim=True) / d + 1e-6) * s["weight"].double()
    if fmt == "int8":
        scale = y.abs().amax(-1) / 127
        return {**out, "values": torch.round(y / scale[:, None]) * scale[:, None], "scales": scale}
    grid = torch.from_numpy(_grid(fmt)).cuda()
    values = torch.zeros_like(y)
    for k in range(0, d, _BLOCK):
        block = y[:, k:k + _BLOCK]
        top = block.abs().amax(-1, keepdim=True)
        power = torch.pow(2.0, (torch.floor(torch.log2(top)) - _TOP[fmt][0]).clamp(-127, 127))
        power = torch.where(top > 0, power, torch.ones_like(power))
        values[:, k:k + _BLOCK] = torch.sign(block) * _nearest(block.abs() / power, grid) * power
    out["values"] = values
    if case["kind"] == "quantise":
        out["sqr"] = (values ** 2).sum(-1)
    return out
