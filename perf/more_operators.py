"""The work that the score operators are measured on: scores against rows kept in 4 bits, and what is done with them.

Four kinds of pass, each through the public entry points on GPU memory:

* ``quantise`` -- float rows become 4-bit codes with a scale (and a zero point) per group of 32, 64 or 128 elements
  (``ixa_op_group_quantise``) and are read back as values (``ixa_op_group_dequantise``), as a store is filled and checked;
* ``product``  -- scores of float rows against such rows (``ixa_op_group_product``), from one query to a batch;
* ``sample``   -- columns drawn from rows of scores under temperature, top-k, top-p and min-p from given random numbers
  (``ixa_op_sample``): one answer per row, or several as sampled negatives;
* ``distil``   -- the loss of rows of scores against a teacher's top entries and its gradient, in one call
  (``ixa_op_distil_step``) or in two (``ixa_op_distil_loss``, ``ixa_op_distil_gradient``), as a training step takes them.

``listed`` holds the named cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes what a program has in
hand and the buffers it keeps for the results, ``run`` is one pass.  Where ``own`` is false ``run`` works the definitions out in
elementary torch operations: in 32 bits, and in 64 where a value decides what is next to a border (codes, running sums of
probabilities).
"""
import ctypes
import math

import torch

own = False

_TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}


def listed():
    return [
        # A collection goes into the 4-bit store: dimensions off every group (200 = 6 groups and a quarter of 32), the float
        # rows with a stride of their own, one scale in half precision per group.
        {"name": "quantise_base", "kind": "quantise", "n": 1_000_003, "d": 200, "pad": 8, "type": "f32", "group": 32,
         "scale": "f16", "zeros": False},
        # A weight matrix or a page of a collection at an embedding's size, with zero points.
        {"name": "quantise_page", "kind": "quantise", "n": 16_384, "d": 768, "pad": 0, "type": "bf16", "group": 128,
         "scale": "bf16", "zeros": True},
        # One query of the headline dimension against 16384 list centroids: the smallest product, latency counts.
        {"name": "product_lists", "kind": "product", "m": 1, "n": 16_384, "d": 128, "group": 32, "scale": "f16",
         "zeros": False, "type": "f32", "out": "f32"},
        # One interactive query against a million stored rows, or one token against a large output table.
        {"name": "product_query", "kind": "product", "m": 1, "n": 1_000_000, "d": 768, "group": 64, "scale": "f16",
         "zeros": True, "type": "bf16", "out": "f32"},
        # Odd everything: 37 rows, 100003 stored rows, 200 dimensions.
        {"name": "product_ragged", "kind": "product", "m": 37, "n": 100_003, "d": 200, "group": 32, "scale": "bf16",
         "zeros": True, "type": "f16", "out": "f16"},
        # A batch of 2048 queries against one stretch of a large base.
        {"name": "product_batch", "kind": "product", "m": 2048, "n": 131_072, "d": 768, "group": 128, "scale": "f16",
         "zeros": False, "type": "bf16", "out": "bf16"},
        # One answer from one row of scores, all filters on: launches and latency count.
        {"name": "sample_one", "kind": "sample", "rows": 1, "n": 32_768, "type": "f32", "draws": 1, "filters": "all"},
        # A serving batch that keeps the likeliest nine tenths of long rows.
        {"name": "sample_nucleus", "kind": "sample", "rows": 64, "n": 131_072, "type": "f32", "draws": 1, "filters": "top_p"},
        # Negatives for a training batch: four draws from each of 1024 odd rows, every row with settings of its own.
        {"name": "sample_negatives", "kind": "sample", "rows": 1024, "n": 100_003, "type": "bf16", "draws": 4,
         "filters": "mixed"},
        # Eight queries against 1024 centroids, ten teacher entries each: the smallest training step.
        {"name": "distil_small", "kind": "distil", "rows": 8, "n": 1024, "k": 10, "type": "f32", "pad": 0, "apart": False,
         "whole": False},
        # Odd rows of a wider buffer, loss first and gradient later with upstream weights.
        {"name": "distil_ragged", "kind": "distil", "rows": 999, "n": 100_003, "k": 64, "type": "f32", "pad": 5, "apart": True,
         "whole": True},
        # A large step: 4096 rows over 131072 columns against a teacher's top hundred.
        {"name": "distil_step", "kind": "distil", "rows": 4096, "n": 131_072, "k": 100, "type": "bf16", "pad": 0,
         "apart": False, "whole": False},
    ]


def _log_int(rng, lo, hi):
    """An integer between lo and hi, uniform over the logarithm; every second one of some size is a multiple of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v = v // 32 * 32
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "sample", "sample", "distil", "distil"])
    kinds = ["f32", "f16", "bf16"]
    if kind in ("quantise", "product"):
        d = _log_int(rng, 32, 4096)
        case = {"kind": kind, "d": d, "group": rng.choice([32, 64, 128]), "scale": rng.choice(["f16", "bf16", "f32"]),
                "zeros": rng.random() < 0.5, "type": rng.choice(kinds)}
        if kind == "quantise":
            return {**case, "n": _log_int(rng, 1, 200_000_000 // d), "pad": rng.choice([0, 0, 8, 3])}
        n = _log_int(rng, 1000, min(1_000_000, 750_000_000 // d))
        m = _log_int(rng, 1, max(1, min(2048, 250_000_000 // n, 200_000_000_000 // (n * d))))
        return {**case, "m": m, "n": n, "out": rng.choice(kinds)}
    n = _log_int(rng, 1000, 131_072)
    if kind == "sample":
        return {"kind": kind, "rows": _log_int(rng, 1, min(1024, 100_000_000 // n)), "n": n, "type": rng.choice(kinds),
                "draws": rng.choice([1, 1, 4, 16]),
                "filters": rng.choice(["none", "top_k", "top_p", "min_p", "all", "mixed"])}
    return {"kind": kind, "rows": _log_int(rng, 1, min(4096, 500_000_000 // n)), "n": n, "k": _log_int(rng, 1, 256),
            "type": rng.choice(kinds), "pad": rng.choice([0, 0, 8, 5]), "apart": rng.random() < 0.5,
            "whole": rng.random() < 0.5}


def _groups(case):
    return (case["d"] + case["group"] - 1) // case["group"]


def _size(kind):
    return 4 if kind == "f32" else 2


def work(case):
    kind = case["kind"]
    if kind in ("quantise", "product"):
        n, d, ng = case["n"], case["d"], _groups(case)
        coded = n * (ng * case["group"] // 2 + ng * (_size(case["scale"]) + (1 if case["zeros"] else 0)))
        if kind == "quantise":      # rows in, codes out and in again, fp32 values out
            return {"bytes": n * d * _size(case["type"]) + 2 * coded + n * d * 4, "flops": 5 * n * d}
        m = case["m"]
        return {"bytes": coded + m * d * _size(case["type"]) + m * n * _size(case["out"]) + n * 4, "flops": 2 * m * n * d}
    rows, n, size = case["rows"], case["n"], _size(case["type"])
    if kind == "sample":
        return {"bytes": rows * n * size + rows * case["draws"] * 16, "flops": 3 * rows * n}
    return {"bytes": 2 * rows * n * size + rows * (case["k"] * 12 + 4), "flops": 7 * rows * n}


# ----- what a program has in hand --------------------------------------------------------------------------------------

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


def _scores(rows, n, gen):
    """Scores as a model's last layer gives them: a few columns stand out, the many others fall off slowly."""
    rank = torch.rand(rows, n, device="cuda", generator=gen).mul_(n).add_(1.0)
    return rank.log_().mul_(-1.3).add_(torch.randn(rows, n, device="cuda", generator=gen)).add_(6.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, s = case["kind"], {"case": case}
    if kind in ("quantise", "product"):
        n, d, ng = case["n"], case["d"], _groups(case)
        row = ng * case["group"] // 2
        scale_type = _TYPES[case["scale"]][1]
        if kind == "quantise":
            s["x"] = _padded(_rows(n, d, gen), case["pad"], _TYPES[case["type"]][1])
            s["codes"] = torch.empty(n, row, device="cuda", dtype=torch.uint8)
            s["scales"] = torch.empty(n, ng, device="cuda", dtype=scale_type)
            s["zeros"] = torch.empty(n, ng, device="cuda", dtype=torch.uint8) if case["zeros"] else None
            s["values"] = torch.empty(n, d, device="cuda")
            return s
        # a store as it is kept: codes of every size, scales that go with rows of different lengths
        m = case["m"]
        codes = torch.randint(0, 256, (n, row), device="cuda", generator=gen, dtype=torch.uint8)
        size = torch.rand(n, 1, device="cuda", generator=gen).add_(0.5).mul_(0.3 * d ** -0.5)
        s["scales"] = (torch.rand(n, ng, device="cuda", generator=gen).add_(0.5) * size).to(scale_type)
        s["zeros"] = torch.randint(5, 11, (n, ng), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None
        s["codes"] = codes
        s["x"] = _rows(m, d, gen).to(_TYPES[case["type"]][1])
        s["bias"] = torch.randn(n, device="cuda", generator=gen).mul_(0.1)
        s["out"] = torch.empty(m, n, device="cuda", dtype=_TYPES[case["out"]][1])
        if own:
            s["work"] = _workspace("ixa_group_product_workspace", _TYPES[case["type"]][0], m, d)
        return s
    rows, n, dtype = case["rows"], case["n"], _TYPES[case["type"]][1]
    if kind == "sample":
        s["scores"] = _scores(rows, n, gen).to(dtype)
        row = torch.arange(rows, device="cuda")
        pick = lambda *options: torch.tensor(options, device="cuda")[row % len(options)]
        f = case["filters"]
        s["temperature"] = pick(0.7, 1.0, 1.3, 0.0) if f == "mixed" else torch.full((rows,), 0.8, device="cuda")
        s["top_k"] = {"top_k": torch.full((rows,), 50, device="cuda"), "all": torch.full((rows,), 40, device="cuda"),
                      "mixed": pick(50, 0, 200, 0, 20)}.get(f)
        s["top_k"] = None if s["top_k"] is None else s["top_k"].int()
        s["top_p"] = {"top_p": torch.full((rows,), 0.9, device="cuda"), "all": torch.full((rows,), 0.95, device="cuda"),
                      "mixed": pick(0.9, 0.8, 1.0)}.get(f)
        s["min_p"] = {"min_p": torch.full((rows,), 0.02, device="cuda"), "all": torch.full((rows,), 0.01, device="cuda"),
                      "mixed": pick(0.0, 0.0, 0.05, 0.1, 0.0, 0.01, 0.0)}.get(f)
        s["uniform"] = torch.rand(rows, case["draws"], device="cuda", generator=gen)
        s["labels"] = torch.empty(rows, case["draws"], device="cuda", dtype=torch.int64)
        s["probs"] = torch.empty(rows, case["draws"], device="cuda")
        if own:
            s["work"] = _workspace("ixa_sample_workspace", rows, n)
        return s
    k = case["k"]
    scores = _scores(rows, n, gen)
    # the teacher agrees with the student on much and has the rest of its own
    near = scores + 0.7 * torch.randn(rows, n, device="cuda", generator=gen)
    top = near.topk(k, dim=1)
    s["teacher"], s["labels"] = top.values.contiguous(), top.indices.contiguous()
    short = torch.randint(0, 8, (rows,), device="cuda", generator=gen) == 0     # lists that ran out end in -1
    s["labels"][short, k - k // 4:] = -1
    s["whole"] = torch.logsumexp(near / 2.0, 1) if case["whole"] else None
    del near
    s["scores"] = _padded(scores, case["pad"], dtype)
    s["weight"] = torch.rand(rows, device="cuda", generator=gen).add_(0.5).div_(rows)
    s["gradient"] = torch.empty(rows, n, device="cuda", dtype=dtype)
    s["loss"] = torch.empty(rows, device="cuda")
    s["stats"] = torch.empty(rows, 2, device="cuda")
    if own:
        s["work"] = _workspace("ixa_distil_workspace", rows, n)
    return s


# ----- plain forms -----------------------------------------------------------------------------------------------------

def _split(x, group):
    """x (n, d) in groups (n, ng, group), zeros behind the last column."""
    n, d = x.shape
    ng = (d + group - 1) // group
    return torch.nn.functional.pad(x, (0, ng * group - d)).view(n, ng, group)


def _plain_quantise(s):
    case = s["case"]
    x = _split(s["x"].double(), case["group"])
    scale_type, top = _TYPES[case["scale"]][1], torch.finfo(_TYPES[case["scale"]][1]).max
    if case["zeros"]:
        low, high = x.amin(-1).clamp_(max=0), x.amax(-1).clamp_(min=0)
        scale = ((high - low) / 15).clamp_(max=top).to(scale_type)
        divisor = torch.where(scale > 0, scale.double(), torch.ones_like(low))
        zero = torch.round(-low / divisor).clamp_(0, 15) * (scale > 0)
    else:
        scale = (x.abs().amax(-1) / 7).clamp_(max=top).to(scale_type)
        divisor = torch.where(scale > 0, scale.double(), torch.ones_like(x[..., 0]))
        zero = torch.full_like(divisor, 8)
    code = (torch.round(x / divisor.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp_(0, 15)
    value = ((code - zero.unsqueeze(-1)) * scale.double().unsqueeze(-1)).view(x.shape[0], -1)[:, :case["d"]]
    out = {"values": value.float(), "scales": scale}
    if case["zeros"]:
        out["zeros"] = zero.to(torch.uint8)
    return out


def _store_values(s, dtype):
    case = s["case"]
    codes = s["codes"]
    n, ng = s["scales"].shape
    v = torch.empty(n, ng * case["group"], device=codes.device, dtype=dtype)
    v[:, 0::2] = codes & 15
    v[:, 1::2] = codes >> 4
    v = v.view(n, ng, case["group"])
    v -= 8 if s["zeros"] is None else s["zeros"].to(dtype).unsqueeze(-1)
    v *= s["scales"].to(dtype).unsqueeze(-1)
    return v.view(n, -1)[:, :case["d"]]


def _plain_product(s):
    g = s["x"].float() @ _store_values(s, torch.float32).t()
    return (g + s["bias"]).to(s["out"].dtype)


def _plain_sample(s):
    scores = s["scores"].float()
    rows, n = scores.shape
    ordered, order = torch.sort(scores, dim=1, descending=True, stable=True)
    t = s["temperature"].double().unsqueeze(1)
    far = ordered.double() - ordered[:, :1].double()
    w = torch.where(t > 0, torch.exp(far / torch.where(t > 0, t, torch.ones_like(t))), torch.zeros_like(far))
    w[:, :1] = 1                                    # the first of the order: all there is at temperature 0
    del far
    if s["top_k"] is not None:
        k = s["top_k"].unsqueeze(1)
        w *= (torch.arange(n, device=w.device) < torch.where(k > 0, k, n))
    if s["top_p"] is not None:
        run_ = w.cumsum(1)
        before = torch.cat((torch.zeros_like(run_[:, :1]), run_[:, :-1]), 1)
        p = s["top_p"].double().unsqueeze(1)
        keep = (before < p * run_[:, -1:]) | (p >= 1)
        keep[:, 0] = True
        w_kept = w * keep
        del run_, before, keep
    else:
        w_kept = w
    if s["min_p"] is not None:
        w_kept = w_kept * (w >= s["min_p"].double().unsqueeze(1))
    del w
    by_column = torch.zeros_like(w_kept).scatter_(1, order, w_kept)
    del w_kept, order
    run_ = by_column.cumsum(1)
    total = run_[:, -1:]
    last = n - 1 - (by_column > 0).flip(1).int().argmax(1, keepdim=True)
    label = torch.searchsorted(run_, s["uniform"].double() * total, right=True)
    label = torch.minimum(label, last)
    return {"labels": label, "probs": (by_column.gather(1, label) / total).float()}


_STUDENT_T = 2.0


def _plain_distil(s):
    x = s["scores"].float() / _STUDENT_T
    n = x.shape[1]
    there = (s["labels"] >= 0) & (s["labels"] < n)
    at = s["labels"].clamp(0, n - 1)
    t = torch.where(there, s["teacher"] / _STUDENT_T, float("-inf"))
    lse = torch.logsumexp(t, 1) if s["whole"] is None else s["whole"]
    log_p = t - lse.unsqueeze(1)
    p = log_p.exp()
    q = x - x.amax(1, keepdim=True)
    total = q.exp().sum(1, keepdim=True)
    q -= total.log()
    # the divergence is a small difference of large numbers: its terms in 64 bits
    terms = torch.where(there, p.double() * (log_p.double() - q.gather(1, at).double()), 0.0)
    loss = (terms.sum(1) * _STUDENT_T ** 2).float()
    g = q.exp_() * p.sum(1, keepdim=True)
    g.scatter_add_(1, at, torch.where(there, -p, torch.zeros_like(p)))
    g *= (_STUDENT_T * s["weight"]).unsqueeze(1)
    return {"loss": loss, "gradient": g.to(s["gradient"].dtype)}


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


def _workspace(what, *shape):
    lib, check = _lib()
    size = ctypes.c_int64()
    check(getattr(lib, what)(*shape, ctypes.byref(size)))
    return torch.empty(size.value, device="cuda", dtype=torch.uint8)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _own_quantise(s):
    lib, check = _lib()
    case, x, stream = s["case"], s["x"], _stream()
    n, d, group, scale = case["n"], case["d"], case["group"], _TYPES[case["scale"]][0]
    check(lib.ixa_op_group_quantise(_at(x), x.stride(0), _TYPES[case["type"]][0], n, d, group, scale, _at(s["codes"]),
                                    _at(s["scales"]), _at(s["zeros"]), stream))
    check(lib.ixa_op_group_dequantise(_at(s["codes"]), _at(s["scales"]), _at(s["zeros"]), group, scale, n, d, 0,
                                      _at(s["values"]), d, stream))
    out = {"values": s["values"], "scales": s["scales"]}
    if case["zeros"]:
        out["zeros"] = s["zeros"]
    return out


def _own_product(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ixa_op_group_product(_at(s["x"]), case["d"], _TYPES[case["type"]][0], case["m"], _at(s["codes"]), _at(s["scales"]),
                                   _at(s["zeros"]), case["group"], _TYPES[case["scale"]][0], case["n"], case["d"], 1.0,
                                   _at(s["bias"]), _TYPES[case["out"]][0], _at(s["out"]), case["n"], _at(s["work"]),
                                   s["work"].numel(), _stream()))
    return s["out"]


def _own_sample(s):
    lib, check = _lib()
    case = s["case"]
    check(lib.ixa_op_sample(_at(s["scores"]), case["n"], _TYPES[case["type"]][0], case["rows"], case["n"], _at(s["temperature"]),
                            _at(s["top_k"]), _at(s["top_p"]), _at(s["min_p"]), _at(s["uniform"]), case["draws"], _at(s["labels"]),
                            _at(s["probs"]), _at(s["work"]), s["work"].numel(), _stream()))
    return {"labels": s["labels"], "probs": s["probs"]}


def _own_distil(s):
    lib, check = _lib()
    case, x, stream = s["case"], s["scores"], _stream()
    rows, n, k, kind = case["rows"], case["n"], case["k"], _TYPES[case["type"]][0]
    given = (_at(x), x.stride(0), kind, rows, n, _at(s["labels"]), _at(s["teacher"]), k, _at(s["whole"]), _STUDENT_T)
    work_ = (_at(s["work"]), s["work"].numel())
    if case["apart"]:
        check(lib.ixa_op_distil_loss(*given, _at(s["loss"]), _at(s["stats"]), *work_, stream))
        check(lib.ixa_op_distil_gradient(*given, _at(s["stats"]), _at(s["weight"]), _at(s["gradient"]), n, stream))
    else:
        check(lib.ixa_op_distil_step(*given, _at(s["weight"]), _at(s["loss"]), _at(s["gradient"]), n, *work_, stream))
    return {"loss": s["loss"], "gradient": s["gradient"]}


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ----- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_quantise(case, s):
    d, group = case["d"], case["group"]
    scale_type = _TYPES[case["scale"]][1]
    values, scales, zeros = torch.empty(case["n"], d, device="cuda", dtype=torch.float64), [], []
    for k in range(0, d, group):
        x = s["x"][:, k:k + group].double()
        if case["zeros"]:
            low = torch.minimum(x.min(1).values, torch.zeros((), device="cuda", dtype=torch.float64))
            high = torch.maximum(x.max(1).values, torch.zeros((), device="cuda", dtype=torch.float64))
            scale = ((high - low) / 15).to(scale_type)
            zero = torch.where(scale > 0, torch.round(-low / scale.double()), torch.zeros_like(low)).clamp(0, 15)
            zeros.append(zero.to(torch.uint8))
            least, most = -zero, 15 - zero
        else:
            scale = (torch.linalg.vector_norm(x, float("inf"), 1) / 7).to(scale_type)
            least, most = torch.full_like(x[:, 0], -8.0), torch.full_like(x[:, 0], 7.0)
        scales.append(scale)
        number = torch.round(x / scale.double()[:, None])
        number = torch.where(scale[:, None] > 0, number, torch.zeros_like(number))
        number = torch.maximum(torch.minimum(number, most[:, None]), least[:, None])
        values[:, k:k + group] = number * scale.double()[:, None]
    out = {"values": values, "scales": torch.stack(scales, 1).double()}
    if case["zeros"]:
        out["zeros"] = torch.stack(zeros, 1)
    return out


def _exact_product(case, s):
    n, d, group = case["n"], case["d"], case["group"]
    x, out = s["x"].double(), torch.zeros(case["m"], n, device="cuda", dtype=torch.float64)
    for i in range(0, n, 65536):
        to = min(i + 65536, n)
        part = out[:, i:to]
        for g in range(_groups(case)):
            k = min(group, d - g * group)
            b = s["codes"][i:to, g * group // 2:(g + 1) * group // 2].int()
            number = torch.stack((b % 16, b // 16), 2).view(to - i, group)[:, :k].double()
            number = number - (8.0 if s["zeros"] is None else s["zeros"][i:to, g:g + 1].double())
            part += (x[:, g * group:g * group + k] @ number.t().contiguous()) * s["scales"][i:to, g].double()
        part += s["bias"][i:to].double()
    return out


def _exact_sample(case, s):
    labels = torch.empty(case["rows"], case["draws"], device="cuda", dtype=torch.int64)
    probs = torch.empty(case["rows"], case["draws"], device="cuda", dtype=torch.float64)
    n = case["n"]
    value = lambda name, r, default: default if s[name] is None else s[name][r].item()
    for r in range(case["rows"]):
        x = s["scores"][r].double()
        order = torch.argsort(-x, stable=True)
        temperature, top_k = value("temperature", r, 1.0), value("top_k", r, 0)
        count = n if top_k <= 0 else min(n, top_k)
        if temperature <= 0:
            count = 1
            temperature = 1.0
        mass = torch.exp((x[order[:count]] - x[order[0]]) / temperature)
        p = value("top_p", r, 1.0)
        if p < 1:
            mass = mass[:max(1, int((mass.cumsum(0) < p * mass.sum()).sum().item()) + 1)]
        mass = mass[mass >= value("min_p", r, 0.0)]
        kept, place = torch.sort(order[:len(mass)])
        mass = mass[place]
        run_ = mass.cumsum(0)
        at = torch.searchsorted(run_, s["uniform"][r].double() * run_[-1], right=True).clamp(max=len(mass) - 1)
        labels[r], probs[r] = kept[at], mass[at] / run_[-1]
    return {"labels": labels, "probs": probs}


def _exact_distil(case, s):
    n, T = case["n"], _STUDENT_T
    loss = torch.empty(case["rows"], device="cuda", dtype=torch.float64)
    gradient = torch.empty(case["rows"], n, device="cuda", dtype=torch.float64)
    for i in range(0, case["rows"], 512):
        r = slice(i, i + 512)
        log_q = torch.log_softmax(s["scores"][r].double() / T, 1)
        there = s["labels"][r] >= 0
        t = (s["teacher"][r].double() / T).masked_fill(~there, float("-inf"))
        log_p = torch.log_softmax(t, 1) if s["whole"] is None else t - s["whole"][r].double()[:, None]
        dense = torch.zeros_like(log_q).scatter_add_(1, s["labels"][r].clamp(min=0), torch.where(there, log_p.exp(), 0.0))
        kl = torch.where(there, log_p.exp() * (log_p - log_q.gather(1, s["labels"][r].clamp(min=0))), 0.0)
        loss[r] = T * T * kl.sum(1)
        gradient[r] = (dense.sum(1, keepdim=True) * log_q.exp() - dense) * (T * s["weight"][r].double())[:, None]
    return {"loss": loss, "gradient": gradient}


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
