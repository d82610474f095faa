"""From a model's hidden states to the nearest stored rows, in 4 bits.

The last step of an embedding model (residual addition and root-mean-square norm) writes its rows straight into a store of
4-bit codes; queries go the same way into 8-bit codes; the products of both on the matrix cores are the squared distances from
which the nearest rows are selected.  Nothing but codes, scales and norms is kept of the rows: 4.25 bits per element.

    python examples/low_precision_search.py --rows 200000 --queries 1000 --dims 768 --k 10

prints, for synthetic hidden states, the time of each step, the size of the store, how well its rows are kept, and how many of
the exact nearest rows were found.
"""
import argparse
import ctypes
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from indexsdk_amd import _capi  # noqa: E402

BF16, F32 = 2, 0
MXFP8, MXFP4 = 1, 2
L2 = 1


def at(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


class Rows:
    """Codes, scales and squared norms of n rows of d elements."""

    def __init__(self, n, d, fmt):
        row, per = ctypes.c_int64(), ctypes.c_int64()
        _capi.check(_capi.load().ixa_code_bytes(fmt, d, ctypes.byref(row), ctypes.byref(per)))
        self.n, self.d, self.fmt = n, d, fmt
        self.codes = torch.empty(n * row.value, dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(n * per.value, dtype=torch.uint8, device="cuda")
        self.norms = torch.empty(n, device="cuda")

    def bytes(self):
        return self.codes.numel() + self.scales.numel() + 4 * self.n

    def fill(self, hidden, residual, weight, eps=1e-6):
        """hidden + residual, normalised and weighted; hidden holds the sum afterwards, as the next layer would want it."""
        _capi.check(_capi.load().ixa_op_rms_norm_quantise(
            at(hidden), self.d, at(residual), self.d, at(weight), BF16, self.n, self.d, eps, at(hidden), self.d, self.fmt, 0.0,
            at(self.codes), at(self.scales), at(self.norms), stream()))

    def read(self):
        out = torch.empty(self.n, self.d, device="cuda")
        _capi.check(_capi.load().ixa_op_dequantise(at(self.codes), at(self.scales), self.fmt, self.n, self.d, F32, at(out),
                                                   self.d, stream()))
        return out


def quantised(x, fmt):
    """fp32 rows that are there already, as codes."""
    rows = Rows(x.shape[0], x.shape[1], fmt)
    _capi.check(_capi.load().ixa_op_quantise(at(x), x.shape[1], F32, rows.n, rows.d, fmt, 0.0, at(rows.codes),
                                             at(rows.scales), at(rows.norms), stream()))
    return rows


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def nearest(queries, store, k, page):
    """Distances and positions of the k nearest stored rows, `page` queries at a time."""
    lib = _capi.load()
    ld = (store.n + 15) // 16 * 16            # rows of scores that start on 64 bytes
    scores = torch.empty(min(page, queries.n), ld, device="cuda")
    dist = torch.empty(queries.n, k, device="cuda")
    label = torch.empty(queries.n, k, dtype=torch.int64, device="cuda")
    row, per = queries.codes.numel() // queries.n, queries.scales.numel() // queries.n
    for i in range(0, queries.n, page):
        m = min(page, queries.n - i)
        _capi.check(lib.ixa_op_mx_product(
            at(queries.codes[i * row:]), at(queries.scales[i * per:]), queries.fmt, m, at(store.codes), at(store.scales), store.n,
            store.d, L2, at(queries.norms[i:]), at(store.norms), F32, at(scores), ld, stream()))
        _capi.check(lib.ixa_op_topk_flat_fp32(at(scores), m, store.n, ld, k, 1, at(dist[i:]), at(label[i:]), stream()))
    return dist, label


def timed(what, step):
    step()                                    # the first call loads the kernels
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    result = step()
    end.record()
    end.synchronize()
    print(f"{what:<48} {begin.elapsed_time(end) * 1e3:10.1f} us")
    return result


def run(n=200_000, m=1000, d=768, k=10, page=1024, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    weight = (1 + 0.1 * draw(d)).bfloat16()
    hidden, residual = draw(n, d).bfloat16(), draw(n, d).bfloat16()
    summed = hidden.float() + residual.float()
    rows = summed * torch.rsqrt(summed.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.float()
    picked = torch.randint(n, (m,), generator=gen, device="cuda")
    asked = rows[picked] + 0.6 * draw(m, d)   # noisy versions of stored rows
    del summed

    store = Rows(n, d, MXFP4)
    first = hidden.clone()

    def write():
        hidden.copy_(first)
        store.fill(hidden, residual, weight)
    timed(f"{n} x {d} rows, normalised into 4 bits (and a copy)", write)
    queries = timed(f"{m} queries into 8 bits", lambda: quantised(asked, MXFP8))
    _, found = timed(f"{k} nearest of {n} rows, {m} queries", lambda: nearest(queries, store, k, page))

    kept = store.read()
    error = ((kept - rows).pow(2).sum() / rows.pow(2).sum()).sqrt().item()
    exact = torch.cat([torch.cdist(q, rows, compute_mode="use_mm_for_euclid_dist").topk(k, largest=False).indices
                       for q in asked.split(256)])
    itself = (found[:, 0] == picked).float().mean().item()
    recall = (found.unsqueeze(2) == exact.unsqueeze(1)).any(2).float().mean().item()
    print(f"store: {store.bytes() / 1e6:.1f} MB instead of {n * d * 2 / 1e6:.1f} in bfloat16; rows kept to {error:.3f} of their norm")
    print(f"the row a query was made from comes first: {itself:.4f}; of the {k} exact nearest found: {recall:.4f}")
    return {"itself": itself, "recall": recall, "error": error, "bytes": store.bytes()}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--rows", type=int, default=200_000)
    parser.add_argument("--queries", type=int, default=1000)
    parser.add_argument("--dims", type=int, default=768)
    parser.add_argument("--k", type=int, default=10)
    parser.add_argument("--page", type=int, default=1024, help="queries scored at a time")
    a = parser.parse_args()
    run(a.rows, a.queries, a.dims, a.k, a.page)
