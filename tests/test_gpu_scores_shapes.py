"""GPU tests of the shapes of kernels on scores that rows of other sizes choose: distillation of rows in registers, draws by the
largest workgroups, and 4-bit rows read back past the caches."""
import numpy as np
import pytest

import group_reference as ref
import test_gpu_distil as distil
import test_gpu_sample as sample
from test_gpu_group import TYPES, Store, as64, at, lib, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,rows,n,k", [("f16", 2100, 10_001, 20), ("f16", 1100, 9003, 20), ("f16", 300, 30_000, 20), ("bf16", 300, 40_001, 20),
                                           ("f32", 300, 20_003, 20), ("f32", 2200, 8000, 20), ("f32", 1030, 9000, 20), ("bf16", 2100, 8200, 256),
                                           ("f16", 260, 65_537, 300)])
def test_distillation_of_rows_in_registers(lib, kind, rows, n, k):  # noqa: F811
    x, labels, teacher = distil.task(11, n, k, n)
    x[1] = -np.inf
    x[3, n // 2], x[4, n - 1] = np.nan, np.inf
    x[5, 1:] = -np.inf
    labels[6] = -1
    labels[7] = n // 3
    first = distil.rows_of(x, kind)
    of = torch.arange(rows, device="cuda") % 11
    dev, dl = first[of], torch.from_numpy(labels).cuda()[of].contiguous()
    dt = torch.from_numpy(teacher.astype(np.float32)).cuda()[of].contiguous()
    weight = (torch.arange(rows, device="cuda") % 7 + 0.5).float()
    out = torch.full((rows + 1, n), 5.0, dtype=dev.dtype, device="cuda")
    value = distil.step(lib, dev, kind, dl, dt, None, 1.5, weight, out)
    some = list(range(11)) + list(range(rows - 11, rows))
    distil.compare(kind, 1.5, as64(dev[some]), labels[of.cpu().numpy()[some]], as64(dt[some]), None, as64(weight[some]), as64(value[some]),
                   as64(out[some]))
    assert value[rows] == 9 and (out[rows] == 5).all() and torch.equal(value[:rows].nan_to_num(7.0), value[:11][of].nan_to_num(7.0))
    both = distil.step(lib, dev, kind, dl, dt, None, 1.5, weight, dev)
    assert torch.equal(both.nan_to_num(7.0), value.nan_to_num(7.0)) and torch.equal(dev.nan_to_num(7.0), out[:rows].nan_to_num(7.0))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(4, 5), (4, 300), (200, 20_000), (4, 30_000)])
def test_rows_without_an_entry_have_no_loss_whatever_is_in_them(lib, rows, n, kind):  # noqa: F811
    x, labels, teacher = distil.task(4, n, 3, n)
    x[0, n // 2], x[1, 0], x[2] = np.nan, np.inf, np.nan
    labels[:] = -1
    of = torch.arange(rows, device="cuda") % 4
    dev, dl = distil.rows_of(x, kind)[of], torch.from_numpy(labels).cuda()[of].contiguous()
    dt = torch.from_numpy(teacher.astype(np.float32)).cuda()[of].contiguous()
    out = torch.full((rows, n), 5.0, dtype=dev.dtype, device="cuda")
    assert (distil.step(lib, dev, kind, dl, dt, None, 1.0, None, out)[:rows] == 0).all() and (out == 0).all()
    value, stats = distil.loss(lib, dev, kind, dl, dt, None, 1.0)
    out.fill_(5)
    distil.gradient(lib, dev, kind, dl, dt, None, 1.0, stats, None, out)
    assert (value[:rows] == 0).all() and (out == 0).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=5000, top_p=0.7)], ids=str)
@pytest.mark.parametrize("rows,n", [(2, 40_000), (150, 33_001)])
def test_draws_of_a_thousand_threads(lib, rows, n, kind, filters):  # noqa: F811
    x = sample.scores(2, n, n, flat=0.5)
    sample.check(lib, np.tile(x, (rows // 2, 1)), kind, draws=8, **filters)


@pytest.mark.parametrize("group,kind", [(32, "f16"), (64, "f16"), (128, "f16"), (32, "bf16"), (64, "bf16"), (128, "bf16"), (32, "f32"), (64, "f32"),
                                        (128, "f32")])
def test_large_results_go_past_the_caches(lib, group, kind):  # noqa: F811
    n, d = 250_000 if kind == "f32" else 500_000, 151
    store = Store(n, d, group, "bf16", True)
    size, gen = n * store.ng, torch.Generator(device="cuda").manual_seed(group)
    store.codes[:size * group // 2] = torch.randint(0, 256, (size * group // 2,), dtype=torch.uint8, device="cuda", generator=gen)
    store.scales[:size] = torch.rand(size, device="cuda", generator=gen).to(torch.bfloat16)
    store.zeros[:size] = torch.randint(0, 16, (size,), dtype=torch.uint8, device="cuda", generator=gen)
    out = torch.full((n + 1, d), 9.0, dtype=TYPES[kind][1], device="cuda")
    lib[1](lib[0].ixa_op_group_dequantise(at(store.codes), at(store.scales), at(store.zeros), group, 2, n, d, TYPES[kind][0], at(out), d, None))
    assert (out[n] == 9).all()
    pick = torch.cat((torch.arange(300), torch.randint(0, n, (2000,)), torch.arange(n - 300, n))).cuda()
    part = lambda t, per: t[:n * per].view(n, per)[pick].cpu()
    code = ref.unpack(part(store.codes, store.ng * group // 2).numpy(), group)
    v = ref.values(code, part(store.scales, store.ng).double().numpy(), part(store.zeros, store.ng).numpy(), d)
    assert np.array_equal(as64(out[:n][pick]), ref.round_to_type(v, TYPES[kind][0]))
