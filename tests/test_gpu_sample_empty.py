"""GPU tests of draws from rows that have no columns at all."""
import numpy as np
import pytest

from test_gpu_sample import as_setting, call, lib, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                                     dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.01)], ids=str)
@pytest.mark.parametrize("rows,draws", [(1, 1), (7, 5), (300, 40)])
def test_rows_of_no_columns(lib, rows, draws, kind, filters):  # noqa: F811
    x = torch.empty(rows, 0, dtype={"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind], device="cuda")
    uniform = torch.from_numpy(np.random.default_rng(rows).random((rows, draws)).astype(np.float32)).cuda()
    s = {k: as_setting(v, rows, torch.int32 if k == "top_k" else torch.float32) for k, v in filters.items()}
    labels, probs, work = call(lib, x, kind, uniform, **s)
    torch.cuda.synchronize()
    assert (labels[:rows] == -1).all() and (probs[:rows] == 0).all()
    assert (labels[rows] == -7).all() and (probs[rows] == 9).all() and (work[-64:] == 0x5a).all()
