"""Registers of the kernels for 4-bit rows with group scales, draws and distillation."""
import re

from test_kernel_resources import kernels  # noqa: F401


def test_products_with_groups_and_distillation_do_not_spill(kernels):  # noqa: F811
    mine = {n: v for n, v in kernels.items() if re.search("group_(quantise|read|stream|tile|pieces|tiny)_kernel|distil_[a-z]+_kernel", n)}
    assert all(spilled == 0 for _, spilled in mine.values()), {n: v for n, v in mine.items() if v[1]}
    # two workgroups of a tile share a CU
    tile = {n: v for n, v in mine.items() if "group_tile" in n}
    assert len(tile) == 24 and all(r <= 256 for r, _ in tile.values())
    # a row in registers: sixteen wavefronts of a CU
    rows = {n: v for n, v in mine.items() if "distil_row" in n}
    assert len(rows) == 18 and all(r <= 128 for r, _ in rows.values())


def test_draws_leave_room_for_their_wavefronts(kernels):  # noqa: F811
    mine = {n: v for n, v in kernels.items() if re.search("sample_(part|join)?_?kernel", n)}
    assert len(mine) == 15
    assert all(r <= (168 if "Li256E" in n else 128) and spilled <= 24 for n, (r, spilled) in mine.items()), mine
