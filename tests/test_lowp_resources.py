"""Registers of the low-precision kernels: none of them spills, since a reload among loads in flight waits for all of these."""
import re

from test_kernel_resources import kernels  # noqa: F401


def test_low_precision_kernels_do_not_spill(kernels):  # noqa: F811
    mine = {n: v for n, v in kernels.items() if re.search("row_quantise_kernel|read_codes_kernel|mx_(stream|tile|wide)_kernel", n)}
    assert all(spilled == 0 for _, spilled in mine.values()), {n: v for n, v in mine.items() if v[1]}
    # one wavefront per SIMD for the wide tiles, two and more for the others
    wide = {n: v for n, v in mine.items() if "mx_wide" in n}
    assert len(wide) == 12 and all(r <= 512 for r, _ in wide.values())
    tile = {n: v for n, v in mine.items() if "mx_tile" in n or "mx_stream" in n}
    assert len(tile) == 15 + 42 and all(r <= 256 for r, _ in tile.values())
