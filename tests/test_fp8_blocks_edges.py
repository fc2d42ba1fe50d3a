"""Edges of the e8m0 block-scaled product's kernels, each with the kernel that
must have run, so that a change of the choice cannot leave an edge untested."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import kernels  # noqa: E402
from tests.test_fp8_blocks import Product  # noqa: E402

# (lengths, n, k), kernel, token rows of its tile.  A pair's last output tile
# (256) may end inside its first CTA's 128 weight rows or its second's, or be whole.
EDGES = [
    (([1500, 900], 4104, 272), "tcgen05_tma_pair", 224),  # 8 outputs in the last tile
    (([1500, 900], 4216, 272), "tcgen05_tma_pair", 224),  # 120
    (([4000], 2184, 1040), "tcgen05_tma_pair", 224),  # 136
    (([1500, 900], 4088, 272), "tcgen05_tma_pair", 224),  # 248
    (([1999], 4088, 144), "tcgen05_tma_pair", 224),
    (([700, 0, 1100], 2312, 2064), "tcgen05_tma_pair", 224),
    (([130, 113, 225, 224, 1, 500], 4232, 656), "tcgen05_tma_pair", 224),  # row blocks of every width
    (([225] * 9, 2056, 400), "tcgen05_tma_pair", 224),
    (([1999], 2248, 1040), "tcgen05_tma", 128),
    (([100, 0, 1, 129], 264, 656), "tcgen05_tma", 128),
    (([20], 264, 2064), "tcgen05_tma", 128),  # with the rows behind: 25
    (([10], 264, 2064), "tcgen05_tma", 64),
    (([40, 0, 1, 3] * 8, 2056, 400), "tcgen05_tma", 64),
    (([9, 3], 24, 400), "tcgen05_tma", 64),  # with the rows behind: 17
    (([4, 3], 24, 400), "warp_mma", 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,path,tile_rows", EDGES, ids=lambda v: f"{sum(v[0])}rows{len(v[0])}e{v[1]}x{v[2]}"
                         if isinstance(v, tuple) else str(v))
def test_last_output_tiles(shape, path, tile_rows):
    product = Product(*shape, seed=6, tail=5, pad=16)
    wide = torch.full((product.rows, product.n + 24), 3.25, device="cuda", dtype=torch.bfloat16)
    product.run(out=wide[:, :product.n])
    info = kernels.last_block_scaled_info()
    kernels.check_device_errors()
    assert (info["path"], info["tile_m"]) == (path, tile_rows)
    product.check(wide[:, :product.n])
    assert bool((wide[:, product.n:] == 3.25).all()), "padding written"
    assert bool((wide[product.used:] == 3.25).all()), "rows behind the last segment written"


@pytest.mark.gpu
def test_scales_of_a_partial_last_tile():
    """The last tile's outputs take the last 128-block's scales, the row before its own."""
    product = Product([1500, 900], 4216, 400, seed=7)
    bytes_b = product.sb.view(torch.uint8)
    bytes_b.fill_(127)
    bytes_b[:, -1] = 131
    bytes_b[1, -2] = 120
    product.check(product.run())
    assert kernels.last_block_scaled_info()["path"] == "tcgen05_tma_pair"
    kernels.check_device_errors()
