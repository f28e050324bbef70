"""The feed-forward sublayer's calls at the ends of their ranges, without a GPU."""
from __future__ import annotations

import pytest

from tiler_amd import _lib as L
from tiler_amd.realize import realize

RE = L.PERMITS_REASSOCIATION
ALL_NORM = L.NORM_WEIGHT | L.NORM_DX | L.NORM_DW | L.NORM_DB


@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
@pytest.mark.parametrize("rows", [0, 1, 5, 1 << 21])
@pytest.mark.parametrize("extent", [(1 << 26) + 70, (1 << 28) - 64, (1 << 28) - 63, 1 << 28, (1 << 32) - 256, (1 << 32) - 1])
def test_norm_gradients_fit_a_launch(dtype, rows, extent):
    """The runtime takes fewer than 2^32 work items along an axis; 2^32 - 1
    elements a row are in the planner's range."""
    for variant in (ALL_NORM, L.NORM_DW, L.NORM_DB):
        rz = realize(L.PROGRAM_LAYER_NORM_BACKWARD, (rows, extent), dtype=dtype, variant=variant, permissions=RE)
        assert rz.dispatches
        for d in rz.dispatches:
            assert all(g * b < 1 << 32 for g, b in zip(d.grid, d.block)), (d.symbol, d.grid, d.block)
