"""The feed-forward sublayer's calls at the ends of their ranges, without a GPU."""
from __future__ import annotations

import pytest

from tiler_amd import _lib as L
from tiler_amd.realize import prepare_route, realize
from tiler_amd.runtime import Refusal

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


@pytest.mark.parametrize("program,extents,variant", [
    (L.PROGRAM_LAYER_NORM_BACKWARD, (600, 512), ALL_NORM),
    (L.PROGRAM_LAYER_NORM_BACKWARD, (600, 40000), ALL_NORM),
    (L.PROGRAM_GATED_CONTRACTION_BACKWARD, (300, 520, 264), L.GATED_DX | L.GATED_DW),
    (L.PROGRAM_GATED_CONTRACTION_BACKWARD, (300, 520, 333), L.GATED_DX | L.GATED_DW)])
def test_routed_scratch_is_aligned(program, extents, variant):
    """Operands at any address; a caller's scratch from a 16-byte boundary, as the
    direct call's workspace.  Refused before the context is asked for anything."""
    rz = realize(program, extents, dtype=L.BF16, variant=variant, permissions=RE, flags=0)
    assert rz.alignment == 1
    scratch = [i for i, (role, _) in enumerate(rz.slots) if role == L.SLOT_SCRATCH]
    assert scratch
    for slot in scratch:
        for off in (2, 8):
            storage = [(4096 if i in scratch else 4098) + (off if i == slot else 0) for i in range(len(rz.slots))]
            with pytest.raises(Refusal) as e:
                prepare_route(None, rz, storage)
            assert e.value.status == L.REFUSE_BINDING_MISMATCH and f"slot {slot} " in str(e.value)


def test_empty_rows():
    """No element, no mean and no scale: refused where one is asked for."""
    eps = (0x3727C5AC, 0)
    for rows in (1, 100):
        for program, kw in ((L.PROGRAM_LAYER_NORM, dict(variant=L.NORM_STATISTICS, scalars=eps)),
                            (L.PROGRAM_LAYER_NORM, dict(variant=L.NORM_WEIGHT | L.NORM_BIAS | L.NORM_STATISTICS, scalars=eps)),
                            (L.PROGRAM_QUANTIZE_ROWS_I8, {})):
            with pytest.raises(Refusal) as e:
                realize(program, (rows, 0), dtype=L.BF16, permissions=RE, **kw)
            assert e.value.status == L.REFUSE_INVALID_ARGUMENT
            assert realize(program, (0, 0), dtype=L.BF16, permissions=RE, **kw).symbols == []
    assert realize(L.PROGRAM_LAYER_NORM, (100, 0), dtype=L.BF16, permissions=RE, scalars=eps).symbols == []


@pytest.mark.parametrize("m,n,k", [(5, 64, 64), (300, 520, 264), (300, 520, 333), (4096, 14336, 4096), (4096, 14336, 4095)])
def test_the_workgroups_that_form_the_middle_gradients(m, n, k):
    """One launch forms dG and dU and copies operands: the kernel is told how many of
    its workgroups do the former (behind six addresses and m, n, k), and the others
    are those of the copies."""
    rz = realize(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (m, n, k), dtype=L.BF16, variant=L.GATED_DX | L.GATED_DW, permissions=RE)
    d, e = rz.dispatches[0], rz.raw.entries[0]
    told = [int.from_bytes(bytes(e.kernargs[o:o + 4]), "little") for o in (48, 52, 56, 60)]
    groups = lambda pieces: min(-(-pieces // 256), 8192)
    assert d.symbol == "tiler_gated_bf16_grad" and told == [m, n, k, groups(m * (-(-n // 64) * 8))]
    assert d.grid[0] - told[3] == (groups((m + 2 * n) * -(-k // 8)) if k % 8 else 0)
