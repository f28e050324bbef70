"""The feed-forward sublayer without a GPU: what the recognizer realizes, what
it refuses, and the workspace queries."""
from __future__ import annotations

import ctypes

import pytest

from tiler_amd import _lib as L
from tiler_amd.realize import realize
from tiler_amd.runtime import Refusal

RE = L.PERMITS_REASSOCIATION
ALL_NORM = L.NORM_WEIGHT | L.NORM_DX | L.NORM_DW | L.NORM_DB


def region(program, extents, dtype=L.BF16, variant=0, permissions=RE, **kw):
    return realize(program, extents, dtype=dtype, variant=variant, permissions=permissions, flags=L.REGION_ALIGNED16, **kw)


def roles(rz):
    return [role for role, _ in rz.slots]


@pytest.mark.parametrize("program,extents,variant,inputs,outputs", [
    (L.PROGRAM_LAYER_NORM, (5, 100), 0, 1, 1),
    (L.PROGRAM_LAYER_NORM, (5, 100), L.NORM_WEIGHT | L.NORM_BIAS | L.NORM_STATISTICS, 3, 3),
    (L.PROGRAM_LAYER_NORM_BACKWARD, (5, 100), ALL_NORM, 5, 3),
    (L.PROGRAM_LAYER_NORM_BACKWARD, (5, 100), L.NORM_DX, 4, 1),
    (L.PROGRAM_GATED_CONTRACTION, (5, 64, 32), L.GATED_KEEP, 3, 3),
    (L.PROGRAM_GATED_CONTRACTION, (5, 64, 32), 0, 3, 1),
    (L.PROGRAM_GATED_CONTRACTION_BACKWARD, (5, 64, 32), L.GATED_DX | L.GATED_DW, 6, 3),
    (L.PROGRAM_QUANTIZE_ROWS_I8, (5, 64), 0, 1, 2),
    (L.PROGRAM_CONTRACTION_I8, (5, 64, 32), 0, 4, 1),
])
def test_slots(program, extents, variant, inputs, outputs):
    scalars = (0x3727C5AC, 0) if program == L.PROGRAM_LAYER_NORM else (0, 0)
    rz = region(program, extents, variant=variant, scalars=scalars)
    r = roles(rz)
    assert r.count(L.SLOT_INPUT) == inputs and r.count(L.SLOT_OUTPUT) == outputs
    assert rz.symbols


@pytest.mark.parametrize("kw,status", [
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0, 0)), L.REFUSE_INVALID_ARGUMENT),  # eps 0
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0x7F800000, 0)), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0x3727C5AC, 0), variant=64), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0x3727C5AC, 0), dtype=2), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0x3727C5AC, 0), permissions=0), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 1 << 32), scalars=(0x3727C5AC, 0)), L.REFUSE_CAPACITY),
    (dict(program=L.PROGRAM_LAYER_NORM, extents=(5, 100), scalars=(0x3727C5AC, 0),
          input_subnormals=L.SUBNORMALS_FLUSH_SIGN), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_LAYER_NORM_BACKWARD, extents=(5, 100), variant=L.NORM_BIAS), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_LAYER_NORM_BACKWARD, extents=(5, 100), variant=ALL_NORM, permissions=0), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_GATED_CONTRACTION, extents=(5, 64, 0)), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_GATED_CONTRACTION, extents=(5, 64, 32), dtype=L.F32), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_GATED_CONTRACTION, extents=(5, 64, 32), variant=2), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_GATED_CONTRACTION, extents=(5, 64, 32), permissions=0), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_GATED_CONTRACTION, extents=(5, 1 << 31, 32)), L.REFUSE_CAPACITY),
    (dict(program=L.PROGRAM_GATED_CONTRACTION_BACKWARD, extents=(5, 64, 32), variant=1), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_QUANTIZE_ROWS_I8, extents=(5, 64), variant=1), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_QUANTIZE_ROWS_I8, extents=(5, 64), dtype=2), L.REFUSE_UNSUPPORTED),
    (dict(program=L.PROGRAM_CONTRACTION_I8, extents=(5, 64, 131072)), L.REFUSE_CAPACITY),
    (dict(program=L.PROGRAM_CONTRACTION_I8, extents=(5, 64, 0)), L.REFUSE_INVALID_ARGUMENT),
    (dict(program=L.PROGRAM_CONTRACTION_I8, extents=(5, 64, 32), dtype=2), L.REFUSE_UNSUPPORTED),
])
def test_refusals(kw, status):
    kw = dict(kw)
    with pytest.raises(Refusal) as e:
        region(kw.pop("program"), kw.pop("extents"), **kw)
    assert e.value.status == status, str(e.value)


def query(name, *args):
    n = ctypes.c_uint64(1)
    st = getattr(L.lib(), name)(None, *args, ctypes.byref(n))
    return st, n.value


def test_workspace_queries():
    st, n = query("tiler_hip_layer_norm_backward_workspace", L.BF16, 8192, 4096)
    assert st == L.OK and 0 < n < 1 << 28
    assert query("tiler_hip_layer_norm_backward_workspace", L.BF16, 0, 0) == (L.OK, 0)
    assert query("tiler_hip_layer_norm_backward_workspace", 2, 1, 1)[0] == L.REFUSE_UNSUPPORTED
    st, n = query("tiler_hip_gated_contract_bf16_backward_workspace", 100, 130, 64)
    assert st == L.OK and n >= 2 * 100 * 130 * 2
    assert query("tiler_hip_gated_contract_bf16_backward_workspace", 100, 130, 0)[0] == L.REFUSE_INVALID_ARGUMENT
    assert L.lib().tiler_hip_gated_contract_bf16_backward_workspace(None, 1, 1, 1, None) == L.REFUSE_INVALID_ARGUMENT


def test_empty_requests_launch_nothing_or_zeros():
    eps = (0x3727C5AC, 0)
    assert region(L.PROGRAM_LAYER_NORM, (0, 100), scalars=eps).symbols == []
    assert region(L.PROGRAM_LAYER_NORM, (100, 0), scalars=eps).symbols == []
    assert region(L.PROGRAM_LAYER_NORM_BACKWARD, (100, 0), variant=ALL_NORM).symbols == []
    # no rows: the weights' gradients are still written (zeros)
    assert len(region(L.PROGRAM_LAYER_NORM_BACKWARD, (0, 100), variant=ALL_NORM).symbols) == 1
    assert region(L.PROGRAM_GATED_CONTRACTION, (0, 64, 32)).symbols == []
    assert len(region(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (0, 64, 32), variant=L.GATED_DX | L.GATED_DW).symbols) == 1
    assert len(region(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (5, 0, 32), variant=L.GATED_DX | L.GATED_DW).symbols) == 1
    assert region(L.PROGRAM_QUANTIZE_ROWS_I8, (0, 64)).symbols == []
    assert region(L.PROGRAM_CONTRACTION_I8, (5, 0, 32)).symbols == []


def test_host_functions_refuse_before_any_device_work():
    """Shapes and dtypes are checked on the host: no context is ever asked for."""
    import numpy as np
    from tiler_amd import families as f
    x, w, i8, s = np.zeros((3, 8), np.uint16), np.zeros((5, 8), np.uint16), np.zeros((3, 8), np.int8), np.ones(3, np.float32)
    mid = np.zeros((3, 5), np.uint16)
    for call in (lambda: f.layer_norm(np.zeros((3, 8)), ctx=0), lambda: f.layer_norm(x[0], ctx=0),
                 lambda: f.layer_norm(x, weights=np.zeros(7, np.uint16), ctx=0),
                 lambda: f.layer_norm(x, bias=np.zeros(8, np.float32), ctx=0),
                 lambda: f.layer_norm_backward(x[:2], x, None, s, s, ctx=0),
                 lambda: f.layer_norm_backward(x, x, None, s[:2], s, ctx=0),
                 lambda: f.gated_contract_bf16(x, w, w[:4], ctx=0), lambda: f.gated_contract_bf16(x, w[:, :7], w, ctx=0),
                 lambda: f.gated_contract_bf16(x.astype(np.float32), w, w, ctx=0),
                 lambda: f.gated_contract_bf16_backward(x, w, w, mid, mid[:2], mid, ctx=0),
                 lambda: f.quantize_rows_i8(i8, ctx=0), lambda: f.contract_i8(i8, i8[:, :7], s, s, ctx=0),
                 lambda: f.contract_i8(i8, i8, s, s[:2], ctx=0), lambda: f.contract_i8(i8, i8, s, s, np.float64, ctx=0)):
        with pytest.raises(Refusal):
            call()
