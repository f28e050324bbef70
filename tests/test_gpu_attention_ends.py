"""The attention sublayer's calls at their ends: heads of every register form."""
from __future__ import annotations

import pytest

import test_gpu_norm_rotate as rotation
from test_gpu_norm_rotate import Case, backward, forward
from tiler_amd import _lib as L

pytestmark = pytest.mark.gpu

# heads, kv_heads, dim, rotary: 32 lanes of bf16 and 64 of f32 to a head
WIDE_FORMS = [(2, 1, 320, 320), (2, 1, 512, 512), (3, 1, 264, 32), (5, 2, 384, 64)]


@pytest.mark.parametrize("dtype", [L.BF16, L.F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary", WIDE_FORMS)
def test_wide_heads(ctx, heads, kv_heads, dim, rotary, pairing, dtype):
    for tokens, norm, gap in ((1, True, 0), (13, True, 3), (6, False, 0), (1100, True, 0)):
        forward(ctx, Case(tokens, heads, kv_heads, dim, rotary, pairing, norm, dtype, seed=tokens + dim, gap=gap))
        backward(ctx, Case(tokens, heads, kv_heads, dim, rotary, pairing, norm, dtype, seed=tokens + dim, gap=gap))


@pytest.mark.parametrize("layout", rotation.LAYOUTS)
@pytest.mark.parametrize("heads,kv_heads,dim,rotary", WIDE_FORMS[::2])
def test_store_of_wide_heads(ctx, heads, kv_heads, dim, rotary, layout):
    rotation.test_store(ctx, heads, kv_heads, dim, rotary, 5, layout)
