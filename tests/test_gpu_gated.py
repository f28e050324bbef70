"""The gated product and its gradients on the device."""
from __future__ import annotations

import numpy as np
import pytest

import feed_forward_reference as ref
import oracle
from tiler_amd import _lib as L
from tiler_amd.realize import realize
from test_gpu_layer_norm import Buffers, within

pytestmark = pytest.mark.gpu

BF = np.uint16


@pytest.fixture
def mem(ctx):
    m = Buffers(ctx)
    yield m
    m.free()


def bf(values):
    return ref.store("bf16", values)


def w64(stored):
    return ref.wide("bf16", stored)


def forward(ctx, mem, x, wg, wu, keep, shift=0, stream=None):
    (m, k), n = x.shape, wg.shape[0]
    h = mem.out(BF, m * n, shift)
    gate = mem.out(BF, m * n, shift) if keep else None
    up = mem.out(BF, m * n, shift) if keep else None
    ctx.gated_contract_bf16(mem.put(x, shift), mem.put(wg, shift), mem.put(wu, shift), m, n, k, h, gate=gate, up=up,
                            stream=stream)
    ctx.synchronize()
    return [mem.get(v, BF, (m, n)) for v in ((h, gate, up) if keep else (h,))]


def backward(ctx, mem, x, wg, wu, gate, up, dh, shift=0, want=(True, True), workspace="given", stream=None):
    (m, k), n = x.shape, wg.shape[0]
    dx = mem.out(BF, m * k, shift) if want[0] else None
    dwg, dwu = (mem.out(BF, n * k, shift), mem.out(BF, n * k, shift)) if want[1] else (None, None)
    ws, nbytes = None, 0
    if workspace == "given":
        nbytes = ctx.gated_contract_bf16_backward_workspace(m, n, k)
        ws = mem.out(np.uint8, max(nbytes, 1))
    ctx.gated_contract_bf16_backward(*(mem.put(v, shift) for v in (x, wg, wu, gate, up, dh)), m, n, k, dx, dwg, dwu,
                                     workspace=ws, workspace_bytes=nbytes, stream=stream)
    ctx.synchronize()
    if ws is not None:
        mem.get(ws, np.uint8, (max(nbytes, 1),))
    return [None if v is None else mem.get(v, BF, s) for v, s in ((dx, (m, k)), (dwg, (n, k)), (dwu, (n, k)))]


# (m, n, k): a token, decode batches, prompts, ragged and odd, tiles exact
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 520), (2, 37, 11), (5, 128, 4096), (16, 256, 512), (17, 72, 136),
          (48, 520, 1024), (64, 96, 200), (65, 96, 512), (100, 264, 72), (128, 128, 64), (129, 127, 65),
          (200, 512, 1000), (256, 256, 128), (257, 200, 264), (300, 1365, 509), (520, 392, 328), (512, 1024, 256),
          (4104, 2056, 72), (520, 4104, 2312), (2056, 72, 8200)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(ctx, mem, m, n, k):
    rng = np.random.default_rng(m + n + k)
    x, wg, wu = bf(rng.standard_normal((m, k))), *(bf(rng.standard_normal((n, k)) * 2 / np.sqrt(k)) for _ in range(2))
    args = (w64(x), w64(wg), w64(wu))
    for shift in (0, 1, 4):
        got = forward(ctx, mem, x, wg, wu, keep=True, shift=shift)
        for g, v, e, what in zip(got, ref.gated(*args), ref.gated_bounds(*args), ("h", "gate", "up")):
            within(w64(g), v, e, (what, shift))
        alone, = forward(ctx, mem, x, wg, wu, keep=False, shift=shift)
        assert np.array_equal(alone, got[0])


def whole(rng, shape, top):
    return rng.integers(-top, top + 1, shape).astype(np.float64)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward_whole_numbers(ctx, mem, m, n, k):
    """G at least 20, where the sigmoid is 1 in binary32: h is G U, exactly
    summed, rounded once -- every index of every operand counts."""
    rng = np.random.default_rng(m * n + k)
    x, wg, wu = whole(rng, (m, k), 2), whole(rng, (n, k), 2), whole(rng, (n, k), 2)
    x[:, 0] = 1
    wg[:, 0] = 0
    low = (x @ wg.T).min()
    lift = 20 - low + (-(20 - low)) % 64
    wg[:, 0] = lift  # a multiple of 64 below 2^14: exact in bf16
    g, u = x @ wg.T, x @ wu.T
    assert (g >= 20).all() and lift < 16384
    got = forward(ctx, mem, bf(x), bf(wg), bf(wu), keep=True)
    for a, v in zip(got, (g * u, g, u)):
        assert np.array_equal(a, bf(v)), np.argwhere(a != bf(v))[:4]


# Every form of the product, shallower and deeper than the slices it keeps in LDS
FORMS = [("few1x1", 3, 24, 528), ("few2x1", 17, 2056, 1040), ("few4x1", 33, 2056, 1040), ("few4x2", 33, 4104, 1040),
         ("t64_d", 33, 4104, 528), ("t64_d", 3, 14344, 528), ("t96_d", 70, 8200, 1040), ("t128_d", 100, 8200, 528),
         ("t64_d", 3, 14344, 272), ("t96", 17, 24, 16), ("t96", 33, 20008, 1040), ("t128", 301, 8200, 16),
         ("t128", 100, 20008, 1040), ("t160_w", 400, 8200, 1040), ("t192_n", 130, 8200, 1040),
         ("t256_n", 200, 12008, 1040), ("t192", 520, 8200, 16), ("t192", 333, 12008, 1040), ("t256", 400, 14344, 80),
         ("t256", 400, 12008, 1040), ("g64", 70, 200, 333), ("g128", 300, 4099, 65)]


@pytest.mark.parametrize("form,m,n,k", FORMS)
def test_forward_forms(ctx, mem, form, m, n, k):
    rz = realize(L.PROGRAM_GATED_CONTRACTION, (m, n, k), dtype=L.BF16, permissions=L.PERMITS_REASSOCIATION,
                 flags=L.REGION_ALIGNED16)
    assert rz.symbols == ["tiler_gated_bf16_" + form]
    test_forward_whole_numbers(ctx, mem, m, n, k)


def operands(rng, m, n, k):
    x, wg, wu = bf(rng.standard_normal((m, k))), *(bf(rng.standard_normal((n, k)) / np.sqrt(k)) for _ in range(2))
    gate, up = bf(rng.standard_normal((m, n)) * 2), bf(rng.standard_normal((m, n)))
    return x, wg, wu, gate, up, bf(rng.standard_normal((m, n)))


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward(ctx, mem, m, n, k):
    rng = np.random.default_rng(m + 2 * n + k)
    a = operands(rng, m, n, k)
    wide = [w64(v) for v in a]
    want, bound = ref.gated_backward(*wide), ref.gated_backward_bounds(*wide)
    for shift in (0, 1):
        for g, v, e, what in zip(backward(ctx, mem, *a, shift=shift), want, bound, ("dx", "dwg", "dwu")):
            within(w64(g), v, e, (what, shift))


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward_whole_numbers(ctx, mem, m, n, k):
    """G = 32: the sigmoid is 1 in binary32, dG = dh U and dU = 32 dh are whole,
    and so are the sums: every bit of every gradient is checked."""
    rng = np.random.default_rng(m * 3 + n + k)
    x, wg, wu = whole(rng, (m, k), 2), whole(rng, (n, k), 2), whole(rng, (n, k), 2)
    up, dh = whole(rng, (m, n), 3), whole(rng, (m, n), 2)
    gate = np.full((m, n), 32.0)
    dg, du = dh * up, 32 * dh
    for g, v in zip(backward(ctx, mem, *(bf(t) for t in (x, wg, wu, gate, up, dh))),
                    (dg @ wg + du @ wu, dg.T @ x, du.T @ x)):
        assert np.array_equal(g, bf(v)), np.argwhere(g != bf(v))[:4]


# dx's form and whether its depth is split, the weights' gradients'; odd k: copied operands
GRADIENT_FORMS = [("t64_d", False, "t64_d", False, 520, 264, 265), ("t64_d", False, "t64_d", True, 1500, 264, 1000),
                  ("t64_d", True, "t64_d", False, 520, 1000, 1000), ("t64_d", False, "t128", True, 4100, 1000, 265),
                  ("t128", True, "t64_d", False, 2050, 2056, 265),
                  ("t128", True, "t128", False, 520, 1000, 1800), ("t128", False, "t128", False, 520, 264, 4104),
                  ("t128", True, "t128", True, 4100, 2056, 71), ("t256", True, "t128", False, 1000, 2056, 4104),
                  ("t256", True, "t256", False, 2050, 2056, 2055), ("t256", False, "t128", True, 4100, 264, 2055),
                  ("t256", False, "t256", True, 4100, 1000, 2055)]


@pytest.mark.parametrize("form_x,split_x,form_w,split_w,m,n,k", GRADIENT_FORMS)
def test_backward_forms(ctx, mem, form_x, split_x, form_w, split_w, m, n, k):
    rz = realize(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (m, n, k), dtype=L.BF16, variant=L.GATED_DX | L.GATED_DW,
                 permissions=L.PERMITS_REASSOCIATION, flags=L.REGION_ALIGNED16)
    names = ["tiler_gated_bf16_grad", f"tiler_gated_bf16_dx_{form_x}", f"tiler_gated_bf16_dw_{form_w}"]
    assert rz.symbols == names + ["tiler_gated_bf16_sum"] * (split_x or split_w)
    assert [d.grid[1] > 1 for d in rz.dispatches[1:3]] == [split_x, split_w]
    test_backward_whole_numbers(ctx, mem, m, n, k)


@pytest.mark.parametrize("want", [(True, False), (False, True), (False, False)])
def test_backward_parts(ctx, mem, want):
    rng = np.random.default_rng(9)
    a = operands(rng, 70, 200, 136)
    full = backward(ctx, mem, *a)
    part = backward(ctx, mem, *a, want=want, workspace=None)
    for g, f in zip(part, full):
        assert g is None or np.array_equal(g, f)


def test_empty_sides(ctx, mem):
    rng = np.random.default_rng(1)
    x, wg, wu, gate, up, dh = operands(rng, 20, 72, 40)
    dx, dwg, dwu = backward(ctx, mem, x[:0], wg, wu, gate[:0], up[:0], dh[:0])
    assert (dwg == 0).all() and (dwu == 0).all()
    dx, dwg, dwu = backward(ctx, mem, x, wg[:0], wu[:0], gate[:, :0], up[:, :0], dh[:, :0])
    assert (dx == 0).all()
    forward(ctx, mem, x[:0], wg, wu, keep=True)
    forward(ctx, mem, x, wg[:0], wu[:0], keep=True)


def test_extreme_gates(ctx, mem):
    """Far gates: silu(G) is G or a zero, its slope 1 or 0; an infinity or a NaN
    in one token or weight row stays in its row or column."""
    k, n, m = 72, 40, 24
    x, wg, wu = np.zeros((m, k)), np.zeros((n, k)), np.ones((n, k))
    x[:, 0] = 1
    wg[:, 0] = np.linspace(-3000, 3000, n)
    x[:, 1] = 0.5
    h, g, u = forward(ctx, mem, bf(x), bf(wg), bf(wu), keep=True)
    gw = w64(g)
    assert np.array_equal(w64(h)[gw > 40], w64(bf(gw * 1.5))[gw > 40]) and (np.abs(w64(h)[gw < -150]) == 0).all()
    ones = np.ones((m, n))
    dx, dwg, dwu = backward(ctx, mem, bf(x), bf(wg), bf(wu), g, u, bf(ones))
    assert np.isfinite(w64(dx)).all() and np.isfinite(w64(dwg)).all() and np.isfinite(w64(dwu)).all()
    x[3, 5] = np.nan
    wg[7, 6] = np.inf
    x[:, 6] = 1
    h, g, u = (w64(v) for v in forward(ctx, mem, bf(x), bf(wg), bf(wu), keep=True))
    assert np.isnan(h[3]).all() and np.isinf(np.delete(g[:, 7], 3)).all()
    clean = np.delete(np.delete(h, 3, 0), 7, 1)
    assert np.isfinite(clean).all()


def test_rows_past_the_end_do_not_leak(ctx, mem):
    """A ragged depth in memory whose next rows are NaN: the zeros past the
    depth never meet them (n and k are not whole tiles)."""
    rng = np.random.default_rng(5)
    for m, n, k in ((40, 72, 72), (130, 136, 200), (300, 264, 520)):
        x, wg, wu, gate, up, dh = operands(rng, m, n, k)
        nan = BF(0x7fc0)

        def tailed(v):  # the operand, then poison
            flat = np.full(v.size + 4096, nan, BF)
            flat[:v.size] = v.reshape(-1)
            return mem.put(flat)

        a = [tailed(v) for v in (x, wg, wu, gate, up, dh)]
        h = mem.out(BF, m * n)
        ctx.gated_contract_bf16(*a[:3], m, n, k, h)
        dx, dwg, dwu = mem.out(BF, m * k), mem.out(BF, n * k), mem.out(BF, n * k)
        ctx.gated_contract_bf16_backward(*a, m, n, k, dx, dwg, dwu)
        ctx.synchronize()
        for v, s in ((h, (m, n)), (dx, (m, k)), (dwg, (n, k)), (dwu, (n, k))):
            assert np.isfinite(w64(mem.get(v, BF, s))).all()


def test_repeats_bit_for_bit(ctx, mem):
    a = operands(np.random.default_rng(6), 301, 520, 264)
    one, two = backward(ctx, mem, *a), backward(ctx, mem, *a, workspace=None)
    assert all(np.array_equal(p, q) for p, q in zip(one, two))


def test_gradient_against_differences(ctx, mem):
    """The gradients against central differences of the 64-bit forward form,
    to the bounds of their bf16 operands."""
    rng = np.random.default_rng(7)
    m, n, k, step = 3, 5, 8, 1e-5
    x, wg, wu = (bf(rng.standard_normal(s)) for s in ((m, k), (n, k), (n, k)))
    dh = bf(rng.standard_normal((m, n)))
    h, gate, up = forward(ctx, mem, x, wg, wu, keep=True)
    got = backward(ctx, mem, x, wg, wu, gate, up, dh)
    wide = [w64(v) for v in (x, wg, wu)]
    kept = [w64(v) for v in (gate, up, dh)]
    bound = ref.gated_backward_bounds(*wide, *kept)
    # the kept G and U are rounded too: slopes of at most 0.5 in G (twice) and 1.1 in U
    slack = 2.0 ** -8 * (0.5 * np.abs(kept[0] * kept[1]) + 1.1 * np.abs(kept[1]) + 1.1 * np.abs(kept[0])) * np.abs(kept[2])
    extra = (slack @ (np.abs(wide[1]) + np.abs(wide[2])), slack.T @ np.abs(wide[0]), slack.T @ np.abs(wide[0]))

    def loss(*v):
        return (ref.gated(*v)[0] * kept[2]).sum()

    for i, g in enumerate(got):
        for at in np.ndindex(wide[i].shape):
            up_, down = [v.copy() for v in wide], [v.copy() for v in wide]
            up_[i][at] += step
            down[i][at] -= step
            want = (loss(*up_) - loss(*down)) / (2 * step)
            assert abs(want - w64(g)[at]) <= bound[i][at] + extra[i][at] + 1e-6, (i, at)
