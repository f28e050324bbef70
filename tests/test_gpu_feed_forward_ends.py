"""The feed-forward sublayer's calls at the ends of their ranges: rows far from
zero, far gates, values that are not finite, empty rows, very many and very
long rows."""
from __future__ import annotations

import numpy as np
import pytest

import feed_forward_reference as ref
from tiler_amd import _lib as L
from tiler_amd import families
from tiler_amd.realize import realize, route
from tiler_amd.runtime import Refusal
from test_gpu_layer_norm import CODE, Buffers, backward, forward, kept, rows_of, within

pytestmark = pytest.mark.gpu

U = ref.U


@pytest.fixture
def mem(ctx):
    m = Buffers(ctx)
    yield m
    m.free()


def bf(values):
    return ref.store("bf16", values)


def w64(stored):
    return ref.wide("bf16", stored)


# -- the norm's gradients far from zero ------------------------------------------

def backward_bounds(dtype, dy, x, w, mean, rstd):
    """mean and rstd are operands, so x - mean rounds by U |x - mean| and xh, one
    more product, by 2 U |xh|, wherever the row lies.  The rest as in
    ref.layer_norm_backward_bounds: the row means 52 U of their magnitudes, the
    terms of dx at most 6 roundings, the column sums rows + 600 additions."""
    dx, dw, db = ref.layer_norm_backward(dy, x, w, mean, rstd)
    xh = np.abs((x - mean[:, None]) * rstd[:, None])
    g = np.abs(dy if w is None else dy * w)
    m1, m2 = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    e_dx = rstd[:, None] * (4 * U * g + (52 + 4) * U * m1 + xh * (56 + 2 + 2 + 6) * U * m2)
    n = min(x.shape[0], 1200) + 600
    e_dw, e_db = (n + 2) * U * (np.abs(dy) * xh).sum(0), n * U * np.abs(dy).sum(0)
    h = ref.half(dtype)
    return e_dx + h * (np.abs(dx) + e_dx), e_dw + h * (np.abs(dw) + e_dw), e_db + h * (np.abs(db) + e_db)


def check_backward(ctx, mem, dtype, dy, x, w, mean, rstd):
    args = (ref.wide(dtype, dy), ref.wide(dtype, x), None if w is None else ref.wide(dtype, w), mean.astype(np.float64),
            rstd.astype(np.float64))
    got = backward(ctx, mem, dtype, dy, x, w, mean, rstd)
    for g, v, e, what in zip(got, ref.layer_norm_backward(*args), backward_bounds(dtype, *args), ("dx", "dw", "db")):
        within(ref.wide(dtype, g), v, e, what)


# the forms of one to sixteen waves a row, two pieces a thread, and streamed rows
@pytest.mark.parametrize("extent", [100, 256, 509, 1023, 2048, 4096, 8190, 20001])
@pytest.mark.parametrize("offset", [3000.0, -1e5])
def test_gradients_do_not_lose_a_row_far_from_zero(ctx, mem, offset, extent):
    rng = np.random.default_rng(extent)
    x = (rows_of(rng, 70, extent, "f32") + np.float32(offset)).astype(np.float32)
    dy, w = rng.standard_normal((70, extent)).astype(np.float32), rng.normal(1, 0.2, extent).astype(np.float32)
    for weight in (w, None):
        check_backward(ctx, mem, "f32", dy, x, weight, *kept("f32", x))


@pytest.mark.parametrize("extent", [100, 1024, 4096, 16384])
def test_gradients_of_nearly_constant_bf16_rows(ctx, mem, extent):
    rng = np.random.default_rng(extent)
    x = np.full((40, extent), 200.0)
    x[np.arange(40), rng.integers(0, extent, 40)] += 1
    x, dy, w = bf(x), bf(rng.standard_normal((40, extent))), bf(rng.normal(1, 0.2, extent))
    check_backward(ctx, mem, "bf16", dy, x, w, *kept("bf16", x))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [100, 4096, 20001])
def test_gradients_of_constant_rows_with_a_tiny_eps(ctx, mem, dtype, extent):
    """rstd = 1 / sqrt(eps) whose square passes binary32's range."""
    rng = np.random.default_rng(extent)
    x, dy = ref.store(dtype, np.full((6, extent), 3.0)), ref.store(dtype, rng.standard_normal((6, extent)))
    mean, rstd = np.full(6, 3, np.float32), np.full(6, 2e20, np.float32)
    check_backward(ctx, mem, dtype, dy, x, None, mean, rstd)


# -- very long rows ---------------------------------------------------------------------

@pytest.mark.parametrize("extent", [(1 << 26) + 70, (1 << 28) + 5])
def test_column_sums_of_very_long_rows(ctx, mem, extent):
    """More columns than the column kernels have threads: each takes further ones.
    Whole numbers, mean 0 and rstd 1: dw is the sum of dy x, exactly."""
    pattern = np.arange(1021) % 13 - 6  # prime: no period of the columns' groups
    dy, x = np.resize(bf(pattern), extent), np.resize(bf(pattern % 5 + 1), extent)
    mean, rstd = mem.put(np.zeros(1, np.float32)), mem.put(np.ones(1, np.float32))
    ws = ctx.alloc(ctx.layer_norm_backward_workspace(L.BF16, 1, extent))
    bufs = [ctx.to_device(dy), ctx.to_device(x), ctx.alloc(2 * extent), ctx.alloc(2 * extent)]
    try:
        ctx.layer_norm_backward(L.BF16, bufs[0], bufs[1], None, mean, rstd, 1, extent, None, bufs[2], bufs[3],
                                workspace=ws, workspace_bytes=ws.nbytes)
        ctx.synchronize()
        assert np.array_equal(bufs[3].download(np.uint16, (extent,)), np.resize(bf(pattern + 0.0), extent))
        assert np.array_equal(bufs[2].download(np.uint16, (extent,)), np.resize(bf(pattern * (pattern % 5 + 1)), extent))
    finally:
        for b in [*bufs, ws]:
            b.free()


# -- routed with the caller's scratch -----------------------------------------------------

@pytest.mark.parametrize("m,n,k", [(300, 520, 264), (300, 520, 333)])
def test_routed_gradients_in_the_callers_scratch(ctx, mem, m, n, k):
    """Operands at odd elements, scratch a 16-byte step past its allocations: the
    direct call's bits, and nothing written past the slots."""
    rng = np.random.default_rng(k)
    shapes = [(m, k), (n, k), (n, k), (m, n), (m, n), (m, n)]
    operands = [mem.put(bf(rng.standard_normal(s)), 1) for s in shapes]
    want = [mem.out(np.uint16, c) for c in (m * k, n * k, n * k)]
    ctx.gated_contract_bf16_backward(*operands, m, n, k, *want)
    rz = realize(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (m, n, k), dtype=L.BF16, variant=L.GATED_DX | L.GATED_DW,
                 permissions=L.PERMITS_REASSOCIATION, flags=0, ctx=ctx)
    got, scratch = [mem.out(np.uint16, c, 1) for c in (m * k, n * k, n * k)], []
    given = iter(operands + got)
    storage = []
    for role, nbytes in rz.slots:
        if role == L.SLOT_SCRATCH:
            scratch.append((mem.out(np.uint8, nbytes, 16), nbytes))
        storage.append(scratch[-1][0] if role == L.SLOT_SCRATCH else next(given))
    assert scratch
    route(ctx, rz, storage)
    for w, g, c in zip(want, got, (m * k, n * k, n * k)):
        assert np.array_equal(mem.get(w, np.uint16, (c,)), mem.get(g, np.uint16, (c,)))
    for v, nbytes in scratch:
        mem.get(v, np.uint8, (nbytes,))


# -- rows without elements ----------------------------------------------------------

def test_empty_rows(ctx, mem):
    """No element, no mean and no scale: refused where one is asked for, and
    nothing is written."""
    mean, rstd, y = mem.out(np.float32, 3), mem.out(np.float32, 3), mem.out(np.uint16, 8)
    x = mem.put(np.zeros(8, np.uint16))
    for call in (lambda: ctx.layer_norm(L.BF16, x, None, None, 3, 0, ref.EPS_BITS, y, mean, rstd),
                 lambda: ctx.quantize_rows_i8(L.BF16, x, 3, 0, y, mean),
                 lambda: families.layer_norm(np.zeros((3, 0), np.uint16), ctx=ctx),
                 lambda: families.quantize_rows_i8(np.zeros((3, 0), np.float32), ctx=ctx)):
        with pytest.raises(Refusal) as e:
            call()
        assert e.value.status == L.REFUSE_INVALID_ARGUMENT
    ctx.layer_norm(L.BF16, x, None, None, 3, 0, ref.EPS_BITS, y)
    ctx.layer_norm(L.BF16, x, None, None, 0, 0, ref.EPS_BITS, y, mean, rstd)
    ctx.quantize_rows_i8(L.BF16, x, 0, 0, y, mean)
    ctx.synchronize()
    for v, t, c in ((mean, np.float32, 3), (rstd, np.float32, 3), (y, np.uint16, 8)):
        assert (mem.get(v, t, (c,)).view(np.uint8) == 0xA5).all()


# -- the norm far from zero -------------------------------------------------------

def forward_bounds(dtype, x, w, b, e_mean):
    """`e_mean`: how far the row's first, binary32 mean may be off.  The
    differences from it round by U of themselves; their mean (52 U of their
    magnitudes) is taken off again, so that y carries rounding of the differences'
    size, not of the row's.  rstd: the variance's 60 U, of its sum of squares
    around the first mean, and 4 U."""
    y, mu, r = ref.layer_norm(x, w, b)
    d, r = np.abs(x - mu[:, None]), r[:, None]
    off = 54 * U * (d.mean(-1, keepdims=True) + e_mean) + 2 * U * e_mean
    e_r = 60 * U * (1 + (e_mean * r) ** 2) + (off * r) * (e_mean * r) + 4 * U
    e_xh = (U * (d + e_mean) + off) * r + d * r * (e_r + 4 * U)
    scale = 1.0 if w is None else np.abs(w)
    e_y = e_xh * scale + 2 * U * (d * r * scale + (0.0 if b is None else np.abs(b)))
    return e_y + ref.half(dtype) * (np.abs(y) + e_y), U * np.abs(mu) + off[:, 0], (e_r * r)[:, 0]


def check_forward(ctx, mem, dtype, x, w, b, e_mean):
    args = (ref.wide(dtype, x), None if w is None else ref.wide(dtype, w), None if b is None else ref.wide(dtype, b))
    bounds = forward_bounds(dtype, *args, e_mean)
    for got, want, bound, what in zip(forward(ctx, mem, dtype, x, w, b), ref.layer_norm(*args), bounds, ("y", "mean", "rstd")):
        within(ref.wide(dtype, got) if what == "y" else got, want, bound, what)


@pytest.mark.parametrize("extent", [100, 509, 1023, 4096, 8190, 16380, 20001])
@pytest.mark.parametrize("offset", [3000.0, -1e5])
def test_norm_of_rows_far_from_zero(ctx, mem, offset, extent):
    rng = np.random.default_rng(extent)
    x = (rows_of(rng, 37, extent, "f32") + np.float32(offset)).astype(np.float32)
    w, b = rng.normal(1, 0.2, extent).astype(np.float32), rng.normal(0, 0.2, extent).astype(np.float32)
    e_mean = 52 * U * np.abs(x.astype(np.float64)).mean(-1, keepdims=True)
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        check_forward(ctx, mem, "f32", x, weight, bias, e_mean)


@pytest.mark.parametrize("extent", [100, 509, 2046, 4096, 8190, 16382, 32766, 40000])
def test_norm_of_nearly_constant_bf16_rows(ctx, mem, extent):
    """Whole numbers: their sum is below 2^24 and exact, so the first mean is off by
    its rounding alone."""
    rng = np.random.default_rng(extent)
    x = np.full((37, extent), 200.0)
    for i in range(37):
        x[i, rng.integers(0, extent, 1 + i % 4)] += rng.integers(1, 4)
    w, b = bf(rng.normal(1, 0.2, extent)), bf(rng.normal(0, 0.2, extent))
    assert x.sum(-1).max() < 1 << 24
    for weight, bias in ((w, b), (None, None)):
        check_forward(ctx, mem, "bf16", bf(x), weight, bias, 256 * U)


# -- far gates --------------------------------------------------------------------

FAR = np.array([-174.0, -160.0, -140.0, -120.0, -100.0, -95.0, -92.0, -90.0, -89.0, -88.5, -88.0, -87.5, -87.0, -85.0,
                -80.0, -60.0, -30.0, -8.0, -1.28125, -0.0, 0.5, 8.0, 30.0, 80.0, 88.0, 90.0, 120.0, 200.0])


def sigmoid(g):
    """s and 1 - s, neither of them a difference."""
    t = np.exp(-np.abs(g))
    return np.where(g < 0, t, 1) / (1 + t), np.where(g < 0, 1, t) / (1 + t)


def gate_bound(value, g, terms=None):
    """The exponent of e^(-|G| / 2) rounds twice, |G| U of relative error in all, and
    the factor enters twice; two exponentials of 2 U, a reciprocal, the products
    and slope's sum 16 U.  Then bf16's rounding, at least half its least step."""
    e = (20 + 2 * np.abs(g)) * U * (np.abs(value) if terms is None else terms)
    return e + np.maximum(ref.half("bf16") * (np.abs(value) + e), 2.0 ** -134)


@pytest.mark.parametrize("m,k", [(3, 64), (40, 333), (70, 5), (200, 1024), (700, 2048)])
def test_far_gates(ctx, mem, m, k):
    """silu(G) down to where bf16 holds nothing of the result: e^-G itself passes
    binary32's range below G = -88.7, silu(G) U need not."""
    n, rng = 2 * len(FAR), np.random.default_rng(m)
    x, wg, wu = np.zeros((m, k)), np.zeros((n, k)), np.zeros((n, k))
    x[:, 0] = x[:, 1] = 1  # one product each of G and U: exact
    wg[:, 0] = np.tile(FAR, 2)
    wu[:, 1] = np.repeat([1.5, -2.0 ** 100], len(FAR))
    args = [bf(v) for v in (x, wg, wu)]
    h, gate, up = (mem.out(np.uint16, m * n) for _ in range(3))
    ctx.gated_contract_bf16(*(mem.put(v) for v in args), m, n, k, h, gate, up)
    ctx.synchronize()
    g, u = (np.broadcast_to(v, (m, n)) for v in (wg[:, 0], wu[:, 1]))
    assert np.array_equal(w64(mem.get(gate, np.uint16, (m, n))), g) and np.array_equal(w64(mem.get(up, np.uint16, (m, n))), u)
    want = g * sigmoid(g)[0] * u
    within(w64(mem.get(h, np.uint16, (m, n))), want, gate_bound(want, g), "h")


def test_slopes_of_far_gates(ctx, mem):
    """dG and dU by themselves: one token, x = 1, and a depth of one."""
    n = 2 * len(FAR)
    g, u = np.tile(FAR, 2)[None, :], np.repeat([1.5, -2.0 ** 100], len(FAR))[None, :]
    d = np.repeat([-3.0, 2.0 ** 10], len(FAR))[None, :]
    one = np.ones((1, 1))
    dwg, dwu = mem.out(np.uint16, n), mem.out(np.uint16, n)
    w = mem.put(bf(np.ones((n, 1))))
    ctx.gated_contract_bf16_backward(mem.put(bf(one)), w, w, *(mem.put(bf(v)) for v in (g, u, d)), 1, n, 1, None, dwg, dwu)
    ctx.synchronize()
    s, t = sigmoid(g)
    want_u, want_g = d * g * s, d * u * s * (1 + g * t)
    terms = np.abs(d * u * s) * (1 + np.abs(g) * t)
    within(w64(mem.get(dwu, np.uint16, (1, n))), want_u, gate_bound(want_u, g), "dU")
    within(w64(mem.get(dwg, np.uint16, (1, n))), want_g, gate_bound(want_g, g, terms), "dG")


# -- very many short rows -------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_rows_than_workgroups(ctx, mem, dtype):
    """Streamed rows past the 2^20 workgroups of a launch: each takes further rows."""
    rows, extent = (1 << 20) + 5, 3
    for program, variant, symbol in ((L.PROGRAM_LAYER_NORM, L.NORM_STATISTICS, "tiler_layer_norm_%s_s"),
                                     (L.PROGRAM_LAYER_NORM_BACKWARD, L.NORM_DX, "tiler_layer_norm_grad_%s_s"),
                                     (L.PROGRAM_QUANTIZE_ROWS_I8, 0, "tiler_quantize_rows_i8_%s_s")):
        rz = realize(program, (rows, extent), dtype=CODE[dtype], variant=variant, scalars=(ref.EPS_BITS, 0),
                     permissions=L.PERMITS_REASSOCIATION)
        assert rz.symbols == [symbol % dtype] and rz.dispatches[0].grid[0] < rows
    rng = np.random.default_rng(3)
    x, dy = rows_of(rng, rows, extent, dtype), ref.store(dtype, rng.standard_normal((rows, extent)))
    args = (ref.wide(dtype, x), None, None)
    y, mean, rstd = forward(ctx, mem, dtype, x, None, None)
    for got, want, bound in zip((ref.wide(dtype, y), mean, rstd), ref.layer_norm(*args), ref.layer_norm_bounds(dtype, *args)):
        within(got, want, bound, "forward")
    back = (ref.wide(dtype, dy), args[0], None, mean.astype(np.float64), rstd.astype(np.float64))
    dx, _, _ = backward(ctx, mem, dtype, dy, x, None, mean, rstd, want=(True, False, False))
    within(ref.wide(dtype, dx), ref.layer_norm_backward(*back)[0], ref.layer_norm_backward_bounds(dtype, *back)[0], "dx")
    q, s = mem.out(np.int8, rows * extent), mem.out(np.float32, rows)
    ctx.quantize_rows_i8(CODE[dtype], mem.put(x), rows, extent, q, s)
    ctx.synchronize()
    codes, scales = ref.quantize_rows(ref.wide(dtype, x))
    assert np.array_equal(mem.get(q, np.int8, codes.shape), codes) and np.array_equal(mem.get(s, np.float32, (rows,)), scales)


# -- values that are not finite -----------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [5, 100, 1023, 4096, 8190, 20001])
def test_norm_of_poisoned_rows(ctx, mem, dtype, extent):
    """A NaN or an infinity takes its own row, and no other."""
    rng = np.random.default_rng(extent)
    v = ref.wide(dtype, rows_of(rng, 9, extent, dtype))
    v[2, extent - 1], v[4, 0], v[7, extent // 2] = np.nan, np.inf, -np.inf
    x, bad = ref.store(dtype, v), [2, 4, 7]
    good = np.delete(np.arange(9), bad)
    y, mean, rstd = forward(ctx, mem, dtype, x, None, None)
    assert np.isnan(ref.wide(dtype, y)[bad]).all() and np.isnan(rstd[bad]).all() and not np.isfinite(mean[bad]).any()
    args = (v[good], None, None)
    within(ref.wide(dtype, y)[good], ref.layer_norm(*args)[0], ref.layer_norm_bounds(dtype, *args)[0], "y")
    # the gradients: NaN in those rows of dx and, as a sum over the rows, all over dw; db is dy's alone
    dy = ref.store(dtype, rng.standard_normal((9, extent)))
    dx, dw, db = (ref.wide(dtype, t) for t in backward(ctx, mem, dtype, dy, x, None, mean, rstd))
    assert np.isnan(dx[bad]).all() and np.isnan(dw).all()
    back = (ref.wide(dtype, dy)[good], v[good], None, mean[good].astype(np.float64), rstd[good].astype(np.float64))
    within(dx[good], ref.layer_norm_backward(*back)[0], ref.layer_norm_backward_bounds(dtype, *back)[0], "dx")
    wide_dy = ref.wide(dtype, dy)
    e = 700 * U * np.abs(wide_dy).sum(0)
    within(db, wide_dy.sum(0), e + ref.half(dtype) * (np.abs(wide_dy.sum(0)) + e), "db")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [5, 100, 1023, 4096, 8190, 20001])
def test_poisoned_gradients_of_the_norm(ctx, mem, dtype, extent):
    """A NaN or an infinity in dy takes its row of dx and its column of dw and db (dx of
    the infinite row: both row means are infinite, so NaN or an infinity by the signs
    of xh)."""
    rng = np.random.default_rng(extent + 1)
    x, v = rows_of(rng, 300, extent, dtype), ref.wide(dtype, ref.store(dtype, rng.standard_normal((300, extent))))
    v[3, 0], v[299, extent - 1] = np.inf, np.nan
    dy, (mean, rstd) = ref.store(dtype, v), kept(dtype, x)
    dx, dw, db = (ref.wide(dtype, t) for t in backward(ctx, mem, dtype, dy, x, None, mean, rstd))
    rows = np.zeros(300, bool)
    rows[[3, 299]] = True
    cols = np.zeros(extent, bool)
    cols[[0, extent - 1]] = True
    assert np.isnan(dx[299]).all() and not np.isfinite(dx[rows]).any() and np.isfinite(dx[~rows]).all()
    for t in (dw, db):
        assert not np.isfinite(t[cols]).any() and np.isfinite(t[~cols]).all()


# a form of each kind: few tiles and many, whole and split depths, copied operands
@pytest.mark.parametrize("m,n,k", [(40, 72, 72), (130, 136, 203), (520, 264, 264), (1500, 264, 1000), (2050, 2056, 2056)])
def test_poisoned_gradients_of_the_gated_product(ctx, mem, m, n, k):
    """In dh a NaN or an infinity takes a token's row of dx, a channel's row of dWg and
    dWu; in x a column of both; in a weight a column of dx: nothing else."""
    rng = np.random.default_rng(m)

    def grads(poison):
        v = {"x": (m, k), "wg": (n, k), "wu": (n, k), "gate": (m, n), "up": (m, n), "dh": (m, n)}
        v = {name: w64(bf(rng.standard_normal(s))) for name, s in v.items()}
        for name, at, value in poison:
            v[name][at] = value
        dx, dwg, dwu = mem.out(np.uint16, m * k), mem.out(np.uint16, n * k), mem.out(np.uint16, n * k)
        ctx.gated_contract_bf16_backward(*(mem.put(bf(t)) for t in v.values()), m, n, k, dx, dwg, dwu)
        ctx.synchronize()
        return [w64(mem.get(t, np.uint16, s)) for t, s in ((dx, (m, k)), (dwg, (n, k)), (dwu, (n, k)))]

    def only(t, rows=(), cols=()):
        bad = np.zeros(t.shape, bool)
        bad[list(rows)] = True
        bad[:, list(cols)] = True
        assert not np.isfinite(t[bad]).any() and np.isfinite(t[~bad]).all(), (np.argwhere(np.isfinite(t) == bad)[:4])

    dx, dwg, dwu = grads([("dh", (m - 1, 0), np.nan), ("dh", (3, n - 1), np.inf)])
    only(dx, rows=(3, m - 1)), only(dwg, rows=(0, n - 1)), only(dwu, rows=(0, n - 1))
    dx, dwg, dwu = grads([("x", (m - 1, k - 1), np.inf), ("x", (0, 0), np.nan)])
    only(dx), only(dwg, cols=(0, k - 1)), only(dwu, cols=(0, k - 1))
    dx, dwg, dwu = grads([("wg", (n - 1, k - 1), np.nan), ("wu", (0, 1), -np.inf)])
    only(dx, cols=(1, k - 1)), only(dwg), only(dwu)


# -- calls that meet nothing, routed --------------------------------------------------

def test_routed_without_tokens(ctx, mem):
    """No token or no channel, through the recognizer: zeros, as the direct call."""
    k = 40
    for m, n in ((0, 72), (20, 0)):
        rz = realize(L.PROGRAM_GATED_CONTRACTION_BACKWARD, (m, n, k), dtype=L.BF16, variant=L.GATED_DX | L.GATED_DW,
                     permissions=L.PERMITS_REASSOCIATION)
        some = mem.put(np.zeros(64, np.uint16))
        outs = [mem.out(np.uint16, c) for c in (m * k, n * k, n * k)]
        storage = iter([some] * 6 + outs)
        route(ctx, rz, [None if role == L.SLOT_SCRATCH else int(next(storage).ptr) for role, _ in rz.slots])
        for v, c in zip(outs, (m * k, n * k, n * k)):
            assert (mem.get(v, np.uint16, (c,)) == 0).all()
