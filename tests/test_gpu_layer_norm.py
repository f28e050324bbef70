"""Layer norm and its gradients on the device, against the 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest

import feed_forward_reference as ref
from tiler_amd import _lib as L
from tiler_amd.realize import realize
from tiler_amd.runtime import Refusal

pytestmark = pytest.mark.gpu

CODE = {"bf16": L.BF16, "f32": L.F32}
# one element, a lane's, a wave's, ragged chunks of each form, the longest
# registers hold, streamed rows
EXTENTS = [1, 2, 7, 8, 63, 64, 100, 255, 256, 509, 512, 1000, 1023, 1024, 2048, 2050, 4096, 5000, 8192, 8200, 12288,
           16384, 16392, 20001]


class Buffers:
    """Device storage at a chosen misalignment (in elements), poisoned around."""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def put(self, host, shift=0):
        host = np.ascontiguousarray(host)
        buf = self.ctx.alloc(host.nbytes + 64)
        self.all.append(buf)
        view = buf.offset(shift * host.itemsize)
        if host.nbytes:
            view.upload(host)
        return view

    def out(self, dtype, count, shift=0):
        item = np.dtype(dtype).itemsize
        raw = np.full(count * item + 64, 0xA5, np.uint8)
        buf = self.ctx.alloc(raw.nbytes)
        buf.upload(raw)
        self.all.append(buf)
        view = buf.offset(shift * item)
        view.guard = (buf, shift * item, count * item, raw.nbytes)
        return view

    def get(self, view, dtype, shape):
        """The result; what lies around it has to be untouched."""
        buf, at, nbytes, total = view.guard
        raw = buf.download(np.uint8, (total,))
        assert (raw[:at] == 0xA5).all() and (raw[at + nbytes:] == 0xA5).all(), "written outside the result"
        return raw[at:at + nbytes].view(dtype).reshape(shape).copy()

    def free(self):
        self.ctx.synchronize()
        for b in self.all:
            b.free()


@pytest.fixture
def mem(ctx):
    m = Buffers(ctx)
    yield m
    m.free()


def storage(dtype):
    return np.uint16 if dtype == "bf16" else np.float32


def rows_of(rng, rows, extent, dtype):
    x = rng.standard_normal((rows, extent)) * rng.uniform(0.5, 2.0, (rows, 1)) + rng.normal(0, 1.0, (rows, 1))
    return ref.store(dtype, x)


def within(got, want, bound, what):
    off = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (off <= 0).all(), (what, float(off.max()), np.unravel_index(off.argmax(), off.shape))


def forward(ctx, mem, dtype, x, w, b, shift=0, stats=True, eps_bits=ref.EPS_BITS, stream=None):
    rows, extent = x.shape
    dx = mem.put(x, shift)
    dw = None if w is None else mem.put(w, shift)
    db = None if b is None else mem.put(b, shift)
    y = mem.out(storage(dtype), rows * extent, shift)
    mean = mem.out(np.float32, rows) if stats else None
    rstd = mem.out(np.float32, rows) if stats else None
    ctx.layer_norm(CODE[dtype], dx, dw, db, rows, extent, eps_bits, y, mean=mean, rstd=rstd, stream=stream)
    ctx.synchronize()
    out = [mem.get(y, storage(dtype), (rows, extent))]
    if stats:
        out += [mem.get(mean, np.float32, (rows,)), mem.get(rstd, np.float32, (rows,))]
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", EXTENTS)
def test_forward(ctx, mem, dtype, extent):
    rng = np.random.default_rng(extent)
    for rows in (1, 5, 67):
        x = rows_of(rng, rows, extent, dtype)
        w, b = ref.store(dtype, rng.normal(1, 0.2, extent)), ref.store(dtype, rng.normal(0, 0.2, extent))
        y, mean, rstd = forward(ctx, mem, dtype, x, w, b)
        args = (ref.wide(dtype, x), ref.wide(dtype, w), ref.wide(dtype, b))
        wy, wmean, wrstd = ref.layer_norm(*args)
        ey, emean, erstd = ref.layer_norm_bounds(dtype, *args)
        within(mean, wmean, emean, "mean")
        within(rstd, wrstd, erstd, "rstd")
        within(ref.wide(dtype, y), wy, ey, "y")


# Every form of the rows (extents of bf16; of f32 half as long): a ragged last piece, ragged last workgroups
ROW_FORMS = [("s", 5, 7), ("w1c1", 1030, 510), ("w1c2", 1030, 1022), ("w1c4", 2051, 2046), ("w4c1", 40, 2046),
             ("w4c2", 40, 4094), ("w4c4", 300, 8190), ("w16c1", 40, 8190), ("w16c2", 9, 16382), ("w16c4", 9, 32766),
             ("s", 9, 32770)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("form,rows,extent", ROW_FORMS)
def test_forward_forms(ctx, mem, dtype, form, rows, extent):
    extent = extent if dtype == "bf16" else extent // 2
    rz = realize(L.PROGRAM_LAYER_NORM, (rows, extent), dtype=CODE[dtype], scalars=(ref.EPS_BITS, 0),
                 permissions=L.PERMITS_REASSOCIATION)
    assert rz.symbols == [f"tiler_layer_norm_{dtype}_{form}"]
    rng = np.random.default_rng(extent)
    x = rows_of(rng, rows, extent, dtype)
    w, b = ref.store(dtype, rng.normal(1, 0.2, extent)), ref.store(dtype, rng.normal(0, 0.2, extent))
    args = (ref.wide(dtype, x), ref.wide(dtype, w), ref.wide(dtype, b))
    for got, want, bound in zip(forward(ctx, mem, dtype, x, w, b), ref.layer_norm(*args), ref.layer_norm_bounds(dtype, *args)):
        within(ref.wide(dtype, got) if got.ndim == 2 else got, want, bound, (form, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [24, 1000, 4096, 16384])
@pytest.mark.parametrize("shift", [1, 3])
def test_forward_unaligned_and_without_operands(ctx, mem, dtype, extent, shift):
    rng = np.random.default_rng(extent + shift)
    x = rows_of(rng, 9, extent, dtype)
    w, b = ref.store(dtype, rng.normal(1, 0.2, extent)), ref.store(dtype, rng.normal(0, 0.2, extent))
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        y, = forward(ctx, mem, dtype, x, ww, bb, shift, stats=False)
        args = (ref.wide(dtype, x), None if ww is None else ref.wide(dtype, ww),
                None if bb is None else ref.wide(dtype, bb))
        within(ref.wide(dtype, y), ref.layer_norm(*args)[0], ref.layer_norm_bounds(dtype, *args)[0], (ww is None, bb is None))


@pytest.mark.parametrize("extent", [64, 4096, 20000])
def test_a_large_offset_keeps_the_variance(ctx, mem, extent):
    """A row far from zero: the squares' difference would cancel to nothing."""
    rng = np.random.default_rng(extent)
    x = (1000.0 + rng.standard_normal((4, extent))).astype(np.float32)
    y, mean, rstd = forward(ctx, mem, "f32", x, None, None)
    wy, wmean, wrstd = ref.layer_norm(x.astype(np.float64), None, None)
    ey, emean, erstd = ref.layer_norm_bounds("f32", x.astype(np.float64), None, None)
    within(rstd, wrstd, erstd, "rstd")
    within(mean, wmean, emean, "mean")
    within(y.astype(np.float64), wy, ey, "y")


def test_constant_rows_and_poisoned_rows(ctx, mem):
    extent = 512
    x = np.zeros((6, extent), np.float32)
    x[1] = 3.0
    x[2] = -7.5
    x[3] = 1.0
    x[3, 100] = np.nan
    x[4] = 1.0
    x[4, 5] = np.inf
    x[5] = np.arange(extent)
    b = np.full(extent, 0.25, np.float32)
    y, mean, rstd = forward(ctx, mem, "f32", x, None, b)
    assert (y[:3] == 0.25).all()  # no spread: the bias
    assert mean[:3].tolist() == [0.0, 3.0, -7.5]
    assert np.allclose(rstd[:3], 1 / np.sqrt(ref.EPS), rtol=8 * ref.U)
    assert np.isnan(y[3]).all() and np.isnan(y[4]).all() and np.isfinite(y[5]).all()


def test_many_short_rows(ctx, mem):
    """More rows than workgroups are launched for at once."""
    rng = np.random.default_rng(0)
    x = rows_of(rng, 70001, 3, "bf16")
    y, mean, rstd = forward(ctx, mem, "bf16", x, None, None)
    args = (ref.wide("bf16", x), None, None)
    within(ref.wide("bf16", y), ref.layer_norm(*args)[0], ref.layer_norm_bounds("bf16", *args)[0], "y")


def backward(ctx, mem, dtype, dy, x, w, mean, rstd, shift=0, want=(True, True, True), workspace="given", stream=None):
    rows, extent = x.shape
    a = [mem.put(dy, shift), mem.put(x, shift), None if w is None else mem.put(w, shift), mem.put(mean), mem.put(rstd)]
    dx = mem.out(storage(dtype), rows * extent, shift) if want[0] else None
    dw = mem.out(storage(dtype), extent, shift) if want[1] else None
    db = mem.out(storage(dtype), extent, shift) if want[2] else None
    ws, nbytes = None, 0
    if workspace == "given":
        nbytes = ctx.layer_norm_backward_workspace(CODE[dtype], rows, extent)
        ws = mem.out(np.uint8, max(nbytes, 1))
    ctx.layer_norm_backward(CODE[dtype], *a, rows, extent, dx, dw, db, workspace=ws, workspace_bytes=nbytes, stream=stream)
    ctx.synchronize()
    if ws is not None:
        mem.get(ws, np.uint8, (max(nbytes, 1),))  # nothing written past it
    return [None if v is None else mem.get(v, storage(dtype), s)
            for v, s in ((dx, (rows, extent)), (dw, (extent,)), (db, (extent,)))]


def kept(dtype, x):
    _, mu, r = ref.layer_norm(ref.wide(dtype, x), None, None)
    return mu.astype(np.float32), r.astype(np.float32)


def check_backward(ctx, mem, dtype, rows, extent, rng, shift=0, with_w=True, want=(True, True, True), workspace="given",
                   offset=0.0):
    x = ref.store(dtype, ref.wide(dtype, rows_of(rng, rows, extent, dtype)) + offset)
    dy = ref.store(dtype, rng.standard_normal((rows, extent)))
    w = ref.store(dtype, rng.normal(1, 0.2, extent)) if with_w else None
    mean, rstd = kept(dtype, x)
    got = backward(ctx, mem, dtype, dy, x, w, mean, rstd, shift, want, workspace)
    args = (ref.wide(dtype, dy), ref.wide(dtype, x), None if w is None else ref.wide(dtype, w), mean.astype(np.float64),
            rstd.astype(np.float64))
    for g, v, e, what in zip(got, ref.layer_norm_backward(*args), ref.layer_norm_backward_bounds(dtype, *args),
                             ("dx", "dw", "db")):
        if g is not None:
            within(ref.wide(dtype, g), v, e, (what, rows, extent))
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", EXTENTS)
def test_backward(ctx, mem, dtype, extent):
    rng = np.random.default_rng(extent + 1)
    for rows in (1, 3, 40, 300):
        check_backward(ctx, mem, dtype, rows, extent, rng)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,extent", [(2049, 128), (5003, 1000), (1100, 4096), (33, 16385)])
def test_backward_many_rows(ctx, mem, dtype, rows, extent):
    check_backward(ctx, mem, dtype, rows, extent, np.random.default_rng(rows), workspace=None)


@pytest.mark.parametrize("dtype,offset", [("f32", 3000.0), ("f32", -1e5), ("bf16", 40.0)])
@pytest.mark.parametrize("extent", [100, 4096, 20001])
def test_backward_far_from_zero(ctx, mem, dtype, offset, extent):
    """Rows whose mean is many deviations from zero."""
    check_backward(ctx, mem, dtype, 70, extent, np.random.default_rng(extent), offset=offset)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [40, 1024, 4095])
def test_backward_parts(ctx, mem, dtype, extent):
    """Each subset of the results, without a weight, unaligned."""
    rng = np.random.default_rng(extent)
    for want in ((True, False, False), (False, True, False), (False, False, True), (True, True, False),
                 (False, True, True), (False, False, False)):
        check_backward(ctx, mem, dtype, 37, extent, rng, shift=1, with_w=want[0] and want[1], want=want)


def test_backward_without_rows_gives_zeros(ctx, mem):
    none = np.zeros((0, 100), np.float32)
    dx, dw, db = backward(ctx, mem, "f32", none, none, np.ones(100, np.float32), none[:, 0], none[:, 0])
    assert (dw == 0).all() and (db == 0).all()


def test_backward_repeats_bit_for_bit(ctx, mem):
    rng = np.random.default_rng(2)
    x, dy = rows_of(rng, 3001, 1000, "f32"), rng.standard_normal((3001, 1000)).astype(np.float32)
    mean, rstd = kept("f32", x)
    one = backward(ctx, mem, "f32", dy, x, None, mean, rstd)
    two = backward(ctx, mem, "f32", dy, x, None, mean, rstd)
    assert all(np.array_equal(a, b) for a, b in zip(one, two))


def test_gradient_against_differences(ctx, mem):
    """dx, dw and db against central differences of the 64-bit forward form."""
    rng = np.random.default_rng(3)
    rows, extent, h = 3, 12, 1e-5
    x, dy = rng.standard_normal((rows, extent)), rng.standard_normal((rows, extent))
    w, b = rng.normal(1, 0.2, extent), rng.normal(0, 0.2, extent)
    x, dy, w, b = (v.astype(np.float32) for v in (x, dy, w, b))
    y, mean, rstd = forward(ctx, mem, "f32", x, w, b)
    got = backward(ctx, mem, "f32", dy, x, w, mean, rstd)

    def loss(xx, ww, bb):
        return (ref.layer_norm(xx, ww, bb)[0] * dy).sum()

    base = [v.astype(np.float64) for v in (x, w, b)]
    for i, g in enumerate(got):
        for at in np.ndindex(base[i].shape):
            up, down = [v.copy() for v in base], [v.copy() for v in base]
            up[i][at] += h
            down[i][at] -= h
            # third derivatives of order r^3 ~ 10: h^2 10 < 1e-8; binary32's share below 1e-4
            assert abs((loss(*up) - loss(*down)) / (2 * h) - g[at]) < 1e-4, (i, at)


def test_capture_with_a_workspace(ctx, mem):
    """A captured backward call replays beside eager calls; without a workspace
    the capture is refused."""
    rng = np.random.default_rng(4)
    rows, extent = 515, 1024
    x, dy = rows_of(rng, rows, extent, "bf16"), ref.store("bf16", rng.standard_normal((rows, extent)))
    mean, rstd = kept("bf16", x)
    want = backward(ctx, mem, "bf16", dy, x, None, mean, rstd)
    a = [mem.put(dy), mem.put(x), None, mem.put(mean), mem.put(rstd)]
    dx, dw, db = (mem.out(np.uint16, c) for c in (rows * extent, extent, extent))
    nbytes = ctx.layer_norm_backward_workspace(L.BF16, rows, extent)
    ws = mem.out(np.uint8, nbytes)
    ctx.capture_begin()
    refused = None
    try:
        ctx.layer_norm_backward(L.BF16, *a, rows, extent, dx, dw, db)
    except Refusal as e:
        refused = e.status
    ctx.layer_norm_backward(L.BF16, *a, rows, extent, dx, dw, db, workspace=ws, workspace_bytes=nbytes)
    graph = ctx.capture_end()
    assert refused == L.REFUSE_CAPACITY
    try:
        for _ in range(3):
            for v, c in ((dx, rows * extent), (dw, extent), (db, extent)):
                v.upload(np.zeros(c, np.uint16))
            ctx.graph_launch(graph)
            ctx.synchronize()
            for v, g in zip((dx, dw, db), want):
                assert np.array_equal(mem.get(v, np.uint16, g.shape), g)
            again = backward(ctx, mem, "bf16", dy, x, None, mean, rstd)
            assert all(np.array_equal(p, q) for p, q in zip(again, want))
    finally:
        ctx.graph_destroy(graph)
