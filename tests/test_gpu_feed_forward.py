"""The feed-forward sublayer's calls as a program makes them: together, in
graphs, on other streams, through the adapter, and refused."""
from __future__ import annotations

import numpy as np
import pytest

import feed_forward_reference as ref
from tiler_amd import _lib as L
from tiler_amd import families
from tiler_amd.realize import propose, realize, route
from tiler_amd.runtime import Refusal
from test_gpu_layer_norm import Buffers, rows_of, within

pytestmark = pytest.mark.gpu

RE = L.PERMITS_REASSOCIATION
BF = np.uint16
EPS = ref.EPS_BITS


@pytest.fixture
def mem(ctx):
    m = Buffers(ctx)
    yield m
    m.free()


def bf(values):
    return ref.store("bf16", values)


def w64(stored):
    return ref.wide("bf16", stored)


class Sublayer:
    """y = (silu(n Wg^T) * (n Wu^T)) Wd^T with n = layer_norm(x), and its
    gradients from dy: every call of one training step, over storage of its own."""

    def __init__(self, ctx, mem, tokens, width, inner, seed):
        self.ctx, self.t, self.d, self.i = ctx, tokens, width, inner
        rng = np.random.default_rng(seed)
        t, d, i = tokens, width, inner
        self.host = {"x": rows_of(rng, t, d, "bf16"), "w": bf(rng.uniform(0.5, 1.5, d)), "b": bf(rng.normal(0, 0.1, d)),
                     "wg": bf(rng.standard_normal((i, d)) / np.sqrt(d)), "wu": bf(rng.standard_normal((i, d)) / np.sqrt(d)),
                     "wd": bf(rng.standard_normal((d, i)) / np.sqrt(i)), "dy": bf(rng.standard_normal((t, d)))}
        self.host["wdt"] = np.ascontiguousarray(self.host["wd"].T)
        self.put = {k: mem.put(v) for k, v in self.host.items()}
        self.shapes = {"n": (t, d), "h": (t, i), "gate": (t, i), "up": (t, i), "y": (t, d), "dh": (t, i), "dn": (t, d),
                       "dwg": (i, d), "dwu": (i, d), "dx": (t, d), "dw": (d,), "db": (d,)}
        self.out = {k: mem.out(BF, int(np.prod(s))) for k, s in self.shapes.items()}
        self.mean, self.rstd = mem.out(np.float32, t), mem.out(np.float32, t)
        self.bytes = max(ctx.layer_norm_backward_workspace(L.BF16, t, d),
                         ctx.gated_contract_bf16_backward_workspace(t, i, d))
        self.ws = mem.out(np.uint8, self.bytes)  # one for both: they follow one another

    def step(self, stream=None):
        c, p, o, t, d, i = self.ctx, self.put, self.out, self.t, self.d, self.i
        kw = dict(workspace=self.ws, workspace_bytes=self.bytes, stream=stream)
        c.layer_norm(L.BF16, p["x"], p["w"], p["b"], t, d, EPS, o["n"], self.mean, self.rstd, stream=stream)
        c.gated_contract_bf16(o["n"], p["wg"], p["wu"], t, i, d, o["h"], o["gate"], o["up"], stream=stream)
        c.contract_bf16(o["h"], p["wd"], t, d, i, o["y"], stream=stream)
        c.contract_bf16(p["dy"], p["wdt"], t, i, d, o["dh"], stream=stream)
        c.gated_contract_bf16_backward(o["n"], p["wg"], p["wu"], o["gate"], o["up"], o["dh"], t, i, d, o["dn"], o["dwg"],
                                       o["dwu"], **kw)
        c.layer_norm_backward(L.BF16, o["dn"], p["x"], p["w"], self.mean, self.rstd, t, d, o["dx"], o["dw"], o["db"], **kw)

    def results(self, mem):
        mem.get(self.ws, np.uint8, (self.bytes,))  # nothing written past it
        return {k: mem.get(self.out[k], BF, s) for k, s in self.shapes.items()}

    def clear(self):
        for k, s in self.shapes.items():
            self.out[k].upload(np.zeros(int(np.prod(s)), BF))


def product_bounds(a, b):
    k = a.shape[1]
    e = k * ref.U * (np.abs(a) @ np.abs(b).T)
    return e + ref.half("bf16") * (np.abs(a @ b.T) + e)


@pytest.mark.parametrize("tokens,width,inner", [(1, 64, 136), (45, 264, 520), (200, 509, 1365), (700, 512, 1024)])
def test_training_step(ctx, mem, tokens, width, inner):
    """Every result of the step against the 64-bit form of its call on what the
    calls before it left."""
    s = Sublayer(ctx, mem, tokens, width, inner, tokens)
    s.step()
    ctx.synchronize()
    r = s.results(mem)
    f = {k: w64(v) for k, v in {**r, **s.host}.items()}
    mean, rstd = (mem.get(v, np.float32, (tokens,)).astype(np.float64) for v in (s.mean, s.rstd))
    norm = (f["x"], f["w"], f["b"])
    within(f["n"], ref.layer_norm(*norm)[0], ref.layer_norm_bounds("bf16", *norm)[0], "n")
    gated = (f["n"], f["wg"], f["wu"])
    for k, v, e in zip(("h", "gate", "up"), ref.gated(*gated), ref.gated_bounds(*gated)):
        within(f[k], v, e, k)
    within(f["y"], f["h"] @ f["wd"].T, product_bounds(f["h"], f["wd"]), "y")
    within(f["dh"], f["dy"] @ f["wd"], product_bounds(f["dy"], f["wdt"]), "dh")
    back = (*gated, f["gate"], f["up"], f["dh"])
    for k, v, e in zip(("dn", "dwg", "dwu"), ref.gated_backward(*back), ref.gated_backward_bounds(*back)):
        within(f[k], v, e, k)
    grad = (f["dn"], f["x"], f["w"], mean, rstd)
    for k, v, e in zip(("dx", "dw", "db"), ref.layer_norm_backward(*grad), ref.layer_norm_backward_bounds("bf16", *grad)):
        within(f[k], v, e, k)


def test_two_captured_steps_beside_eager_ones(ctx, mem):
    """Two graphs, each with a workspace of its own, replayed in turn with eager
    steps of both between them: every replay gives the eager bits."""
    steps = [Sublayer(ctx, mem, 130, 264, 520, 1), Sublayer(ctx, mem, 77, 509, 265, 2)]
    want = []
    for s in steps:
        s.step()
        ctx.synchronize()
        want.append(s.results(mem))
    graphs = []
    try:
        for s in steps:
            ctx.capture_begin()
            s.step()
            graphs.append(ctx.capture_end())
        for _ in range(3):
            for s in steps:
                s.clear()
            for g in graphs:
                ctx.graph_launch(g)
            ctx.synchronize()
            for s, w in zip(steps, want):
                for k, v in s.results(mem).items():
                    assert np.array_equal(v, w[k]), k
            steps[0].step()
            steps[1].step()
            ctx.synchronize()
            for s, w in zip(steps, want):
                assert all(np.array_equal(v, w[k]) for k, v in s.results(mem).items())
    finally:
        for g in graphs:
            ctx.graph_destroy(g)


def test_two_streams(ctx, mem):
    """A step on another stream than the context's, beside one on its own."""
    import tiler_amd
    other = tiler_amd.Context(0)
    try:
        a, b = Sublayer(ctx, mem, 300, 512, 1024, 3), Sublayer(ctx, mem, 90, 264, 520, 4)
        want = []
        for s in (a, b):
            s.step()
            ctx.synchronize()
            want.append(s.results(mem))
            s.clear()
        ctx.synchronize()
        for _ in range(5):
            a.step()
            b.step(stream=other.stream)
        ctx.synchronize()
        other.synchronize()
        for s, w in zip((a, b), want):
            assert all(np.array_equal(v, w[k]) for k, v in s.results(mem).items())
        # without a workspace: an allocation on the stream it is given
        p, o = b.put, b.out
        o["dn"].upload(np.zeros(b.t * b.d, BF))
        ctx.synchronize()
        ctx.gated_contract_bf16_backward(o["n"], p["wg"], p["wu"], o["gate"], o["up"], o["dh"], b.t, b.i, b.d, o["dn"],
                                         o["dwg"], o["dwu"], stream=other.stream)
        other.synchronize()
        assert all(np.array_equal(v, want[1][k]) for k, v in b.results(mem).items())
    finally:
        other.close()


def test_quantized_layer_behind_a_norm(ctx, mem):
    """layer_norm, its rows in 8 bits, the 8-bit product, captured and replayed."""
    rng = np.random.default_rng(5)
    t, d, n = 77, 500, 264
    x, w = rows_of(rng, t, d, "bf16"), rng.standard_normal((n, d)).astype(np.float32)
    y, q, s = mem.out(BF, t * d), mem.out(np.int8, t * d), mem.out(np.float32, t)
    wq, ws, c = mem.out(np.int8, n * d), mem.out(np.float32, n), mem.out(BF, t * n)
    dx = mem.put(x)
    ctx.quantize_rows_i8(L.F32, mem.put(w), n, d, wq, ws)
    ctx.synchronize()

    def forward():
        ctx.layer_norm(L.BF16, dx, None, None, t, d, EPS, y)
        ctx.quantize_rows_i8(L.BF16, y, t, d, q, s)
        ctx.contract_i8(q, wq, s, ws, t, n, d, L.BF16, c)

    ctx.capture_begin()
    forward()
    graph = ctx.capture_end()
    try:
        for _ in range(3):
            c.upload(np.zeros(t * n, BF))
            ctx.graph_launch(graph)
            ctx.synchronize()
            got, ny = mem.get(c, BF, (t, n)), mem.get(y, BF, (t, d))
            (eq, es), (ewq, ews) = ref.quantize_rows(w64(ny)), ref.quantize_rows(w)
            assert np.array_equal(got, bf(ref.contract_i8(eq, ewq, es, ews)))
            forward()
            ctx.synchronize()
            assert np.array_equal(mem.get(c, BF, (t, n)), got)
    finally:
        ctx.graph_destroy(graph)


def test_host_functions(ctx):
    rng = np.random.default_rng(8)
    t, d, i = 33, 100, 72
    for dtype in ("bf16", "f32"):
        x, w, b = rows_of(rng, t, d, dtype), ref.store(dtype, rng.uniform(0.5, 1.5, d)), ref.store(dtype, rng.normal(0, 1, d))
        y, mean, rstd = families.layer_norm(x, w, b, EPS, ctx=ctx)
        args = [ref.wide(dtype, v) for v in (x, w, b)]
        within(ref.wide(dtype, y), ref.layer_norm(*args)[0], ref.layer_norm_bounds(dtype, *args)[0], "y")
        dy = ref.store(dtype, rng.standard_normal((t, d)))
        args = (ref.wide(dtype, dy), args[0], args[1], mean.astype(np.float64), rstd.astype(np.float64))
        for g, v, e in zip(families.layer_norm_backward(dy, x, w, mean, rstd, ctx=ctx), ref.layer_norm_backward(*args),
                           ref.layer_norm_backward_bounds(dtype, *args)):
            within(ref.wide(dtype, g), v, e, dtype)
        q, s = families.quantize_rows_i8(x, ctx=ctx)
        eq, es = ref.quantize_rows(ref.wide(dtype, x))
        assert np.array_equal(q, eq) and np.array_equal(s, es)
        for out in (np.float32, np.uint16):
            want = ref.contract_i8(eq, eq, es, es)
            got = families.contract_i8(q, q, s, s, out, ctx=ctx)
            assert np.array_equal(got, want if out == np.float32 else bf(want))
    x, wg, wu = bf(rng.standard_normal((t, d))), bf(rng.standard_normal((i, d)) / 10), bf(rng.standard_normal((i, d)) / 10)
    args = [w64(v) for v in (x, wg, wu)]
    h, gate, up = families.gated_contract_bf16(x, wg, wu, ctx=ctx)
    for g, v, e in zip((h, gate, up), ref.gated(*args), ref.gated_bounds(*args)):
        within(w64(g), v, e, "gated")
    dh = bf(rng.standard_normal((t, i)))
    args += [w64(v) for v in (gate, up, dh)]
    for g, v, e in zip(families.gated_contract_bf16_backward(x, wg, wu, gate, up, dh, ctx=ctx), ref.gated_backward(*args),
                       ref.gated_backward_bounds(*args)):
        within(w64(g), v, e, "gradients")
    assert families.layer_norm(np.zeros((0, 8), np.uint16), ctx=ctx)[0].shape == (0, 8)


# -- the adapter --------------------------------------------------------------

def routed(ctx, mem, rz, inputs, outputs):
    ins, outs = iter(inputs), iter(outputs)
    storage = [next(ins) if role == L.SLOT_INPUT else next(outs) if role == L.SLOT_OUTPUT else None for role, _ in rz.slots]
    route(ctx, rz, storage)


def proposals(ctx, program, extents, **kw):
    """What realize gives, and every proposal's realization."""
    offer = propose(program, extents, permissions=RE, ctx=ctx, **kw)
    assert offer.proposals and not offer.declined
    for flags in (0, L.REGION_ALIGNED16):
        yield realize(program, extents, permissions=RE, flags=flags, ctx=ctx, **kw)
    for p in offer.proposals:
        yield p.realize(ctx)


@pytest.mark.parametrize("rows,extent", [(5, 100), (600, 512), (3, 20000)])
def test_routed_layer_norm(ctx, mem, rows, extent):
    rng = np.random.default_rng(rows)
    x, w, b = rows_of(rng, rows, extent, "bf16"), bf(rng.uniform(0.5, 1.5, extent)), bf(rng.standard_normal(extent))
    dy = bf(rng.standard_normal((rows, extent)))
    dx_, dw_, db_, ddy = mem.put(x), mem.put(w), mem.put(b), mem.put(dy)
    want = [mem.out(BF, rows * extent), mem.out(np.float32, rows), mem.out(np.float32, rows)]
    ctx.layer_norm(L.BF16, dx_, dw_, db_, rows, extent, EPS, *want)
    grads = [mem.out(BF, rows * extent), mem.out(BF, extent), mem.out(BF, extent)]
    ctx.layer_norm_backward(L.BF16, ddy, dx_, dw_, want[1], want[2], rows, extent, *grads)
    ctx.synchronize()
    want_h = [mem.get(v, BF if k == 0 else np.float32, (rows, extent) if k == 0 else (rows,)) for k, v in enumerate(want)]
    grads_h = [mem.get(v, BF, (rows, extent) if k == 0 else (extent,)) for k, v in enumerate(grads)]
    for rz in proposals(ctx, L.PROGRAM_LAYER_NORM, (rows, extent), dtype=L.BF16, scalars=(EPS, 0),
                        variant=L.NORM_WEIGHT | L.NORM_BIAS | L.NORM_STATISTICS):
        got = [mem.out(BF, rows * extent), mem.out(np.float32, rows), mem.out(np.float32, rows)]
        routed(ctx, mem, rz, [dx_, dw_, db_], got)
        for v, h in zip(got, want_h):
            assert np.array_equal(mem.get(v, h.dtype, h.shape), h)
    for rz in proposals(ctx, L.PROGRAM_LAYER_NORM_BACKWARD, (rows, extent), dtype=L.BF16,
                        variant=L.NORM_WEIGHT | L.NORM_DX | L.NORM_DW | L.NORM_DB):
        got = [mem.out(BF, rows * extent), mem.out(BF, extent), mem.out(BF, extent)]
        routed(ctx, mem, rz, [ddy, dx_, dw_, want[1], want[2]], got)
        for v, h in zip(got, grads_h):
            assert np.array_equal(mem.get(v, BF, h.shape), h)


@pytest.mark.parametrize("m,n,k", [(5, 100, 64), (300, 520, 264), (70, 200, 333)])
def test_routed_gated_contraction(ctx, mem, m, n, k):
    rng = np.random.default_rng(m)
    whole = lambda *s: bf(rng.integers(-2, 3, s))  # sums below 2^24: any form's bits
    x, wg, wu, dh = whole(m, k), whole(n, k), whole(n, k), whole(m, n)
    a = [mem.put(v) for v in (x, wg, wu)]
    ddh = mem.put(dh)
    want = [mem.out(BF, m * n) for _ in range(3)]
    ctx.gated_contract_bf16(*a, m, n, k, *want)
    ctx.synchronize()
    want_h = [mem.get(v, BF, (m, n)) for v in want]
    for rz in proposals(ctx, L.PROGRAM_GATED_CONTRACTION, (m, n, k), dtype=L.BF16, variant=L.GATED_KEEP):
        got = [mem.out(BF, m * n) for _ in range(3)]
        routed(ctx, mem, rz, a, got)
        assert all(np.array_equal(mem.get(v, BF, (m, n)), h) for v, h in zip(got, want_h))
    f = [w64(v) for v in (x, wg, wu, want_h[1], want_h[2], dh)]
    for rz in proposals(ctx, L.PROGRAM_GATED_CONTRACTION_BACKWARD, (m, n, k), dtype=L.BF16, variant=L.GATED_DX | L.GATED_DW):
        got = [mem.out(BF, m * k), mem.out(BF, n * k), mem.out(BF, n * k)]
        routed(ctx, mem, rz, [*a, want[1], want[2], ddh], got)
        for v, shape, r, e in zip(got, ((m, k), (n, k), (n, k)), ref.gated_backward(*f), ref.gated_backward_bounds(*f)):
            within(w64(mem.get(v, BF, shape)), r, e, rz.symbols)


@pytest.mark.parametrize("m,n,k", [(5, 100, 64), (300, 520, 272), (70, 200, 333)])
def test_routed_int8(ctx, mem, m, n, k):
    rng = np.random.default_rng(m)
    x, w = bf(rng.standard_normal((m, k))), rng.integers(-127, 128, (n, k)).astype(np.int8)
    sw = rng.uniform(0.01, 1, n).astype(np.float32)
    eq, es = ref.quantize_rows(w64(x))
    for rz in proposals(ctx, L.PROGRAM_QUANTIZE_ROWS_I8, (m, k), dtype=L.BF16):
        q, s = mem.out(np.int8, m * k), mem.out(np.float32, m)
        routed(ctx, mem, rz, [mem.put(x)], [q, s])
        assert np.array_equal(mem.get(q, np.int8, (m, k)), eq) and np.array_equal(mem.get(s, np.float32, (m,)), es)
    for rz in proposals(ctx, L.PROGRAM_CONTRACTION_I8, (m, n, k), dtype=L.F32):
        c = mem.out(np.float32, m * n)
        routed(ctx, mem, rz, [mem.put(eq), mem.put(w), mem.put(es), mem.put(sw)], [c])
        assert np.array_equal(mem.get(c, np.float32, (m, n)), ref.contract_i8(eq, w, es, sw))


# -- refusals: nothing is launched, the outputs stay as they were ---------------

def refused(call, status):
    with pytest.raises(Refusal) as e:
        call()
    assert e.value.status == status, str(e.value)


def test_refusals(ctx, mem):
    m, n, k = 40, 72, 64
    v = [mem.put(np.zeros(8192, np.uint16)) for _ in range(6)]
    st = [mem.put(np.ones(m, np.float32)) for _ in range(2)]
    o = [mem.out(BF, 8192) for _ in range(3)]
    bad, cap, unsupported = L.REFUSE_INVALID_ARGUMENT, L.REFUSE_CAPACITY, L.REFUSE_UNSUPPORTED
    # halves of a pair
    refused(lambda: ctx.layer_norm(L.BF16, v[0], None, None, m, k, EPS, o[0], mean=st[0]), bad)
    refused(lambda: ctx.layer_norm(L.BF16, v[0], None, None, m, k, EPS, o[0], rstd=st[0]), bad)
    refused(lambda: ctx.gated_contract_bf16(*v[:3], m, n, k, o[0], gate=o[1]), bad)
    refused(lambda: ctx.gated_contract_bf16_backward(*v, m, n, k, o[0], dwg=o[1]), bad)
    # operands that are missing
    refused(lambda: ctx.layer_norm(L.BF16, None, None, None, m, k, EPS, o[0]), bad)
    refused(lambda: ctx.layer_norm(L.BF16, v[0], None, None, m, k, EPS, None), bad)
    refused(lambda: ctx.layer_norm_backward(L.BF16, None, v[1], None, *st, m, k, o[0]), bad)
    refused(lambda: ctx.layer_norm_backward(L.BF16, v[0], v[1], None, st[0], None, m, k, o[0]), bad)
    refused(lambda: ctx.gated_contract_bf16(v[0], v[1], None, m, n, k, o[0]), bad)
    for i in range(6):
        refused(lambda: ctx.gated_contract_bf16_backward(*v[:i], None, *v[i + 1:], m, n, k, o[0], o[1], o[2]), bad)
    refused(lambda: ctx.quantize_rows_i8(L.BF16, v[0], m, k, o[0], None), bad)
    refused(lambda: ctx.contract_i8(v[0], v[1], None, st[0], m, n, k, L.F32, o[0]), bad)
    # types and sizes
    refused(lambda: ctx.layer_norm(2, v[0], None, None, m, k, EPS, o[0]), unsupported)
    refused(lambda: ctx.layer_norm(L.BF16, v[0], None, None, m, k, 0, o[0]), bad)
    refused(lambda: ctx.layer_norm(L.BF16, v[0], None, None, 1, 1 << 32, EPS, o[0]), cap)
    refused(lambda: ctx.gated_contract_bf16(*v[:3], m, n, 0, o[0]), bad)
    refused(lambda: ctx.gated_contract_bf16(*v[:3], m, n, 1 << 24, o[0]), cap)
    refused(lambda: ctx.gated_contract_bf16_backward(*v, m, 1 << 22, k, o[0]), cap)
    refused(lambda: ctx.gated_contract_bf16_backward(*v, m, n, 1 << 22, o[0]), cap)
    refused(lambda: ctx.contract_i8(v[0], v[1], *st, m, n, 131072, L.F32, o[0]), cap)
    refused(lambda: ctx.contract_i8(v[0], v[1], *st, m, n, k, 2, o[0]), unsupported)
    # workspaces: unaligned, too small
    for call, need in ((lambda **kw: ctx.layer_norm_backward(L.BF16, v[0], v[1], None, *st, m, k, o[0], o[1], **kw),
                        ctx.layer_norm_backward_workspace(L.BF16, m, k)),
                       (lambda **kw: ctx.gated_contract_bf16_backward(*v, m, n, k, o[0], **kw), 2 * m * 128 * 2)):
        ws = mem.out(np.uint8, 1 << 20)
        refused(lambda: call(workspace=ws.offset(8), workspace_bytes=1 << 19), bad)
        refused(lambda: call(workspace=ws, workspace_bytes=need // 2), cap)
        mem.get(ws, np.uint8, (1 << 20,))
        assert (ws.download(np.uint8, (1 << 20,)) == 0xA5).all()
    ctx.synchronize()
    assert all((b.download(np.uint8, (16384,)) == 0xA5).all() for b in o)


def test_capture_refuses_without_a_workspace(ctx, mem):
    s = Sublayer(ctx, mem, 40, 64, 72, 6)
    p, o = s.put, s.out
    s.step()
    ctx.synchronize()
    want = s.results(mem)
    ctx.capture_begin()
    status = None
    try:
        ctx.gated_contract_bf16_backward(o["n"], p["wg"], p["wu"], o["gate"], o["up"], o["dh"], s.t, s.i, s.d, o["dn"])
    except Refusal as e:
        status = e.status
    s.step()  # the capture goes on
    graph = ctx.capture_end()
    assert status == L.REFUSE_CAPACITY
    try:
        for _ in range(2):
            s.clear()
            ctx.graph_launch(graph)
            ctx.synchronize()
            assert all(np.array_equal(v, want[k]) for k, v in s.results(mem).items())
    finally:
        ctx.graph_destroy(graph)


def test_offsets_past_32_bits(ctx, mem):
    """Rows and products whose element offsets pass 2^32: the last row of x and
    of y, the last rows of an 8-bit product's left operand."""
    rows, extent = (1 << 20) + 3, 4112
    big = ctx.alloc(rows * extent * 2)
    try:
        rng = np.random.default_rng(7)
        tail = rows_of(rng, 4, extent, "bf16")
        at = (rows - 4) * extent * 2
        big.offset(at).upload(tail)
        y, mean, rstd = ctx.alloc(rows * extent * 2), ctx.alloc(rows * 4), ctx.alloc(rows * 4)
        try:
            ctx.layer_norm(L.BF16, big, None, None, rows, extent, EPS, y, mean, rstd)
            ctx.synchronize()
            got = y.offset(at).download(BF, (4, extent))
            args = (w64(tail), None, None)
            within(w64(got), ref.layer_norm(*args)[0], ref.layer_norm_bounds("bf16", *args)[0], "y")
            # the same storage as 8-bit rows: 2^33 codes of a and more
            m = rows * 2 - 8
            a = rng.integers(-127, 128, (8, extent)).astype(np.int8)
            b = rng.integers(-127, 128, (3, extent)).astype(np.int8)
            big.offset((m - 8) * extent).upload(a)
            ones = ctx.to_device(np.ones(m, np.float32))
            c = ctx.alloc(m * 3 * 4)
            try:
                ctx.contract_i8(big, mem.put(b), ones, ones, m, 3, extent, L.F32, c)
                ctx.synchronize()
                last = c.offset((m - 8) * 3 * 4).download(np.float32, (8, 3))
                assert np.array_equal(last, (a.astype(np.float64) @ b.astype(np.float64).T).astype(np.float32))
            finally:
                ones.free()
                c.free()
        finally:
            for v in (y, mean, rstd):
                v.free()
    finally:
        big.free()
