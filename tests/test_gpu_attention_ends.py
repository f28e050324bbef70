"""The attention sublayer's calls at their ends: heads of every register form,
lists that break their contract between guarded operands, many windowed
sequences."""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_norm_rotate as rotation
from test_gpu_attention_sublayer import region_of, routed
from test_gpu_norm_rotate import Case, backward, forward
from test_gpu_paged_attention import Batch, widen
from tiler_amd import _lib as L
from tiler_amd.realize import propose, realize, route
from tiler_amd.runtime import Refusal

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


MARGIN = 4096


class Guarded:
    """Storage between two margins of bytes that nothing may touch."""

    def __init__(self, ctx, nbytes, fill=0xA5):
        self.nbytes, self.fill = nbytes, fill
        self.whole = ctx.to_device(np.full(nbytes + 2 * MARGIN, fill, np.uint8))
        self.at = self.whole.offset(MARGIN)

    def reset(self):
        self.whole.upload(np.full(self.whole.nbytes, self.fill, np.uint8))

    def inside(self):
        """The bytes between the margins, which are as they were."""
        got = self.whole.download(np.uint8, (self.whole.nbytes,))
        assert (got[:MARGIN] == self.fill).all() and (got[MARGIN + self.nbytes:] == self.fill).all()
        return got[MARGIN:MARGIN + self.nbytes]


def broken_lists(rng, sequences, tokens):
    top, low = 2 ** 31 - 1, -2 ** 31
    down = np.linspace(tokens, 0, sequences + 1).astype(np.int64)
    yield down, rng.integers(0, 400, sequences)
    yield np.where(np.arange(sequences + 1) % 2, top, low), np.where(np.arange(sequences) % 2, low, top)
    yield np.r_[0, -5, np.full(sequences - 1, tokens)], np.full(sequences, top)
    yield np.r_[np.zeros(sequences, np.int64), top], np.r_[np.full(sequences - 1, -1), 4000]
    for _ in range(2):
        yield rng.integers(-10, tokens + 10, sequences + 1), rng.integers(-10, 4000, sequences)


@pytest.mark.parametrize("dim,heads,kv_heads,lengths,window,sinks", [
    (64, 4, 2, [(40, 3), (10, 50), (3, 20)], 0, 0), (128, 64, 4, [(40, 30), (1900, 50), (3, 20)], 0, 0),
    (256, 8, 2, [(2000, 1), (10, 1), (3, 1)], 0, 0), (64, 4, 2, [(2000, 9), (10, 1), (3, 90)], 70, 5),
    (64, 64, 8, [(900, 275), (3000, 257), (0, 275), (400, 265)], 1030, 3)])
def test_broken_lists_stay_inside(ctx, dim, heads, kv_heads, lengths, window, sinks):
    """starts and lengths out of order and range, in every form: nothing beside out's rows
    and the scratch is written, nothing of the inputs."""
    b = Batch(lengths, heads, kv_heads, dim, page=32, window=window, sinks=sinks, pad=4, gap=2, seed=dim)
    rng = np.random.default_rng(dim)
    row, joins = heads * dim, []
    for starts, lens in broken_lists(rng, len(lengths), b.tokens):
        b.starts, b.lengths = starts.astype(np.int32), lens.astype(np.int32)
        bufs = b.upload(ctx)
        inputs, before = bufs[:6], [x.download(np.uint8, (x.nbytes,)) for x in bufs[:6]]
        region, kw = region_of(b)
        for p in propose(*region, ctx=ctx, **kw).proposals:
            rz = p.realize(ctx)
            joins += p.symbols[1:]
            out, scratch = Guarded(ctx, b.tokens * b.out_stride * 2, 0x40), []
            for role, nbytes in rz.slots:
                if role == L.SLOT_SCRATCH:
                    scratch.append(Guarded(ctx, nbytes))
            print(p.symbols, starts, lens, flush=True)
            routed_with(ctx, rz, inputs, out.at, [s.at for s in scratch])
            rows = out.inside().view(np.uint16).reshape(b.tokens, b.out_stride)
            assert (rows[:, row:] == 0x4040).all(), p.symbols
            for s in scratch:
                s.inside()
                s.whole.free()
            out.whole.free()
            for x, was in zip(inputs, before):
                np.testing.assert_array_equal(x.download(np.uint8, was.shape), was, str(p.symbols))
        b.free()
    assert window < 1000 or any("_join_t" in j for j in joins)


def routed_with(ctx, rz, inputs, out, scratch):
    ins, spare = iter(inputs), iter(scratch)
    storage = [next(ins) if role == L.SLOT_INPUT else out if role == L.SLOT_OUTPUT else next(spare) for role, _ in rz.slots]
    route(ctx, rz, storage)
    ctx.synchronize()


def test_many_windowed_sequences(ctx):
    """Equal tiles of one sequence each, one round and a few more: those in parts, most of
    which have no rows."""
    rng = np.random.default_rng(0)
    lengths = [(int(k), int(f)) for k, f in zip(rng.integers(1300, 1400, 33), rng.integers(26, 32, 33))]
    b = Batch(lengths, 64, 8, 16, page=64, window=600, sinks=3, pad=40, gap=4, seed=33)
    want, bound = b.want()
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    offered = [p for p in propose(*region, ctx=ctx, **kw).proposals if any("_join_t" in s for s in p.symbols)]
    assert offered
    for rz in [realize(*region, ctx=ctx, **kw)] + [p.realize(ctx) for p in offered]:
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        routed(ctx, rz, [q, k, v, table, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride)))
        assert (np.abs(got[:, :1024].reshape(want.shape) - want) <= bound).all(), rz.symbols
        assert (got[:, 1024:] == 5.25).all()
    b.free()
    b.check(ctx)


def test_routed_by_its_longest_sequence(ctx):
    """A region that names its longest sequence runs what the direct call with that hint
    runs, bit for bit, in a table with room for far more."""
    for lengths in ([(3000, 1), (20, 1)], [(900, 40), (3, 2)]):
        b = Batch(lengths, 8, 2, 64, width=1500, seed=7)
        want = b.run(ctx)
        q, k, v, table, starts, lens, out = b.upload(ctx)
        region, kw = region_of(b)
        kw["scalars"] += (int(b.lengths.max()),)
        out.upload(np.zeros((b.tokens, b.out_stride), np.uint16))
        routed(ctx, realize(*region, ctx=ctx, **kw), [q, k, v, table, starts, lens], [out])
        np.testing.assert_array_equal(out.download(np.uint16, want.shape), want)
        b.free()
        b.check(ctx)


@pytest.mark.parametrize("dim", [64, 22])  # in registers, and the form of any size
def test_far_angles(ctx, dim):
    """Angles up to 2^61 keep binary32's digits: the product of position and frequency is
    the same 64 bits here and there."""
    for scale in (2.0 ** 10, 2.0 ** 20, 2.0 ** 22, 2.0 ** 25, 2.0 ** 30):
        c = Case(200, 2, 1, dim, dim, "halves", False, L.F32, far=2 ** 31 - 1, seed=dim)
        c.positions[:4] = [2 ** 31 - 1, 2 ** 24 + 1, 0, -(2 ** 31)]
        c.frequencies = c.frequencies * scale
        forward(ctx, c)
        backward(ctx, c)


def test_a_cache_without_pages(ctx):
    """As in attention, one without pages has no address; no slot names it."""
    c = Case(5, 4, 2, 64, 64, "halves", True, L.BF16, seed=1)
    wq, wk = c.upload(ctx)
    out, slots = ctx.alloc(5 * 4 * 64 * 2), ctx.to_device(np.array([-1, 0, 7, -1, 2 ** 31 - 1], np.int32))
    empty = L.PagedCache(k=None, v=None, pages=0, page=16, heads=2, head_dim=64, page_stride=2048, token_stride=128, head_stride=64)
    ctx.norm_rotate(c.dtype, c.layout(), c.d_row.ptr, c.d_row.ptr + c.part("k")[1], c.d_row.ptr + c.part("v")[1], wq, wk, c.d_pos,
                    c.d_freq, out, None, empty, slots)
    ctx.synchronize()
    want, bound = c.want("q")
    rotation.close(rotation.values(out.download(np.uint16, want.shape), L.BF16), want, bound, L.BF16, "q")
    some = L.PagedCache.from_buffer_copy(empty)
    some.pages = 1
    with pytest.raises(Refusal) as e:
        ctx.norm_rotate(c.dtype, c.layout(), c.d_row.ptr, c.d_row.ptr + c.part("k")[1], c.d_row.ptr + c.part("v")[1], wq, wk,
                        c.d_pos, c.d_freq, out, None, some, slots)
    assert e.value.status == L.REFUSE_INVALID_ARGUMENT
    for b in (out, slots):
        b.free()
    c.free()


@pytest.mark.parametrize("window,sinks", [(1 << 31, 0), (2 ** 32 - 1, 2 ** 32 - 1), (2 ** 31 - 1, 5), (40, 2 ** 32 - 1)])
def test_windows_and_sinks_past_every_length(ctx, window, sinks):
    """Each sees all that is before it: the results of no window."""
    b = Batch([(300, 1), (90, 40), (0, 3), (1500, 2)], 4, 2, 64, seed=3)
    want, bound = b.want()
    b.window, b.sinks = window, sinks
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    for p in propose(*region, ctx=ctx, **kw).proposals:
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride))).reshape(want.shape)
        assert (np.abs(got - want) <= bound).all(), p.symbols
    b.free()


@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("length", [2 ** 31 - 1024 - 700, 2 ** 31 - 1024, 2 ** 31 - 1024 + 20, 2 ** 31 - 1])
def test_positions_next_to_2_to_31(ctx, length, fresh):
    """A window at the end of the longest table, first tokens visible: what a short sequence
    of the same first and last pages gives.  Keys past the table are not seen."""
    page, width, near, window, sinks = 1024, 2 ** 21 - 1, 8, 1500, 70
    moved = (width - near) * page  # tokens between the pages that either sequence has
    b = Batch([(length - moved - fresh, fresh), (30, 2)], 6, 2, 64, page=page, window=window, sinks=sinks, seed=5, width=near)
    want, bound = b.want()
    q, k, v, _, starts, _, out = b.upload(ctx)
    table = np.full((2, width), -1, np.int32)
    table[0, 0], table[0, width - near + 1:] = b.table[0, 0], b.table[0, 1:]
    table[1, :near] = b.table[1]
    b.lengths[0], b.width = length, width
    wide, lens = ctx.to_device(table), ctx.to_device(b.lengths)
    region, kw = region_of(b)
    for p in propose(*region, ctx=ctx, **kw).proposals:
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        routed(ctx, p.realize(ctx), [q, k, v, wide, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride))).reshape(want.shape)
        assert (np.abs(got - want) <= bound).all(), p.symbols
    for x in (wide, lens):
        x.free()
    b.free()


@pytest.mark.parametrize("dim,rotary,dtype", [(128, 128, L.BF16), (90, 34, L.F32)])
def test_captured_gradients(ctx, dim, rotary, dtype):
    """The rotation and its gradients in a graph, replayed on other inputs between eager
    calls, a workspace of its own; without one the capture is refused."""
    c = Case(300, 5, 2, dim, rotary, "halves", True, dtype, seed=1)
    wq, wk = c.upload(ctx)
    heads, store = c.layout(), np.uint16 if dtype == L.BF16 else np.float32
    need = ctx.norm_rotate_backward_workspace(dtype, heads)
    shapes = [(300, 5, dim), (300, 2, dim), (300, c.stride), (300, c.stride), (dim,), (dim,)]
    # of the graph and of the eager calls: rotated queries and keys (which are their own gradients), dq and dk, dwq, dwk
    sides = [[ctx.alloc(int(np.prod(s)) * c.elem) for s in shapes] + [ctx.alloc(need)] for _ in range(2)]
    for side in sides:
        for x, s in zip(side, shapes):
            x.upload(np.zeros(s, store))

    def step(side):
        q, k, dq, dk, dwq, dwk, space = side
        ctx.norm_rotate(dtype, heads, c.d_row.ptr, c.d_row.ptr + c.part("k")[1], None, wq, wk, c.d_pos, c.d_freq, q, k)
        ctx.norm_rotate_backward(dtype, heads, q, k, c.d_row.ptr, c.d_row.ptr + c.part("k")[1], wq, wk, c.d_pos, c.d_freq,
                                 dq, dk, dwq, dwk, workspace=space, workspace_bytes=need)

    ctx.capture_begin()
    step(sides[0])
    with pytest.raises(Refusal) as e:
        ctx.norm_rotate_backward(dtype, heads, *sides[0][:2], c.d_row.ptr, c.d_row.ptr + c.part("k")[1], wq, wk, c.d_pos,
                                 c.d_freq, *sides[0][2:6])
    graph = ctx.capture_end()
    assert e.value.status == L.REFUSE_CAPACITY
    for i in range(4):
        rng = np.random.default_rng(i)
        c.d_row.upload(rotation.stored(rng.standard_normal((300, c.stride)), dtype)[0])
        c.d_pos.upload(rng.integers(0, 10 ** 6, 300).astype(np.int32))
        ctx.graph_launch(graph)
        ctx.synchronize()
        step(sides[1])
        ctx.synchronize()
        for a, b, s in zip(*sides, shapes):
            np.testing.assert_array_equal(a.download(store, s), b.download(store, s), str(i))
    ctx.graph_destroy(graph)
    for side in sides:
        for x in side:
            x.free()
    c.free()
