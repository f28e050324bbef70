"""The attention sublayer's calls as a server makes them: page tables, rotation
with the store into the cache and attention, one after another, captured, on other
streams, through the recognizer's programs and the host functions; and what the
calls refuse."""
from __future__ import annotations

import numpy as np
import pytest

import attention_reference as ref
import oracle
import tiler_amd
from attention_reference import U16
from test_gpu_norm_rotate import Case, backward, forward
from test_gpu_paged_attention import Batch, bf16, widen
from tiler_amd import _lib as L
from tiler_amd import families
from tiler_amd.realize import propose, realize, route
from tiler_amd.runtime import Refusal

pytestmark = pytest.mark.gpu
RE = L.PERMITS_REASSOCIATION
EPS_BITS = 0x358637BD
EPS = float(np.uint32(EPS_BITS).view(np.float32))


class Server:
    """Sequences of one layer's cache on the device, their tokens one step after
    another, and the same in 64 bits."""

    def __init__(self, ctx, sequences, heads, kv_heads, dim, page, pages, width, rows, window=0, sinks=0, seed=0, fresh=None,
                 longest=None):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.n, self.heads, self.kv_heads, self.dim = ctx, sequences, heads, kv_heads, dim
        self.page, self.pages, self.width, self.rows, self.window, self.sinks = page, pages, width, rows, window, sinks
        self.stride = (heads + 2 * kv_heads) * dim
        self.free = rng.permutation(pages).astype(np.int32)
        self.frequencies = 10000.0 ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
        self.w_up, self.w = bf16(1 + 0.1 * rng.standard_normal((2, dim)))
        self.kept = np.zeros(sequences, np.int32)
        self.table = np.full((sequences, width), -1, np.int32)
        put, i32 = ctx.to_device, np.int32
        self.row = ctx.alloc(rows * self.stride * 2)
        self.q, self.out = ctx.alloc(rows * heads * dim * 2), ctx.alloc(rows * heads * dim * 2)
        self.d_free, self.d_table, self.d_w, self.d_f = put(self.free), put(self.table), put(self.w_up), put(self.frequencies)
        self.d_kept, self.d_fresh, self.lengths = (put(np.zeros(sequences, i32)) for _ in range(3))
        self.starts, self.positions, self.slots, self.taken = (put(np.zeros(c, i32)) for c in (sequences + 1, rows, rows, 1))
        fill = bf16(rng.standard_normal((2, pages, page, kv_heads, dim)))[0]
        self.k, self.v = put(fill[0]), put(fill[1])
        self.cache = L.PagedCache(k=self.k.ptr, v=self.v.ptr, pages=pages, page=page, heads=kv_heads, head_dim=dim,
                                  page_stride=page * kv_heads * dim, token_stride=kv_heads * dim, head_stride=dim)
        self.layout = L.HeadLayout(tokens=rows, q_heads=heads, kv_heads=kv_heads, head_dim=dim, rotary=dim,
                                   pairing=L.ROTATE_HALVES, eps_bits=EPS_BITS, q_stride=self.stride, k_stride=self.stride,
                                   v_stride=self.stride, q_out_stride=heads * dim, k_out_stride=kv_heads * dim)
        self.shape = L.AttentionShape(tokens=rows, sequences=sequences, q_heads=heads, scale=dim ** -0.5,
                                      q_stride=heads * dim, out_stride=heads * dim, table_width=width, window=window,
                                      sinks=sinks, max_fresh=fresh or rows, max_length=longest or width * page)
        self.need = ctx.paged_attention_bf16_workspace(self.shape, self.cache)
        self.space = ctx.alloc(max(self.need, 1))
        self.used = 0
        self.history = [[] for _ in range(sequences)]  # (row of k, row of v, bound of k) a token

    def close(self):
        for b in vars(self).copy().values():
            if isinstance(b, type(self.row)):
                b.free()

    def fill_table(self):
        """Pages of their own for every row of the table; the free ones are the rest."""
        named = self.n * self.width
        self.table = np.arange(named, dtype=np.int32).reshape(self.n, self.width)
        self.free = (named + np.arange(self.pages - named)).astype(np.int32)
        self.d_table.upload(self.table)
        self.d_free.upload(self.free)

    def load(self, fresh, kept=None, seed=None):
        """The next step's lists and projections on the device."""
        rng = self.rng if seed is None else np.random.default_rng(seed)
        self.fresh = np.array(fresh, np.int32)
        if kept is not None:
            self.kept = np.array(kept, np.int32)
        self.row_up, self.row_64 = bf16(rng.standard_normal((self.rows, self.stride)))
        self.row.upload(self.row_up)
        self.d_kept.upload(self.kept)
        self.d_fresh.upload(self.fresh)
        self.out.upload(bf16(np.full(self.rows * self.heads * self.dim, 5.25))[0])

    def step(self, stream=None, free=None, count=None):
        c, d, at = self.ctx, self.dim, self.row.ptr
        free = self.d_free.ptr + 4 * self.used if free is None else free
        c.page_slots(self.d_kept, self.d_fresh, self.n, self.page, free, len(self.free) - self.used if count is None else count,
                     self.d_table, self.width, self.rows, self.starts, self.lengths, self.positions, self.slots, self.taken,
                     stream=stream)
        c.norm_rotate(L.BF16, self.layout, at, at + 2 * self.heads * d, at + 2 * (self.heads + self.kv_heads) * d,
                      self.d_w.ptr, self.d_w.ptr + 2 * d, self.positions, self.d_f, self.q, None, self.cache, self.slots,
                      stream=stream)
        c.paged_attention_bf16(self.shape, self.q, self.cache, self.d_table, self.starts, self.lengths, self.out,
                               workspace=self.space, workspace_bytes=self.need, stream=stream)

    def got(self):
        return self.out.download(np.uint16, (self.rows, self.heads, self.dim))

    def check(self):
        """The step's lists, cache and results; then its tokens are kept."""
        n, rows, d, page = self.n, self.rows, self.dim, self.page
        table, starts, lengths, positions, slots, taken = ref.page_slots(
            self.kept, self.fresh, page, self.free[self.used:], self.table, rows)
        for buf, want in ((self.d_table, table), (self.starts, starts), (self.lengths, lengths), (self.positions, positions),
                          (self.slots, slots)):
            np.testing.assert_array_equal(buf.download(np.int32, want.shape), want)
        assert self.taken.download(np.int32, (1,))[0] == taken
        at = self.heads * d
        turn = (positions, self.frequencies, d, "halves", EPS)
        q, q_bound = ref.norm_rotate(self.row_64[:, :at].reshape(rows, self.heads, d), self.w[0], *turn)
        k, k_bound = ref.norm_rotate(self.row_64[:, at:at + self.kv_heads * d].reshape(rows, self.kv_heads, d), self.w[1], *turn)
        v = self.row_64[:, at + self.kv_heads * d:].reshape(rows, self.kv_heads, d)
        q_got = widen(self.q.download(np.uint16, (rows, self.heads, d)))
        assert (np.abs(q_got - q) <= q_bound + U16 * (np.abs(q) + q_bound)).all()
        for s in range(n):
            self.history[s] = self.history[s][:self.kept[s]]
            self.history[s] += [(k[r], v[r], k_bound[r]) for r in range(starts[s], starts[s + 1])]
        cached = [widen(b.download(np.uint16, (self.pages, page, self.kv_heads, d))) for b in (self.k, self.v)]
        for s in range(n):
            for j, (k_row, v_row, off) in enumerate(self.history[s]):
                where = table[s, j // page], j % page
                assert (np.abs(cached[0][where] - k_row) <= off + U16 * (np.abs(k_row) + off)).all(), (s, j)
                assert (cached[1][where] == v_row).all(), (s, j)
        want, bound = ref.paged_attention(q_got, *cached, table, starts, lengths, np.float32(d ** -0.5).astype(np.float64),
                                          self.window, self.sinks, np.full((rows, self.heads, d), 5.25))
        off = np.abs(widen(self.got()) - want)
        assert (off <= bound).all(), f"worst {np.nanmax(off / np.maximum(bound, 1e-30))} of the bound"
        self.table, self.kept, self.used = table, lengths, self.used + taken


@pytest.mark.parametrize("heads,kv_heads,dim,page,window,sinks", [
    (8, 2, 64, 16, 0, 0), (4, 4, 128, 8, 40, 4), (6, 1, 80, 5, 0, 0), (4, 2, 256, 32, 33, 0)])
def test_served_sequences(ctx, heads, kv_heads, dim, page, window, sinks):
    """Prompts, chunks beside decodes, decodes, a draft taken back, a sequence that
    ends and one that takes its place."""
    s = Server(ctx, 4, heads, kv_heads, dim, page, 400 // page, 200 // page, 100, window, sinks, seed=dim)
    for fresh, kept in (([70, 0, 1, 20], None), ([1, 45, 1, 30], None), ([1, 1, 1, 1], None), ([5, 0, 5, 3], None),
                        ([1, 2, 1, 1], [72, 45, 4, 54]),  # four, none, four and none of the last taken back
                        ([1, 1, 30, 1], [73, 47, 0, 55])):  # the third begins anew on its pages
        s.load(fresh, kept)
        s.step()
        ctx.synchronize()
        s.check()
    s.close()


def test_a_large_step(ctx):
    """Tokens enough that a workgroup takes several at a time."""
    s = Server(ctx, 4, 4, 2, 64, 16, 200, 90, 2100, seed=6)
    for fresh in ([1050, 3, 0, 1040], [1, 60, 900, 0]):
        s.load(fresh)
        s.step()
        ctx.synchronize()
        s.check()
    s.close()


@pytest.mark.parametrize("tokens", [1025, 2051, 4100])
def test_rotation_of_several_tokens_a_workgroup(ctx, tokens):
    for dim, rotary, pairing, dtype in ((64, 64, "halves", L.BF16), (40, 16, "neighbours", L.F32), (22, 6, "halves", L.BF16)):
        forward(ctx, Case(tokens, 3, 1, dim, rotary, pairing, True, dtype, seed=tokens))
        backward(ctx, Case(tokens, 3, 1, dim, rotary, pairing, True, dtype, seed=tokens))


@pytest.mark.parametrize("sequences", [64, 65, 200])
def test_many_sequences_in_every_form(ctx, sequences):
    """More than a wave's worth of them, many of no new tokens: each tile finds its own."""
    rng = np.random.default_rng(sequences)
    lengths = [(int(k), int(f)) for k, f in zip(rng.integers(0, 90, sequences), rng.integers(-8, 9, sequences).clip(0))]
    b = Batch(lengths, 6, 2, 64, page=8, pad=4, seed=sequences)
    want, bound = b.want()
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    for p in propose(*region, ctx=ctx, **kw).proposals:
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride))).reshape(want.shape)
        assert (np.abs(got - want) <= bound).all(), p.symbols
    b.free()


@pytest.mark.parametrize("rows,fresh,kept,most,longest", [
    (8, [[1, 1, 1, 1, 1], [1, 0, 1, 1, 0], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]],
     [[1300, 3, 0, 640, 17], [1301, 4, 1, 641, 18], [1301, 5, 2, 641, 18], [1302, 5, 2, 642, 18]], 1, 1400),
    (130, [[120, 3, 1, 1, 0], [1, 60, 0, 0, 69], [128, 0, 1, 0, 1], [26, 26, 26, 26, 26]],
     [[1000, 3, 0, 640, 17], [1120, 6, 1, 641, 17], [0, 66, 1, 641, 86], [40, 66, 2, 641, 87]], 130, 1400)])
def test_captured_steps(ctx, rows, fresh, kept, most, longest):
    """One graph, replayed with other lists and projections, eager steps of another
    server between: the bits of an eager step on the same lists."""
    a = Server(ctx, 5, 8, 2, 64, 16, 510, 90, rows, seed=1, fresh=most, longest=longest)
    b = Server(ctx, 5, 8, 2, 64, 16, 510, 90, rows, seed=1, fresh=most, longest=longest)
    beside = Server(ctx, 3, 4, 1, 128, 8, 60, 20, 40, seed=2)
    assert a.need > 0  # parts of the keys: a workspace
    for s in (a, b):
        s.fill_table()
    a.load(fresh[0], kept[0], seed=0)
    ctx.capture_begin()
    a.step(free=a.d_free.ptr, count=60)
    graph = ctx.capture_end()
    try:
        for i, (f, n) in enumerate(zip(fresh, kept)):
            a.load(f, n, seed=i)
            b.load(f, n, seed=i)
            if i:  # a page is handed out once: the list goes on behind the taken ones
                left = np.roll(a.d_free.download(np.int32, a.free.shape), -b.taken.download(np.int32, (1,))[0])
                a.d_free.upload(left)
                b.d_free.upload(left)
            ctx.graph_launch(graph)
            ctx.synchronize()
            beside.load([20, 1, 3], [9, 9, 9])
            beside.step()
            b.step(free=b.d_free.ptr, count=60)
            ctx.synchronize()
            for p, q in ((a.out, b.out), (a.k, b.k), (a.v, b.v), (a.d_table, b.d_table), (a.slots, b.slots)):
                np.testing.assert_array_equal(p.download(np.uint8, (p.nbytes,)), q.download(np.uint8, (q.nbytes,)), str(i))
            ends = int(b.starts.download(np.int32, (6,))[-1])
            assert (widen(a.got())[ends:] == 5.25).all()
    finally:
        ctx.graph_destroy(graph)
        for s in (a, b, beside):
            s.close()


def test_a_capture_without_a_workspace_is_refused(ctx):
    b = Batch([(3000, 1), (10, 1)], 4, 2, 64, seed=1)
    want = b.run(ctx)
    q, k, v, table, starts, lengths, out = b.upload(ctx)
    shape, cache = b.shape(), b.cache(k.ptr, v.ptr)
    need = ctx.paged_attention_bf16_workspace(shape, cache)
    space = ctx.alloc(need)
    ctx.capture_begin()
    status = None
    try:
        ctx.paged_attention_bf16(shape, q, cache, table, starts, lengths, out)
    except Refusal as e:
        status = e.status
    ctx.paged_attention_bf16(shape, q, cache, table, starts, lengths, out, workspace=space, workspace_bytes=need)
    graph = ctx.capture_end()
    assert need > 0 and status == L.REFUSE_CAPACITY
    for _ in range(3):
        out.upload(np.zeros((b.tokens, b.out_stride), np.uint16))
        ctx.graph_launch(graph)
        ctx.synchronize()
        np.testing.assert_array_equal(out.download(np.uint16, (b.tokens, b.out_stride)), want)
    ctx.graph_destroy(graph)
    space.free()
    b.free()


def test_two_streams(ctx):
    """Steps on another context's stream beside steps on this one's, a workspace each."""
    other = tiler_amd.Context(0)
    servers = [Server(ctx, 5, 8, 2, 64, 16, 510, 90, 8, seed=3, fresh=1, longest=1400),
               Server(ctx, 3, 16, 2, 128, 32, 190, 50, 90, seed=4)]
    try:
        want = []
        for s, fresh, kept in zip(servers, ([1, 1, 1, 1, 1], [30, 2, 58]), ([1300, 3, 0, 640, 17], [900, 1, 0])):
            s.fill_table()
            s.load(fresh, kept, seed=5)
            s.step()
            ctx.synchronize()
            want.append(s.got())
            want[-1][sum(fresh):] = 0  # rows of no sequence stay
            s.out.upload(np.zeros(s.out.nbytes, np.uint8))
        ctx.synchronize()
        for _ in range(5):
            servers[0].step()
            servers[1].step(stream=other.stream)
        ctx.synchronize()
        other.synchronize()
        for s, w in zip(servers, want):
            np.testing.assert_array_equal(s.got(), w)
        s = servers[1]  # without a workspace, on the other stream
        s.out.upload(np.zeros(s.out.nbytes, np.uint8))
        ctx.synchronize()
        ctx.paged_attention_bf16(s.shape, s.q, s.cache, s.d_table, s.starts, s.lengths, s.out, stream=other.stream)
        other.synchronize()
        np.testing.assert_array_equal(s.got()[:90], want[1][:90])
    finally:
        for s in servers:
            s.close()
        other.close()


# -- tiles of 256 rows, and forms at their edges ----------------------------------
def region_of(b):
    """A batch's program and extents, and what else names its region."""
    row = b.kv_heads * b.dim
    return ((L.PROGRAM_PAGED_ATTENTION, (b.tokens, len(b.lengths), b.width, b.pages, b.page, b.kv_heads, b.heads, b.dim)),
            dict(dtype=L.BF16, strides=(b.q_stride, b.out_stride, b.page * row, row, b.dim), permissions=RE,
                 grouping=(b.window, b.sinks, max(b.fresh)), scalars=(int(np.float32(b.scale).view(np.uint32)),)))


@pytest.mark.parametrize("dim", [8, 64, 80, 96, 104, 128, 160, 256])
@pytest.mark.parametrize("heads,kv_heads,lengths,page,window,sinks", [
    (6, 2, [(90, 170), (0, 5), (300, 0), (7, 93)], 24, 0, 0), (28, 4, [(90, 17), (700, 5), (2, 60)], 24, 100, 5),
    (3, 1, [(1500, 260), (0, 3), (1100, 90)], 64, 900, 70), (4, 2, [(40, 1), (2000, 1), (0, 1), (31, 2)], 16, 0, 0)])
def test_every_form(ctx, dim, heads, kv_heads, lengths, page, window, sinks):
    """The same batch in every form that is offered for it, parts of the keys among them."""
    b = Batch(lengths, heads, kv_heads, dim, page=page, pad=3, gap=4, window=window, sinks=sinks, seed=dim)
    want, bound = b.want()
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    offer = propose(*region, ctx=ctx, **kw)
    assert [p.symbols[0].rstrip("0123456789") for p in offer.proposals] == [
        "tiler_paged_attention_bf16_" + f for f in ("few", "t128_d", "t256_d")[:2 if dim > 128 else 3]]
    for p in offer.proposals:
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride)))
        off = np.abs(got[:, :heads * dim].reshape(want.shape) - want)
        assert (off <= bound).all(), f"{p.symbols}: worst {np.nanmax(off / np.maximum(bound, 1e-30))} of the bound"
        assert (got[:, heads * dim:] == 5.25).all(), p.symbols
    b.free()


def test_rows_before_the_first_sequence(ctx):
    """starts[0] above zero: the rows before it are no sequence's and stay, in every form
    and where parts are joined."""
    for lengths in ([(1900, 40), (0, 3)], [(20, 9), (70, 1)]):
        b = Batch(lengths, 4, 2, 64, page=16, seed=3, width=130, pad=9)
        b.starts = b.starts + 5
        want, bound = b.want()
        q, k, v, table, starts, lens, out = b.upload(ctx)
        region, kw = region_of(b)
        for p in propose(*region, ctx=ctx, **kw).proposals:
            out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
            routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
            got = widen(out.download(np.uint16, (b.tokens, b.out_stride))).reshape(want.shape)
            assert (np.abs(got - want) <= bound).all(), p.symbols
            assert (got[:5] == 5.25).all() and (got[b.starts[-1]:] == 5.25).all(), p.symbols
        b.free()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("of", ["keys", "values"])
def test_nan_reaches_the_rows_that_see_it(ctx, dim, of):
    """In every form, the keys in parts: a row of nothing else but one, rows of many
    others; the rows before it keep out of it where a key is meant."""
    b = Batch([(1900, 40), (0, 3)], 4, 2, dim, page=16, seed=dim, width=130)
    want, bound = b.want()
    for s, j in ((0, 1920), (1, 0)):
        up = b.k_up if of == "keys" else b.v_up
        up[b.table[s, j // 16], j % 16] = 0x7FC0
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    for p in propose(*region, ctx=ctx, **kw).proposals:
        assert len(p.symbols) == 2  # joined
        routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
        got = widen(out.download(np.uint16, (b.tokens, b.out_stride))).reshape(want.shape)
        sees = np.r_[20:40, 40:43]
        assert np.isnan(got[sees]).all(), p.symbols
        if of == "keys":
            assert (np.abs(got[:20] - want[:20]) <= bound[:20]).all(), p.symbols
    b.free()


@pytest.mark.parametrize("dim,heads,kv_heads,lengths,window,sinks", [
    (64, 64, 8, [(900, 275), (3000, 257), (0, 275), (400, 265)], 1030, 3), (256, 64, 8, [(2200, 273), (90, 273)], 1100, 0),
    (64, 70, 7, [(900, 275), (3000, 257), (0, 275), (400, 265)], 1030, 0), (96, 192, 8, [(2000, 350)], 800, 30), (128, 192, 8, [(10, 175), (3000, 172), (9, 3)], 1100, 0)])
def test_a_last_round_in_parts(ctx, dim, heads, kv_heads, lengths, window, sinks):
    """Equal tiles a few more than fill the CUs: whole ones, then parts of the others;
    sequences that end inside tiles of either kind."""
    b = Batch(lengths, heads, kv_heads, dim, page=32, window=window, sinks=sinks, pad=5, gap=2, seed=dim)
    want, bound = b.want()
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    joins = []
    for p in propose(*region, ctx=ctx, **kw).proposals[1:]:
        joins += p.symbols[1:]
        out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
        for _ in range(2):
            routed(ctx, p.realize(ctx), [q, k, v, table, starts, lens], [out])
            got = widen(out.download(np.uint16, (b.tokens, b.out_stride)))
            off = np.abs(got[:, :heads * dim].reshape(want.shape) - want)
            assert (off <= bound).all(), f"{p.symbols}: worst {np.nanmax(off / np.maximum(bound, 1e-30))} of the bound"
            assert (got[:, heads * dim:] == 5.25).all(), p.symbols
    assert any("_join_t" in j for j in joins)
    b.check(ctx)
    b.free()


def test_rows_for_tiles_of_256(ctx):
    """Work enough that they are chosen, whole and in parts of the keys."""
    for lengths, heads, kv_heads, window in (([(0, 4096), (0, 4096)], 16, 1, 64), ([(3000, 300)], 32, 8, 0)):
        b = Batch(lengths, heads, kv_heads, 96 if window else 128, page=64, window=window, sinks=2 if window else 0, seed=1)
        region, kw = region_of(b)
        assert "_t256_" in realize(*region, ctx=ctx, **kw).symbols[0]
        b.check(ctx, max_length=0)


def test_one_token_to_a_page_and_axes_of_one(ctx):
    """What an axis of one says of its stride does not matter."""
    for lengths, page in (([(70, 3), (0, 40)], 1), ([(70, 1), (9, 1)], 1)):
        b = Batch(lengths, 3, 1, 64, page=page, seed=1)
        want = b.run(ctx)
        q, k, v, table, starts, lens, out = b.upload(ctx)
        for strides in ((64, 0, 0), (64, 5, 1 << 40), (64, 1 << 50, 7)):
            out.upload(np.full((b.tokens, b.out_stride), 0x40A8, np.uint16))
            cache = L.PagedCache(k=k.ptr, v=v.ptr, pages=b.pages, page=page, heads=1, head_dim=64, page_stride=strides[0],
                                 token_stride=strides[1], head_stride=strides[2])
            ctx.paged_attention_bf16(b.shape(), q, cache, table, starts, lens, out)
            ctx.synchronize()
            np.testing.assert_array_equal(out.download(np.uint16, want.shape), want)
        b.check(ctx)
        b.free()


def test_lists_out_of_range_in_every_form(ctx):
    """starts and lengths that break their contract: nothing faults, nothing beside
    the rows is written."""
    for dim, heads, kv_heads, lengths, fresh in ((64, 4, 2, [(40, 3), (10, 50), (3, 20)], 50), (128, 64, 4, [(40, 30), (100, 50), (3, 20)], 50),
                                                 (64, 4, 2, [(2000, 1), (10, 1), (3, 1)], 1)):
        b = Batch(lengths, heads, kv_heads, dim, pad=4, gap=2, seed=14)
        n = int(b.starts[-1])
        for starts, lens in (([0, -5, n, n], [43, 60, 4]), ([0, 3, 2 ** 31 - 1, 9], [43, 2 ** 31 - 1, 4]),
                             ([n, 6, 3, 0], [43, 60, 4]), ([-2 ** 31, 3, n + 4, n], [-2 ** 31, -1, 2 ** 31 - 1]),
                             ([0, n, n, 2 ** 31 - 1], [5, 0, 1])):
            b.starts, b.lengths = np.array(starts, np.int32), np.array(lens, np.int32)
            got = widen(b.run(ctx, max_length=60 if fresh > 1 else 2001, max_fresh=fresh))
            assert np.isfinite(got).all() and (got[:, heads * dim:] == 5.25).all()


# -- the store ----------------------------------------------------------------------
def test_two_tokens_of_one_slot(ctx):
    """Either token's row, whole or in 16-byte pieces, and every other row as it was."""
    heads, dim, page, pages, tokens = 2, 64, 4, 3, 6
    row_up, row = bf16(np.random.default_rng(0).standard_normal((tokens, 2 * heads * dim)))
    before = np.full((pages, page, heads, dim), 0x4000, np.uint16)
    d_row, k, v = ctx.to_device(row_up), ctx.to_device(before), ctx.to_device(before)
    slots = ctx.to_device(np.array([5, 5, 0, -1, 12, 5], np.int32))
    cache = L.PagedCache(k=k.ptr, v=v.ptr, pages=pages, page=page, heads=heads, head_dim=dim, page_stride=page * heads * dim,
                         token_stride=heads * dim, head_stride=dim)
    layout = L.HeadLayout(tokens=tokens, kv_heads=heads, head_dim=dim, k_stride=2 * heads * dim, v_stride=2 * heads * dim)
    ctx.norm_rotate(L.BF16, layout, None, d_row, d_row.ptr + 2 * heads * dim, None, None, None, None, None, None, cache, slots)
    ctx.synchronize()
    for buf, at in ((k, 0), (v, heads * dim)):
        got = buf.download(np.uint16, before.shape)
        mine = row_up[:, at:at + heads * dim].reshape(tokens, heads, dim)
        assert (got[0, 0] == mine[2]).all()
        pieces = got[1, 1].reshape(-1, 8)
        assert all(any((p == mine[t].reshape(-1, 8)[i]).all() for t in (0, 1, 5)) for i, p in enumerate(pieces))
        rest = np.ones((pages, page), bool)
        rest[0, 0] = rest[1, 1] = False
        assert (got[rest] == 0x4000).all()
    for b in (d_row, k, v, slots):
        b.free()


# -- programs of the recognizer -------------------------------------------------------
def routed(ctx, rz, inputs, outputs):
    ins, outs = iter(inputs), iter(outputs)
    route(ctx, rz, [next(ins) if role == L.SLOT_INPUT else next(outs) if role == L.SLOT_OUTPUT else None for role, _ in rz.slots])
    ctx.synchronize()


def realizations(ctx, program, extents, **kw):
    yield realize(program, extents, permissions=RE, ctx=ctx, **kw)
    for p in propose(program, extents, permissions=RE, ctx=ctx, **kw).proposals:
        yield p.realize(ctx)


@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
@pytest.mark.parametrize("dim,rotary,pairing", [(128, 128, 0), (90, 34, 1), (64, 32, 1)])
def test_routed_rotation(ctx, dim, rotary, pairing, dtype):
    tokens, heads, kv_heads = 300, 5, 2
    rng, store = np.random.default_rng(dim), np.uint16 if dtype == L.BF16 else np.float32
    host = lambda *s: bf16(rng.standard_normal(s))[0] if dtype == L.BF16 else rng.standard_normal(s).astype(np.float32)
    q, k, dy_q, dy_k, w = (host(tokens, heads, dim), host(tokens, kv_heads, dim), host(tokens, heads, dim),
                           host(tokens, kv_heads, dim), host(2, dim))
    positions = rng.integers(0, 9999, tokens).astype(np.int32)
    frequencies = 10000.0 ** (-np.arange(0, rotary, 2, dtype=np.float64) / rotary)
    pairs = ("halves", "neighbours")[pairing]
    want = families.norm_rotate(q, k, *w, positions, frequencies, rotary, pairs, EPS_BITS, ctx=ctx)
    grads = families.norm_rotate_backward(dy_q, dy_k, q, k, *w, positions, frequencies, rotary, pairs, EPS_BITS, ctx=ctx)
    put = [ctx.to_device(a) for a in (q, k, w[0], w[1], positions, frequencies, dy_q, dy_k)]
    outs = [ctx.alloc(a.nbytes) for a in grads]
    kw = dict(dtype=dtype, strides=(heads * dim, kv_heads * dim) * 2, grouping=(pairing,), scalars=(EPS_BITS,))
    extents = (tokens, heads, kv_heads, dim, rotary)
    for flags in (0, L.REGION_ALIGNED16):
        for rz in realizations(ctx, L.PROGRAM_NORM_ROTATE, extents, flags=flags,
                               variant=L.ROTATE_WQ | L.ROTATE_WK | L.ROTATE_K_OUT, **kw):
            routed(ctx, rz, put[:6], outs[:2])
            for b, a in zip(outs, want):
                np.testing.assert_array_equal(b.download(store, a.shape), a)
        for rz in realizations(ctx, L.PROGRAM_NORM_ROTATE_BACKWARD, extents, flags=flags,
                               variant=L.ROTATE_WQ | L.ROTATE_WK | L.ROTATE_DQ | L.ROTATE_DK | L.ROTATE_DWQ | L.ROTATE_DWK, **kw):
            routed(ctx, rz, [*put[6:], *put[:6]], outs)
            for b, a in zip(outs, grads):
                np.testing.assert_array_equal(b.download(store, a.shape), a)
    for b in (*put, *outs):
        b.free()


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,window,sinks", [
    ([(3000, 1), (20, 1)], 8, 2, 64, 0, 0), ([(30, 70), (200, 9)], 6, 2, 128, 40, 3), ([(100, 200)], 4, 1, 256, 0, 0)])
def test_routed_attention(ctx, lengths, heads, kv_heads, dim, window, sinks):
    b = Batch(lengths, heads, kv_heads, dim, window=window, sinks=sinks, seed=dim)
    want = b.run(ctx, max_length=0)
    q, k, v, table, starts, lens, out = b.upload(ctx)
    region, kw = region_of(b)
    offer = propose(*region, ctx=ctx, **kw)
    for rz in (realize(*region, ctx=ctx, **kw), offer.proposals[offer.chosen].realize(ctx)):
        out.upload(np.zeros((b.tokens, b.out_stride), np.uint16))
        routed(ctx, rz, [q, k, v, table, starts, lens], [out])
        np.testing.assert_array_equal(out.download(np.uint16, want.shape), want)
    b.free()


# -- host functions -------------------------------------------------------------------
def test_host_functions(ctx):
    rng = np.random.default_rng(0)
    kept, fresh, table = [5, 0, 30], [3, 9, 1], np.array([[7, 1, -1, -1, -1, -1, -1, -1]] * 3, np.int32)
    table[2, :8] = np.arange(20, 28)
    free = rng.permutation(20).astype(np.int32)
    got = families.page_slots(kept, fresh, 4, free, table, 15, ctx=ctx)
    for g, w in zip(got, ref.page_slots(kept, fresh, 4, free, table, 15)):
        np.testing.assert_array_equal(g.reshape(-1), np.reshape(w, -1))
    assert families.page_slots([], [], 4, [], np.zeros((0, 3)), ctx=ctx)[1].tolist() == [0]
    b = Batch([(50, 3), (0, 20)], 4, 2, 64, pad=2, seed=1)
    want, bound = b.want()
    n = int(b.starts[-1])
    out = families.paged_attention_bf16(b.q_up.reshape(-1, 4, 64), b.k_up, b.v_up, b.table, b.starts, b.lengths, b.scale, ctx=ctx)
    assert (np.abs(widen(out)[:n] - want[:n]) <= bound[:n]).all() and not out[n:].any()
    none = families.norm_rotate(np.zeros((0, 2, 64), np.uint16), np.zeros((0, 1, 64), np.uint16), None, None,
                                np.zeros(0, np.int32), np.ones(32), 64, ctx=ctx)
    assert none[0].shape == (0, 2, 64)
    q, k = bf16(rng.standard_normal((4, 2, 64)))[0], bf16(rng.standard_normal((4, 1, 64)))[0]
    grads = families.norm_rotate_backward(q, k, q, k, None, None, np.zeros(4, np.int32), np.ones(32), 64, eps_bits=0, ctx=ctx)
    assert (grads[0] == q).all() and (grads[1] == k).all() and grads[2] is None  # position 0, no norm


# -- refusals of the calls themselves ---------------------------------------------------
def status_of(call):
    with pytest.raises(Refusal) as e:
        call()
    return e.value.status


def test_refused_calls(ctx):
    bufs = [ctx.alloc(1 << 16) for _ in range(8)]
    p = [b.ptr for b in bufs]
    bad, cap, unsup, mis = L.REFUSE_INVALID_ARGUMENT, L.REFUSE_CAPACITY, L.REFUSE_UNSUPPORTED, L.REFUSE_BINDING_MISMATCH

    def slots(kept=p[0], fresh=p[0], n=2, page=4, free=p[1], count=4, table=p[2], width=3, tokens=5, starts=p[3], lengths=p[4],
              positions=p[5], slot=p[6], taken=p[7]):
        ctx.page_slots(kept, fresh, n, page, free, count, table, width, tokens, starts, lengths, positions, slot, taken)

    for kw in ("kept", "fresh", "free", "table", "starts", "lengths", "positions", "slot", "taken"):
        assert status_of(lambda: slots(**{kw: None})) == bad, kw
    assert status_of(lambda: slots(page=0)) == bad
    for kw in (dict(page=1 << 31), dict(n=1 << 31), dict(tokens=1 << 31), dict(count=1 << 31), dict(width=1 << 31)):
        assert status_of(lambda: slots(**kw)) == cap, kw
    cache = L.PagedCache(k=p[0], v=p[1], pages=3, page=4, heads=2, head_dim=8, page_stride=64, token_stride=16, head_stride=8)
    layout = dict(tokens=2, q_heads=4, kv_heads=2, head_dim=8, rotary=8, eps_bits=EPS_BITS, q_stride=32, k_stride=16, v_stride=16,
                  q_out_stride=32, k_out_stride=16)

    def rotate(dtype=L.BF16, q=p[0], k=p[1], v=None, wq=None, wk=None, at=p[2], f=p[3], q_out=p[4], k_out=p[5], cache=None,
               slots=None, **kw):
        ctx.norm_rotate(dtype, L.HeadLayout(**{**layout, **kw}), q, k, v, wq, wk, at, f, q_out, k_out, cache, slots)

    for kw in ("q", "k", "at", "f", "q_out"):
        assert status_of(lambda: rotate(**{kw: None})) == bad, kw
    for kw in (dict(k_out=None), dict(v=p[6]), dict(slots=p[6]), dict(cache=cache), dict(v=p[6], cache=cache),
               dict(v=p[6], slots=p[7]), dict(cache=cache, slots=p[7]), dict(wq=p[6], eps_bits=0), dict(rotary=10), dict(rotary=3),
               dict(v=p[6], slots=p[7], cache=cache, head_dim=4, rotary=4), dict(v=p[6], slots=p[7], cache=cache, kv_heads=1),
               dict(v=p[6], slots=p[7], cache=cache, v_stride=15)):
        assert status_of(lambda: rotate(**kw)) == bad, kw
    assert status_of(lambda: rotate(dtype=L.F32, v=p[6], slots=p[7], cache=cache)) == unsup

    def back(dq_out=p[0], dk_out=p[1], q=p[2], k=p[3], wq=None, wk=None, at=p[4], f=p[5], dq=p[6], dk=p[7], dwq=None, dwk=None,
             ws=None, n=0, dtype=L.BF16, **kw):
        ctx.norm_rotate_backward(dtype, L.HeadLayout(**{**layout, **kw}), dq_out, dk_out, q, k, wq, wk, at, f, dq, dk, dwq, dwk,
                                 workspace=ws, workspace_bytes=n)

    for kw in ("dq_out", "dk_out", "q", "k", "at", "f"):
        assert status_of(lambda: back(**{kw: None})) == bad, kw
    assert status_of(lambda: back(dwq=p[6], dq=None, eps_bits=0)) == bad
    assert status_of(lambda: back(dtype=7)) == unsup
    shape = dict(tokens=2, sequences=2, q_heads=4, scale=1.0, q_stride=32, out_stride=32, table_width=300)

    def attend(q=p[2], c=cache, table=p[3], starts=p[4], lengths=p[5], out=p[6], ws=None, n=0, **kw):
        ctx.paged_attention_bf16(L.AttentionShape(**{**shape, **kw}), q, c, table, starts, lengths, out, workspace=ws,
                                 workspace_bytes=n)

    for kw in ("q", "table", "starts", "lengths", "out"):
        assert status_of(lambda: attend(**{kw: None})) == bad, kw
    for at in (dict(k=None), dict(v=None)):
        c = L.PagedCache.from_buffer_copy(cache)
        for name, value in at.items():
            setattr(c, name, value)
        assert status_of(lambda: attend(c=c)) == bad
    c = L.PagedCache.from_buffer_copy(cache)
    c.k = p[0] + 8
    assert status_of(lambda: attend(c=c)) == unsup  # off 16 bytes
    n = ctx.paged_attention_bf16_workspace(L.AttentionShape(**shape), cache)
    assert n > 0
    assert status_of(lambda: attend(ws=p[7], n=n - 1)) == cap
    assert status_of(lambda: attend(ws=p[7] + 4, n=n)) == bad
    nothing = dict(tokens=0, sequences=0, q=None, table=None, starts=None, lengths=None, out=None)
    attend(**nothing)
    rotate(tokens=0, q=None, k=None, q_out=None, at=None, f=None)
    ctx.synchronize()
    lib = L.lib()
    assert lib.tiler_hip_paged_attention_bf16(None, None, *[None] * 6, None, 0, None) == bad
    assert lib.tiler_hip_norm_rotate(ctx.handle, L.BF16, None, *[None] * 9, None, None, None) == bad
    for b in bufs:
        b.free()
