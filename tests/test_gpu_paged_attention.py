"""Attention over the paged cache against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from attention_reference import paged_attention
from tiler_amd import _lib as L

pytestmark = pytest.mark.gpu


def bf16(a):
    a = np.ascontiguousarray(a, np.float32)
    b = oracle.bf16_narrow(a.reshape(-1)).reshape(a.shape)
    return b, oracle.bf16_widen(b.reshape(-1)).reshape(a.shape).astype(np.float64)


def widen(b):
    return oracle.bf16_widen(b.reshape(-1)).reshape(b.shape).astype(np.float64)


class Batch:
    """Sequences of (kept, fresh) tokens, their pages at random places of a pool."""

    def __init__(self, lengths, heads, kv_heads, dim, page=16, layout="tokens", window=0, sinks=0, pad=0, seed=0, spread=1.0,
                 gap=0, width=None, scale=None):
        rng = self.rng = np.random.default_rng(seed)
        self.kept, self.fresh = [a for a, _ in lengths], [b for _, b in lengths]
        self.heads, self.kv_heads, self.dim, self.page, self.layout = heads, kv_heads, dim, page, layout
        self.window, self.sinks, self.scale = window, sinks, dim ** -0.5 if scale is None else scale
        need = [-(-(a + b) // page) for a, b in lengths]
        self.pages = sum(need) + 2
        self.width = max(need + [1]) + 1 if width is None else width
        order = rng.permutation(self.pages)
        self.table = np.full((len(lengths), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :min(n, self.width)] = order[at:at + min(n, self.width)]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.fresh)]).astype(np.int32)
        self.lengths = np.array([a + b for a, b in lengths], np.int32)
        self.tokens = int(self.starts[-1]) + pad
        self.q_stride, self.out_stride = heads * dim + gap, heads * dim + 3 * gap
        self.q_up, self.q = bf16(spread * rng.standard_normal((self.tokens, self.q_stride)))
        shape = (self.pages, page, kv_heads, dim)
        self.k_up, self.k = bf16(rng.standard_normal(shape))
        self.v_up, self.v = bf16(rng.standard_normal(shape))

    def cache(self, k, v):
        h, d, p = self.kv_heads, self.dim, self.page
        token, head = (h * d, d) if self.layout == "tokens" else (d, p * d)
        return L.PagedCache(k=k, v=v, pages=self.pages, page=p, heads=h, head_dim=d, page_stride=p * h * d,
                            token_stride=token, head_stride=head)

    def shape(self, **kw):
        a = dict(tokens=self.tokens, sequences=len(self.lengths), q_heads=self.heads, scale=self.scale, q_stride=self.q_stride,
                 out_stride=self.out_stride, table_width=self.width, window=self.window, sinks=self.sinks,
                 max_fresh=max(self.fresh), max_length=int(self.lengths.max()))
        a.update(kw)
        return L.AttentionShape(**a)

    def stored(self, x):
        return np.ascontiguousarray(x if self.layout == "tokens" else x.transpose(0, 2, 1, 3))

    def upload(self, ctx):
        marker = bf16(np.full((self.tokens, self.out_stride), 5.25))[0]
        self.bufs = [ctx.to_device(a) for a in (self.q_up, self.stored(self.k_up), self.stored(self.v_up), self.table,
                                                self.starts, self.lengths, marker)]
        return self.bufs

    def free(self):
        for b in self.bufs:
            b.free()

    def run(self, ctx, workspace=True, **kw):
        q, k, v, table, starts, lengths, out = self.upload(ctx)
        shape, cache = self.shape(**kw), self.cache(k.ptr, v.ptr)
        need = ctx.paged_attention_bf16_workspace(shape, cache)
        space = ctx.alloc(max(need, 1))
        ctx.paged_attention_bf16(shape, q, cache, table, starts, lengths, out, workspace=space if workspace else None,
                                 workspace_bytes=need)
        ctx.synchronize()
        got = out.download(np.uint16, (self.tokens, self.out_stride))
        space.free()
        self.free()
        return got

    def want(self):
        n = self.heads * self.dim
        return paged_attention(self.q[:, :n].reshape(self.tokens, self.heads, self.dim), self.k, self.v, self.table, self.starts,
                               self.lengths, np.float32(self.scale).astype(np.float64), self.window, self.sinks,
                               np.full((self.tokens, self.heads, self.dim), 5.25))

    def check(self, ctx, **kw):
        got = widen(self.run(ctx, **kw))
        n = self.heads * self.dim
        want, bound = self.want()
        off = np.abs(got[:, :n].reshape(want.shape) - want)
        over = ~(off <= bound)
        assert not over.any(), (f"{over.sum()} of {over.size}, rows {np.unique(np.nonzero(over)[0])[:20]}, worst "
                                f"{np.nanmax(off / np.maximum(bound, 1e-30))} of the bound")
        assert (got[:, n:] == 5.25).all()  # between the rows


DIMS = [8, 16, 40, 64, 72, 80, 96, 128, 136, 160, 192, 256]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_decode(ctx, dim, layout):
    Batch([(0, 1), (1, 1), (30, 1), (31, 1), (32, 1), (200, 1)], 4, 2, dim, layout=layout, seed=dim).check(ctx)


@pytest.mark.parametrize("dim", DIMS)
def test_prompts(ctx, dim):
    Batch([(0, 70), (0, 1), (0, 33)], 4, 2, dim, page=8, seed=dim).check(ctx)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (3, 1), (5, 5), (14, 2), (16, 1), (17, 1), (40, 1), (130, 1), (12, 4)])
def test_groups(ctx, heads, kv_heads):
    Batch([(20, 1), (50, 3), (0, 9)], heads, kv_heads, 64, seed=heads).check(ctx)
    Batch([(5, 20)], heads, kv_heads, 128, seed=heads).check(ctx)


@pytest.mark.parametrize("page", [1, 2, 3, 7, 16, 24, 31, 32, 33, 64, 100, 128, 1000])
def test_pages(ctx, page):
    Batch([(90, 1), (3, 40), (64, 2)], 4, 2, 64, page=page, seed=page).check(ctx)


@pytest.mark.parametrize("kept", [0, 1, 63, 64, 65, 127, 128, 500])
@pytest.mark.parametrize("fresh", [1, 2, 15, 16, 17, 63, 64, 65, 130])
def test_lengths(ctx, kept, fresh):
    Batch([(kept, fresh)], 2, 1, 64, seed=kept + fresh).check(ctx)


@pytest.mark.parametrize("window", [1, 2, 5, 31, 32, 33, 64, 100, 1000])
@pytest.mark.parametrize("sinks", [0, 1, 4, 31, 32, 40, 70])
def test_window_and_sinks(ctx, window, sinks):
    Batch([(300, 1), (0, 3), (150, 70), (64, 1), (33, 2)], 4, 2, 64, window=window, sinks=sinks, seed=window).check(ctx)


def test_window_of_large_heads(ctx):
    for dim in (128, 256):
        Batch([(300, 1), (150, 40)], 4, 2, dim, window=50, sinks=3, seed=dim).check(ctx)


def test_long_context_is_split(ctx):
    """A context that several workgroups share, and one row that leaves most of them
    without keys."""
    for dim in (64, 128, 256):
        Batch([(5000, 1), (3, 1), (0, 1), (2047, 1)], 4, 2, dim, seed=dim).check(ctx)
    Batch([(4000, 5)], 8, 1, 64, page=64, seed=1).check(ctx)
    Batch([(4000, 40), (10, 1)], 2, 1, 128, page=64, seed=2).check(ctx)
    Batch([(4000, 2), (3000, 1)], 4, 1, 128, page=64, window=1500, sinks=600, seed=3).check(ctx)


def test_batch_with_empty_sequences_and_padding(ctx):
    Batch([(10, 0), (0, 5), (7, 0), (0, 0), (33, 1), (5, 0)], 6, 2, 64, pad=9, seed=4).check(ctx)
    Batch([(3000, 0), (2500, 1)], 6, 2, 64, pad=3, seed=5).check(ctx)


def test_strides_and_alignment(ctx):
    for gap in (1, 3, 8):
        Batch([(20, 9), (100, 1)], 5, 1, 72, gap=gap, seed=gap).check(ctx)
        Batch([(3000, 1)], 5, 1, 72, gap=gap, seed=gap).check(ctx)


def test_hints_do_not_matter(ctx):
    """max_fresh and max_length choose how the work is cut, not what comes out of it
    but for the rounding."""
    lengths = [(900, 1), (10, 60), (0, 3)]
    for hints in (dict(max_fresh=0, max_length=0), dict(max_fresh=1, max_length=1), dict(max_fresh=1000, max_length=10 ** 6)):
        Batch(lengths, 8, 2, 128, seed=6).check(ctx, **hints)
        Batch(lengths, 8, 2, 128, seed=6, window=40, sinks=2).check(ctx, **hints)


def test_peaked_and_flat_softmax(ctx):
    Batch([(300, 1), (0, 80)], 4, 2, 64, spread=20.0, seed=7).check(ctx)
    Batch([(300, 1), (0, 80)], 4, 2, 64, spread=0.0, seed=8).check(ctx)
    b = Batch([(300, 3), (0, 80)], 4, 2, 64, spread=1.0, seed=9, scale=1.0)
    b.q_up[0], b.q[0] = bf16(np.full(b.q_stride, 100.0))  # logits in the hundreds
    b.check(ctx)


def test_growing_maximum(ctx):
    """Logits that rise with the key: every step moves the running maximum."""
    b = Batch([(700, 2)], 2, 1, 64, page=16, scale=1.0, seed=10)
    slope = np.zeros((b.pages, 16, 1, 64))
    for j in range(702):
        slope[b.table[0, j // 16], j % 16, 0, 0] = j
    b.k_up, b.k = bf16(slope)
    q = np.zeros((b.tokens, b.q_stride))
    q[:, 0], q[:, 64] = 0.5, -0.5
    b.q_up, b.q = bf16(q)
    b.check(ctx)


def test_pages_that_are_not_there(ctx):
    """Entries that name no page read as zeros; keys past the table are not seen."""
    b = Batch([(200, 2), (100, 1)], 4, 2, 64, seed=11)
    b.table[0, 3], b.table[0, 5], b.table[1, 0] = -1, b.pages, 2 ** 31 - 1
    b.check(ctx)
    Batch([(200, 2), (100, 1), (0, 20)], 4, 2, 64, width=4, seed=12).check(ctx)
    Batch([(200, 2)], 4, 2, 64, width=0, seed=12).check(ctx)


def test_rows_that_see_nothing(ctx):
    """Fewer tokens in all than new ones: the first rows stand before the sequence."""
    b = Batch([(0, 20), (40, 3)], 4, 2, 64, seed=13)
    b.lengths[:] = [5, 0]
    b.check(ctx)
    assert not b.want()[0][:15].any()


def test_lists_out_of_range_touch_nothing_else(ctx):
    """starts and lengths that break their contract: nothing but rows of out is
    written, and what lies beside it stays."""
    b = Batch([(40, 3), (10, 5), (3, 1)], 4, 2, 64, pad=4, seed=14)
    for starts, lengths in (([0, -5, 9, 9], [43, 15, 4]), ([0, 3, 2 ** 31 - 1, 9], [43, 2 ** 31 - 1, 4]),
                            ([9, 6, 3, 0], [43, 15, 4]), ([-2 ** 31, 3, 8, 9], [-2 ** 31, -1, 4])):
        b.starts, b.lengths = np.array(starts, np.int32), np.array(lengths, np.int32)
        got = widen(b.run(ctx, max_length=60, max_fresh=5))
        assert np.isfinite(got).all()


def test_what_no_row_sees_does_not_matter(ctx):
    """NaN and infinities behind the sequence, before the window and in other pages."""
    for window, sinks in ((0, 0), (20, 3)):
        b = Batch([(61, 1), (200, 1), (0, 1)], 4, 2, 64, window=window, sinks=sinks, seed=15)
        seen = np.zeros((b.pages, b.page), bool)
        for s, n in enumerate(b.lengths):
            j = np.arange(n)
            if window:
                j = j[(j > n - 1 - window) | (j < sinks)]
            seen[b.table[s, j // b.page], j % b.page] = True
        want = b.want()
        for up, fill in ((b.k_up, 0x7FC0), (b.v_up, 0x7F80)):
            up[~seen] = fill
        b.want = lambda: want
        b.check(ctx)


def test_hidden_keys_of_a_chunk(ctx):
    """Keys that a row does not see but others of its chunk do: NaN and infinities
    there stay out of the row's weights."""
    b = Batch([(0, 40)], 2, 1, 64, seed=16)
    want = b.want()
    k = b.k_up[b.table[0, 39 // 16], 39 % 16]
    k[:] = 0x7FC0
    got = widen(b.run(ctx))[:, :128].reshape(40, 2, 64)
    assert np.isnan(got[39]).all()
    assert (np.abs(got - want[0]) <= want[1])[:39].all()


def test_infinite_logits(ctx):
    """A key whose logit is -infinity has no weight; a row of nothing else is zeros."""
    b = Batch([(40, 1), (3, 1)], 1, 1, 64, seed=17)
    b.q_up, b.q = bf16(np.abs(b.q) + 0.5)
    b.k_up[b.table[0, 1]] = 0xFF80
    b.k[b.table[0, 1]] = -np.inf
    b.k_up[b.table[1, 0]] = 0xFF80
    b.k[b.table[1, 0]] = -np.inf
    got = widen(b.run(ctx))
    with np.errstate(all="ignore"):
        w = b.want()[0]
    assert not got[1].any() and np.isfinite(got[0]).all()
    assert np.abs(got[0].reshape(1, 64) - w[0]).max() < 0.05


def test_far_offsets(ctx):
    """A cache whose rows lie beyond 2^32 elements."""
    pages, page, dim = 3, 16, 64
    stride = (1 << 31) + 64  # elements from page to page: 4 GiB and more
    b = Batch([(20, 2)], 2, 1, dim, page=page, seed=18)
    assert b.pages >= pages
    b.table[0, :2] = [2, 1]
    b.pages = pages
    q, k, v, table, starts, lengths, out = b.upload(ctx)
    wide = [ctx.alloc((2 * stride + page * dim) * 2) for _ in range(2)]
    for n in range(pages):
        for src, dst in ((k, wide[0]), (v, wide[1])):
            ctx.copy(dst.ptr + n * stride * 2, src.ptr + n * page * dim * 2, page * dim * 2)
    cache = L.PagedCache(k=wide[0].ptr, v=wide[1].ptr, pages=pages, page=page, heads=1, head_dim=dim, page_stride=stride,
                         token_stride=dim, head_stride=dim)
    ctx.paged_attention_bf16(b.shape(), q, cache, table, starts, lengths, out)
    ctx.synchronize()
    got = widen(out.download(np.uint16, (b.tokens, b.out_stride)))
    b.k, b.v = b.k[:pages], b.v[:pages]
    want, bound = b.want()
    assert (np.abs(got.reshape(want.shape) - want) <= bound).all()
    for w in wide:
        w.free()
    b.free()


def test_runs_are_equal(ctx):
    for lengths in ([(3000, 1), (100, 1)], [(200, 150)]):
        b = Batch(lengths, 8, 2, 128, seed=19)
        first = b.run(ctx)
        for workspace in (True, False):
            np.testing.assert_array_equal(b.run(ctx, workspace=workspace), first)
