"""Head norms with the rotation, their store into the paged cache and their
gradients, against the definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from attention_reference import U16, U32, norm_rotate, norm_rotate_backward
from tiler_amd import _lib as L

pytestmark = pytest.mark.gpu

EPS_BITS = 0x358637BD
EPS = float(np.uint32(EPS_BITS).view(np.float32))
PAIRINGS = {"halves": L.ROTATE_HALVES, "neighbours": L.ROTATE_NEIGHBOURS}


def stored(a, dtype):
    """(what is uploaded, the values it stands for)."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == L.F32:
        return a, a.astype(np.float64)
    b = oracle.bf16_narrow(a.reshape(-1)).reshape(a.shape)
    return b, oracle.bf16_widen(b.reshape(-1)).reshape(a.shape).astype(np.float64)


def values(a, dtype):
    return a.astype(np.float64) if dtype == L.F32 else oracle.bf16_widen(a.reshape(-1)).reshape(a.shape).astype(np.float64)


def close(got, want, bound, dtype, what):
    unit = U16 if dtype == L.BF16 else U32
    # the bound, and the one rounding of the result to its type (subnormal steps besides)
    limit = bound + unit * (np.abs(want) + bound) + 2.0 ** -133
    over = ~(np.abs(got - want) <= limit)
    assert not over.any(), f"{what}: {over.sum()} of {over.size}, worst {np.nanmax(np.abs(got - want) / limit)} of the bound"


class Case:
    """Slices of one projection with odd gaps between them."""

    def __init__(self, tokens, heads, kv_heads, dim, rotary, pairing, norm, dtype, seed=0, far=50000, gap=0, weights=True):
        rng = np.random.default_rng(seed)
        self.rng, self.tokens, self.heads, self.kv_heads, self.dim = rng, tokens, heads, kv_heads, dim
        self.rotary, self.pairing, self.norm, self.dtype = rotary, pairing, norm, dtype
        self.elem = 2 if dtype == L.BF16 else 4
        self.stride = (heads + 2 * kv_heads) * dim + gap
        row = rng.standard_normal((tokens, self.stride)) * np.exp(rng.standard_normal((tokens, 1)))
        self.row_up, self.row = stored(row, dtype)
        self.positions = rng.integers(0, far, tokens).astype(np.int32)
        self.frequencies = 10000.0 ** (-np.arange(0, rotary, 2, dtype=np.float64) / max(rotary, 1))
        self.weights = weights and norm
        self.w_up, self.w = stored(1 + 0.1 * rng.standard_normal((2, dim)), dtype)

    def layout(self, **kw):
        a = dict(tokens=self.tokens, q_heads=self.heads, kv_heads=self.kv_heads, head_dim=self.dim, rotary=self.rotary,
                 pairing=PAIRINGS[self.pairing], eps_bits=EPS_BITS if self.norm else 0, q_stride=self.stride,
                 k_stride=self.stride, v_stride=self.stride, q_out_stride=self.heads * self.dim,
                 k_out_stride=self.kv_heads * self.dim)
        a.update(kw)
        return L.HeadLayout(**a)

    def part(self, which):
        at = {"q": 0, "k": self.heads * self.dim, "v": (self.heads + self.kv_heads) * self.dim}[which]
        n = self.heads if which == "q" else self.kv_heads
        return self.row[:, at:at + n * self.dim].reshape(self.tokens, n, self.dim), at * self.elem

    def want(self, which):
        return norm_rotate(self.part(which)[0], self.w["qk".index(which)] if self.weights else None, self.positions,
                           self.frequencies, self.rotary, self.pairing, EPS if self.norm else None)

    def upload(self, ctx):
        self.d_row, self.d_w = ctx.to_device(self.row_up), ctx.to_device(self.w_up)
        self.d_pos, self.d_freq = ctx.to_device(self.positions), ctx.to_device(self.frequencies if self.rotary else np.zeros(1))
        self.bufs = [self.d_row, self.d_w, self.d_pos, self.d_freq]
        wq = self.d_w.ptr if self.weights else None
        wk = self.d_w.ptr + self.dim * self.elem if self.weights else None
        return wq, wk

    def free(self):
        for b in self.bufs:
            b.free()


def forward(ctx, c, check=True, stream=None):
    wq, wk = c.upload(ctx)
    store = np.uint16 if c.dtype == L.BF16 else np.float32
    shape_q, shape_k = (c.tokens, c.heads, c.dim), (c.tokens, c.kv_heads, c.dim)
    dq, dk = ctx.alloc(max(int(np.prod(shape_q)) * c.elem, 1)), ctx.alloc(max(int(np.prod(shape_k)) * c.elem, 1))
    c.bufs += [dq, dk]
    ctx.norm_rotate(c.dtype, c.layout(), c.d_row.ptr, c.d_row.ptr + c.part("k")[1], None, wq, wk, c.d_pos, c.d_freq, dq,
                    dk if c.kv_heads else None, stream=stream)
    ctx.synchronize()
    got = dq.download(store, shape_q), dk.download(store, shape_k)
    if check:
        for which, g in zip("qk", got):
            want, bound = c.want(which)
            close(values(g, c.dtype), want, bound, c.dtype, which)
    c.free()
    return got


FORMS = [  # heads, kv_heads, dim, rotary
    (32, 8, 128, 128), (4, 2, 64, 64), (2, 1, 256, 256), (5, 1, 80, 80), (3, 3, 96, 32), (7, 1, 90, 34), (1, 1, 2, 2),
    (2, 1, 1, 0), (3, 2, 33, 16), (2, 2, 1024, 1024), (4, 1, 128, 0), (1, 2, 40, 24), (2, 1, 520, 512), (9, 3, 16, 16),
]


@pytest.mark.parametrize("dtype", [L.BF16, L.F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary", FORMS)
def test_forward(ctx, heads, kv_heads, dim, rotary, pairing, dtype):
    for tokens, norm, gap in ((1, True, 0), (13, True, 3), (6, False, 0)):
        forward(ctx, Case(tokens, heads, kv_heads, dim, rotary, pairing, norm, dtype, seed=tokens + dim, gap=gap))


@pytest.mark.parametrize("tokens", [2, 3, 5, 31, 257, 1000])
def test_forward_tokens(ctx, tokens):
    forward(ctx, Case(tokens, 4, 2, 128, 128, "halves", True, L.BF16, seed=tokens))


def test_forward_without_weights_queries_or_keys(ctx):
    forward(ctx, Case(5, 4, 2, 64, 64, "halves", True, L.BF16, weights=False))
    forward(ctx, Case(5, 4, 0, 64, 64, "halves", True, L.BF16))
    forward(ctx, Case(5, 0, 3, 64, 64, "neighbours", True, L.F32))


def test_far_positions(ctx):
    """Angles of positions up to 2^31 - 1 keep binary32's digits."""
    c = Case(64, 2, 1, 64, 64, "halves", False, L.F32, far=2 ** 31 - 1)
    c.positions[:4] = [2 ** 31 - 1, 2 ** 24 + 1, 0, 1]
    # beyond the bound: the product's own rounding, 2^-53 of the angle
    wq, _ = c.upload(ctx)
    dq = ctx.alloc(64 * 2 * 64 * 4)
    ctx.norm_rotate(c.dtype, c.layout(kv_heads=0), c.d_row.ptr, None, None, None, None, c.d_pos, c.d_freq, dq, None)
    got = dq.download(np.float32, (64, 2, 64)).astype(np.float64)
    want, bound = c.want("q")
    slack = 2.0 ** -52 * c.positions[:, None, None] * (bound / U32 / 32)
    close(got, want, bound + slack, c.dtype, "q")
    c.free()
    dq.free()


def test_ends_of_a_heads_values(ctx):
    """Zeros, a NaN, an infinity, heads of tiny and of large values."""
    c = Case(6, 2, 1, 64, 64, "halves", True, L.F32, seed=3)
    c.row_up[0] = 0
    c.row_up[1, 5] = np.nan
    c.row_up[2, 5] = np.inf
    c.row_up[3] *= 1e-30
    c.row_up[4] *= 1e15
    c.row = c.row_up.astype(np.float64)
    q, k = forward(ctx, c, check=False)
    assert np.isnan(q[1, 0]).all() and np.isnan(q[2, 0]).any() and np.isfinite(q[1, 1]).all() and not q[0].any()
    rows = [0, 3, 4, 5]
    for which, g in (("q", q), ("k", k)):
        with np.errstate(all="ignore"):
            want, bound = c.want(which)
        close(g[rows].astype(np.float64), want[rows], bound[rows] + 2.0 ** -140, c.dtype, which)


LAYOUTS = ["tokens", "heads", "padded"]


def paged(ctx, c, layout, page, pages, seed=1):
    """A cache of random bf16 values: (struct, host k, host v, buffers, strides)."""
    rng = np.random.default_rng(seed)
    token, head = (c.kv_heads * c.dim, c.dim) if layout == "tokens" else (c.dim, page * c.dim)
    page_stride = page * c.kv_heads * c.dim
    if layout == "padded":  # rows with gaps: heads outermost
        token, page_stride = c.dim + 8, page * (c.dim + 8) + 16
        head = pages * page_stride + 8
    at = (np.arange(pages)[:, None, None] * page_stride + np.arange(page)[None, :, None] * token
          + np.arange(c.kv_heads)[None, None, :] * head)[..., None] + np.arange(c.dim)
    host = [stored(rng.standard_normal(int(at.max()) + 1), L.BF16)[0] for _ in range(2)]
    bufs = [ctx.to_device(h) for h in host]
    struct = L.PagedCache(k=bufs[0].ptr, v=bufs[1].ptr, pages=pages, page=page, heads=c.kv_heads, head_dim=c.dim,
                          page_stride=page_stride, token_stride=token, head_stride=head)
    return struct, host, bufs, at


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page", [(32, 8, 128, 128, 16), (3, 3, 96, 32, 5), (5, 1, 80, 80, 1),
                                                            (2, 2, 33, 16, 7), (4, 2, 64, 64, 64)])
def test_store(ctx, heads, kv_heads, dim, rotary, page, layout):
    """Keys and values at their slots, all other bytes of the cache as they were;
    slots outside it store nothing."""
    for tokens, also in ((1, False), (19, True)):
        c = Case(tokens, heads, kv_heads, dim, rotary, "halves", True, L.BF16, seed=dim + tokens, gap=1 if dim == 33 else 0)
        pages = tokens // page + 3
        struct, host, bufs, at = paged(ctx, c, layout, page, pages)
        slots = c.rng.permutation(pages * page)[:tokens].astype(np.int32)
        if tokens > 4:
            slots[[2, 4]] = [-1, pages * page]
            slots[-1] = 2 ** 31 - 1
        wq, wk = c.upload(ctx)
        d_slots, dq, dk = ctx.to_device(slots), ctx.alloc(tokens * heads * dim * 2), ctx.alloc(tokens * kv_heads * dim * 2)
        ctx.norm_rotate(c.dtype, c.layout(), c.d_row.ptr, c.d_row.ptr + c.part("k")[1], c.d_row.ptr + c.part("v")[1], wq, wk,
                        c.d_pos, c.d_freq, dq, dk if also else None, struct, d_slots)
        ctx.synchronize()
        after = [b.download(np.uint16, h.shape) for b, h in zip(bufs, host)]
        want, bound = c.want("k")
        v = stored(c.part("v")[0], L.BF16)[0]
        rest = np.ones(host[0].shape, bool)
        for t, slot in enumerate(slots):
            if 0 <= slot < pages * page:
                where = at[slot // page, slot % page]
                close(values(after[0][where], L.BF16), want[t], bound[t], L.BF16, f"key {t}")
                np.testing.assert_array_equal(after[1][where], v[t])
                rest[where] = False
        for a, h in zip(after, host):
            np.testing.assert_array_equal(a[rest], h[rest])
        q_want, q_bound = c.want("q")
        close(values(dq.download(np.uint16, q_want.shape), L.BF16), q_want, q_bound, L.BF16, "q")
        if also:
            close(values(dk.download(np.uint16, want.shape), L.BF16), want, bound, L.BF16, "k")
        for b in bufs + [d_slots, dq, dk]:
            b.free()
        c.free()


def backward(ctx, c, wanted=("dq", "dk", "dwq", "dwk"), workspace=True):
    wq, wk = c.upload(ctx)
    dy_up, dy = {}, {}
    for which, n in (("q", c.heads), ("k", c.kv_heads)):
        dy_up[which], dy[which] = stored(0.1 * c.rng.standard_normal((c.tokens, n, c.dim)), c.dtype)
    d_dy = [ctx.to_device(dy_up[w]) for w in "qk"]
    marker = np.full((c.tokens, c.stride), 7.5, np.float32)
    d_dx = ctx.to_device(stored(marker, c.dtype)[0])
    d_dw = ctx.to_device(stored(np.full((2, c.dim), 7.5), c.dtype)[0])
    c.bufs += d_dy + [d_dx, d_dw]
    heads = c.layout()
    need = ctx.norm_rotate_backward_workspace(c.dtype, heads)
    space = ctx.alloc(max(need, 1))
    c.bufs.append(space)
    at = {"dq": d_dx.ptr, "dk": d_dx.ptr + c.part("k")[1], "dwq": d_dw.ptr, "dwk": d_dw.ptr + c.dim * c.elem}
    args = {name: at[name] for name in wanted if c.norm or not name.startswith("dw")}
    ctx.norm_rotate_backward(c.dtype, heads, d_dy[0], d_dy[1], c.d_row.ptr, c.d_row.ptr + c.part("k")[1], wq, wk, c.d_pos,
                             c.d_freq, **args, workspace=space if workspace else None, workspace_bytes=need)
    ctx.synchronize()
    store = np.uint16 if c.dtype == L.BF16 else np.float32
    dx = values(d_dx.download(store, (c.tokens, c.stride)), c.dtype)
    dw = values(d_dw.download(store, (2, c.dim)), c.dtype)
    rest = np.ones(c.stride, bool)
    for n, which in enumerate("qk"):
        x, offset = c.part(which)
        count = x.shape[1] * c.dim
        cols = slice(offset // c.elem, offset // c.elem + count)
        want, want_w, bound, bound_w = norm_rotate_backward(
            dy[which], x, c.w[n] if c.weights else None, c.positions, c.frequencies, c.rotary, c.pairing, EPS if c.norm else None)
        if "d" + which in args:
            close(dx[:, cols].reshape(want.shape), want, bound, c.dtype, "d" + which)
            rest[cols] = False
        if "dw" + which in args:
            close(dw[n], want_w, bound_w, c.dtype, "dw" + which)
        else:
            assert (dw[n] == 7.5).all()
    assert (dx[:, rest] == 7.5).all()  # columns of nothing that was asked for
    c.free()


@pytest.mark.parametrize("dtype", [L.BF16, L.F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary", FORMS)
def test_backward(ctx, heads, kv_heads, dim, rotary, pairing, dtype):
    for tokens, norm, gap in ((1, True, 0), (13, True, 3), (6, False, 0)):
        backward(ctx, Case(tokens, heads, kv_heads, dim, rotary, pairing, norm, dtype, seed=tokens + dim, gap=gap))


@pytest.mark.parametrize("tokens", [2, 3, 5, 31, 257, 1300])
def test_backward_tokens(ctx, tokens):
    backward(ctx, Case(tokens, 4, 2, 128, 128, "halves", True, L.BF16, seed=tokens))
    backward(ctx, Case(tokens, 2, 1, 24, 10, "halves", True, L.F32, seed=tokens))


@pytest.mark.parametrize("wanted", [("dq",), ("dk", "dwk"), ("dwq",), ("dwq", "dwk"), ("dq", "dwk")])
def test_backward_of_what_is_wanted(ctx, wanted):
    backward(ctx, Case(9, 4, 2, 64, 64, "halves", True, L.BF16), wanted)
    backward(ctx, Case(9, 4, 2, 34, 12, "neighbours", True, L.F32, weights=False), wanted, workspace=False)


def test_gradients_against_differences(ctx):
    """dx and dw of sum(dy * y) against central differences of the forward call, in
    f32 on steps that are exact: the forward's own rounding (bound above) over the
    step, and the third derivative's step^2, below 1e-3 of the sizes here."""
    c = Case(2, 1, 1, 8, 6, "halves", True, L.F32, seed=5)
    c.row_up[:] = np.random.default_rng(1).uniform(0.5, 1.5, c.row_up.shape).astype(np.float32)
    c.row = c.row_up.astype(np.float64)
    dy = np.random.default_rng(2).uniform(-1, 1, (2, 1, 8))
    want, want_w, _, _ = norm_rotate_backward(dy, c.part("q")[0], c.w[0], c.positions, c.frequencies, 6, "halves", EPS)
    step = np.float32(2.0 ** -6)

    def loss():
        return float((forward(ctx, c, check=False)[0].astype(np.float64) * dy).sum())

    for t in range(2):
        for i in range(8):
            at = c.row_up[t, i]
            sides = []
            for d in (step, -step):
                c.row_up[t, i] = at + d
                sides.append(loss())
            c.row_up[t, i] = at
            assert abs((sides[0] - sides[1]) / (2 * step) - want[t, 0, i]) < 1e-3
    for i in range(8):
        at = c.w_up[0, i]
        sides = []
        for d in (step, -step):
            c.w_up[0, i] = at + d
            sides.append((loss(), float(c.w_up[0, i])))
        c.w_up[0, i] = at
        assert abs((sides[0][0] - sides[1][0]) / (sides[0][1] - sides[1][1]) - want_w[i]) < 1e-3


def test_no_tokens(ctx):
    heads = Case(1, 2, 1, 8, 8, "halves", True, L.F32).layout(tokens=0)
    dw = ctx.to_device(np.full(16, 3, np.float32))
    ctx.norm_rotate(L.F32, heads, None, None, None, None, None, None, None, None, dw)
    ctx.norm_rotate_backward(L.F32, heads, None, None, None, None, None, None, None, None, dwq=dw, dwk=dw.ptr + 32)
    ctx.synchronize()
    assert not dw.download(np.float32, (16,)).any()
    dw.free()
