"""Host-level entry points mirroring tiler-reference's family functions, run on
the MI355X through the C ABI.

Each function takes and returns host numpy arrays with the reference's
argument meaning and refusal behaviour, moves the operands to HBM, launches the
gfx950 realization, and reads the result back.  The device kernels reduce the
last axis; a reduction over another axis is presented to them by moving that
axis last on the host (a pure relayout that changes no value).

Reference functions mirrored (paths under /root/reference/crates/):
  strict_sum                tiler-reference/src/evaluate.rs:498-589
  strict_partitioned_sum    tiler-reference/src/evaluate.rs:788-832
  cooperative_grouped_sum   tiler-reference/src/evaluate.rs:536-659
  rms_norm_f32              tiler-reference/src/rms_norm.rs:405-451
  softmax_f32               tiler-reference/src/softmax.rs:200-234
  silu_f32                  tiler-reference/src/silu.rs:486-533
  gather                    tiler-reference/src/structural.rs:513-606
  contract_strict_f32       tiler-reference/src/contraction.rs:297-333 (td,od->to)
"""
from __future__ import annotations

import numpy as np

from . import _lib as L
from .runtime import Context, GatherIndexOutOfBounds, Refusal, validate_gather_index

_default: Context | None = None


def default_context() -> Context:
    global _default
    if _default is None:
        _default = Context(0)
    return _default


def _ctx(ctx):
    return ctx if ctx is not None else default_context()


def _axis_last(values: np.ndarray, shape, axis: int):
    shape = tuple(int(s) for s in shape)
    if not 0 <= axis < len(shape):
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, "axis outside the shape")
    arr = np.asarray(values).reshape(shape)
    moved = np.moveaxis(arr, axis, -1)
    return np.ascontiguousarray(moved), moved.shape


def _run_rows(ctx, x: np.ndarray, out_dtype, out_count, launch):
    ctx = _ctx(ctx)
    dx = ctx.to_device(x)
    dy = ctx.alloc(max(out_count * np.dtype(out_dtype).itemsize, 1))
    try:
        launch(ctx, dx, dy)
        ctx.synchronize()
        return dy.download(out_dtype, (out_count,))
    finally:
        dx.free()
        dy.free()


# --- sums --------------------------------------------------------------------

def _sum(values, shape, axis, topology, ctx=None, **plan):
    x, moved_shape = _axis_last(np.asarray(values, dtype=np.float32), shape, axis)
    extent = moved_shape[-1]
    rows = int(np.prod(moved_shape[:-1], dtype=np.int64)) if len(moved_shape) > 1 else 1
    out = _run_rows(ctx, x.reshape(-1), np.float32, rows,
                    lambda c, dx, dy: c.sum_f32(dx, rows, extent, dy, topology=topology, **plan))
    return out.reshape(moved_shape[:-1])


def strict_sum(values, shape, axis: int, ctx=None) -> np.ndarray:
    """Serial topology: bit-exact with the strict left fold."""
    return _sum(values, shape, axis, L.SUM_SERIAL, ctx)


def strict_partitioned_sum(values, shape, axis: int, partitions: int,
                           contributors_per_partition: int, ctx=None) -> np.ndarray:
    return _sum(values, shape, axis, L.SUM_MULTIPASS, ctx, partitions=partitions,
                per_partition=contributors_per_partition)


def cooperative_grouped_sum(values, shape, axis: int, participants: int,
                            contributors_per_partition: int, rounds: int,
                            participant_major: bool = False, ctx=None) -> np.ndarray:
    return _sum(values, shape, axis, L.SUM_COOPERATIVE, ctx, participants=participants,
                per_partition=contributors_per_partition, rounds=rounds,
                participant_major=participant_major)


def tree_sum(values, shape, axis: int, ctx=None) -> np.ndarray:
    """The reassociating two-level tree (declared grouping)."""
    return _sum(values, shape, axis, L.SUM_TREE, ctx)


# --- row families --------------------------------------------------------------

def rms_norm_f32(shape, axis: int, eps_bits: int, values, weights, ctx=None) -> np.ndarray:
    """weights has the input's shape, as the reference requires."""
    x, moved_shape = _axis_last(np.asarray(values, dtype=np.float32), shape, axis)
    w, _ = _axis_last(np.asarray(weights, dtype=np.float32), shape, axis)
    extent = moved_shape[-1]
    rows = x.size // extent if extent else 0
    ctx = _ctx(ctx)
    dw = ctx.to_device(w.reshape(-1))
    try:
        out = _run_rows(ctx, x.reshape(-1), np.float32, x.size,
                        lambda c, dx, dy: c.rms_norm(L.F32, dx, dw, rows, extent, eps_bits, dy,
                                                     weight_broadcast=False))
    finally:
        dw.free()
    return np.moveaxis(out.reshape(moved_shape), -1, axis).reshape(-1)


def rms_norm_bf16(values_bits: np.ndarray, weight_bits: np.ndarray, eps_bits: int,
                  ctx=None) -> np.ndarray:
    """bf16 [rows, extent] x bf16 [extent] -> bf16 [rows, extent] (bit patterns)."""
    x = np.ascontiguousarray(values_bits, dtype=np.uint16)
    rows, extent = x.shape
    ctx = _ctx(ctx)
    dw = ctx.to_device(np.ascontiguousarray(weight_bits, dtype=np.uint16))
    try:
        out = _run_rows(ctx, x.reshape(-1), np.uint16, x.size,
                        lambda c, dx, dy: c.rms_norm(L.BF16, dx, dw, rows, extent, eps_bits, dy,
                                                     weight_broadcast=True))
    finally:
        dw.free()
    return out.reshape(rows, extent)


def softmax_f32(shape, axis: int, values, ctx=None) -> np.ndarray:
    x, moved_shape = _axis_last(np.asarray(values, dtype=np.float32), shape, axis)
    extent = moved_shape[-1]
    rows = x.size // extent if extent else 0
    out = _run_rows(ctx, x.reshape(-1), np.float32, x.size,
                    lambda c, dx, dy: c.softmax_f32(dx, rows, extent, dy))
    return np.moveaxis(out.reshape(moved_shape), -1, axis).reshape(-1)


def silu_f32(values, ctx=None) -> np.ndarray:
    x = np.ascontiguousarray(values, dtype=np.float32).reshape(-1)
    return _run_rows(ctx, x, np.float32, x.size,
                     lambda c, dx, dy: c.map(L.MAP_SILU, L.F32, dx, x.size, dy))


# --- bf16 <-> binary32 conversion (ADR 0091 decision 2) -------------------------

def narrow_f32_bf16(values, ctx=None) -> np.ndarray:
    """binary32 -> bf16 bit patterns: round to nearest even, overflow to a
    signed infinity at the inclusive midpoint, every NaN -> 0x7fc0."""
    x = np.ascontiguousarray(values, dtype=np.float32).reshape(-1)
    return _run_rows(ctx, x, np.uint16, x.size,
                     lambda c, dx, dy: c.convert(L.CONVERT_NARROW_F32_BF16, dx, x.size, dy))


def widen_bf16_f32(bits, ctx=None) -> np.ndarray:
    """bf16 bit patterns -> binary32, exactly (a NaN keeps its payload)."""
    b = np.ascontiguousarray(bits, dtype=np.uint16).reshape(-1)
    return _run_rows(ctx, b, np.float32, b.size,
                     lambda c, dx, dy: c.convert(L.CONVERT_WIDEN_BF16_F32, dx, b.size, dy))


# --- gather --------------------------------------------------------------------

def gather(source: np.ndarray, axis: int, index: np.ndarray, index_signed: bool = False,
           ctx=None) -> np.ndarray:
    """Result shape = source.shape[:axis] + index.shape + source.shape[axis+1:].
    An out-of-range index raises GatherIndexOutOfBounds before any device work."""
    src = np.ascontiguousarray(source)
    idx = np.ascontiguousarray(np.asarray(index).astype(np.int64).astype(np.uint32)
                               if np.asarray(index).dtype != np.uint32 else index)
    gathered = src.shape[axis]
    validate_gather_index(idx.reshape(-1), gathered, index_signed)
    outer = int(np.prod(src.shape[:axis], dtype=np.int64)) if axis else 1
    inner = int(np.prod(src.shape[axis + 1:], dtype=np.int64)) if axis + 1 < src.ndim else 1
    out_shape = src.shape[:axis] + np.asarray(index).shape + src.shape[axis + 1:]
    count = idx.size
    ctx = _ctx(ctx)
    ds = ctx.to_device(src.reshape(-1))
    di = ctx.to_device(idx.reshape(-1))
    n_out = outer * count * inner
    do = ctx.alloc(max(n_out * src.itemsize, 1))
    try:
        ctx.gather(ds, outer, gathered, inner, src.itemsize, di, count, do,
                   index_signed=index_signed)
        ctx.gather_status()
        out = do.download(src.dtype, (n_out,))
    finally:
        ds.free()
        di.free()
        do.free()
    return out.reshape(out_shape)


# --- contraction ------------------------------------------------------------------

def contract_strict_f32(a: np.ndarray, b: np.ndarray, ctx=None) -> np.ndarray:
    """td,od->to: A [m, k], B [n, k] -> C [m, n], the strict fold."""
    a = np.ascontiguousarray(a, dtype=np.float32)
    b = np.ascontiguousarray(b, dtype=np.float32)
    m, k = a.shape
    n, k2 = b.shape
    if k != k2:
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, "contracted extents disagree")
    ctx = _ctx(ctx)
    da, db = ctx.to_device(a), ctx.to_device(b)
    dc = ctx.alloc(max(m * n * 4, 1))
    try:
        ctx.contract_strict_f32(da, db, m, n, k, dc)
        ctx.synchronize()
        return dc.download(np.float32, (m, n))
    finally:
        da.free()
        db.free()
        dc.free()


def contract_bf16(a_bits: np.ndarray, b_bits: np.ndarray, epilogue: int = L.EPILOGUE_NONE,
                  ctx=None) -> np.ndarray:
    """bf16 A [m, k], B [n, k] (bit patterns) -> bf16 C [m, n] on MFMA."""
    a = np.ascontiguousarray(a_bits, dtype=np.uint16)
    b = np.ascontiguousarray(b_bits, dtype=np.uint16)
    m, k = a.shape
    n, k2 = b.shape
    if k != k2:
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, "contracted extents disagree")
    ctx = _ctx(ctx)
    da, db = ctx.to_device(a), ctx.to_device(b)
    dc = ctx.alloc(max(m * n * 2, 1))
    try:
        ctx.contract_bf16(da, db, m, n, k, dc, epilogue)
        ctx.synchronize()
        return dc.download(np.uint16, (m, n))
    finally:
        da.free()
        db.free()
        dc.free()


def dequantize_u4(packed: np.ndarray, n: int, scale_bits: int, zero_point: int, ctx=None) -> np.ndarray:
    """Strict-affine U4 -> f32 on the device (quantization.rs:218-246):
    `packed` holds n U4 codes LSB-first in (n + 1) // 2 U8 carriers."""
    p = np.ascontiguousarray(np.asarray(packed, dtype=np.uint8))
    if p.size < (n + 1) // 2:
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, "dequantize_u4", "fewer carriers than codes")
    ctx = _ctx(ctx)
    dc = ctx.to_device(p) if p.size else ctx.alloc(1)
    dy = ctx.alloc(max(4 * n, 1))
    try:
        ctx.dequantize_u4(dc, n, scale_bits, zero_point, dy)
        ctx.synchronize()
        return dy.download(np.float32, (n,))
    finally:
        dc.free()
        dy.free()


# --- the feed-forward sublayer (no reference counterpart) ----------------------
# Storage by numpy dtype: float32, or uint16 holding bf16 patterns.

def _storage(values, what: str):
    a = np.ascontiguousarray(values)
    if a.ndim != 2 or a.dtype not in (np.float32, np.uint16):
        raise Refusal(L.REFUSE_UNSUPPORTED, what, "rows in two dimensions, float32 or uint16 (bf16 patterns)")
    return a, L.F32 if a.dtype == np.float32 else L.BF16


def _operand(values, dtype, shape, what: str):
    a = np.ascontiguousarray(values)
    if a.dtype != dtype or a.shape != tuple(shape):
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, what, f"an operand is {a.dtype}{list(a.shape)}, not {np.dtype(dtype)}{list(shape)}")
    return a


def _run(ctx, inputs, outputs, launch):
    """launch(context, device inputs, device outputs); the outputs, (dtype, shape) each, on the host."""
    ctx = _ctx(ctx)
    bufs = []
    try:
        for a in inputs:
            bufs.append(None if a is None else ctx.to_device(a))
        for dtype, shape in outputs:
            bufs.append(ctx.alloc(max(int(np.prod(shape, dtype=np.int64)) * np.dtype(dtype).itemsize, 1)))
        out = bufs[len(inputs):]
        launch(ctx, bufs[:len(inputs)], out)
        ctx.synchronize()
        return [b.download(dtype, shape) for b, (dtype, shape) in zip(out, outputs)]
    finally:
        for b in bufs:
            if b is not None:
                b.free()


def layer_norm(values, weights=None, bias=None, eps_bits: int = 0x3727C5AC, ctx=None):
    """(y, mean, rstd) of the rows of `values` [rows, extent]; weights and bias
    [extent] or None (ones, zeros)."""
    x, code = _storage(values, "layer_norm")
    rows, extent = x.shape
    wb = [None if v is None else _operand(v, x.dtype, (extent,), "layer_norm") for v in (weights, bias)]
    return tuple(_run(ctx, [x, *wb], [(x.dtype, x.shape), (np.float32, (rows,)), (np.float32, (rows,))],
                      lambda c, i, o: c.layer_norm(code, *i, rows, extent, eps_bits, *o)))


def layer_norm_backward(dy, values, weights, mean, rstd, ctx=None):
    """(dx, dw, db) from dy and what layer_norm returned."""
    x, code = _storage(values, "layer_norm_backward")
    rows, extent = x.shape
    dy = _operand(dy, x.dtype, x.shape, "layer_norm_backward")
    w = None if weights is None else _operand(weights, x.dtype, (extent,), "layer_norm_backward")
    stats = [_operand(v, np.float32, (rows,), "layer_norm_backward") for v in (mean, rstd)]
    return tuple(_run(ctx, [dy, x, w, *stats], [(x.dtype, x.shape), (x.dtype, (extent,)), (x.dtype, (extent,))],
                      lambda c, i, o: c.layer_norm_backward(code, *i, rows, extent, *o)))


def _gated_operands(x, wg, wu, what: str):
    x = np.ascontiguousarray(x)
    wg = np.ascontiguousarray(wg)
    if x.ndim != 2 or wg.ndim != 2 or x.dtype != np.uint16:
        raise Refusal(L.REFUSE_UNSUPPORTED, what, "rows in two dimensions, uint16 (bf16 patterns)")
    (m, k), n = x.shape, wg.shape[0]
    return m, n, k, [x, _operand(wg, np.uint16, (n, k), what), _operand(wu, np.uint16, (n, k), what)]


def gated_contract_bf16(x, wg, wu, ctx=None):
    """(h, gate, up): h = silu(x wg^T) * (x wu^T) of bf16 patterns, x [m, k],
    wg and wu [n, k]; gate and up are the two products."""
    m, n, k, operands = _gated_operands(x, wg, wu, "gated_contract_bf16")
    return tuple(_run(ctx, operands, [(np.uint16, (m, n))] * 3, lambda c, i, o: c.gated_contract_bf16(*i, m, n, k, *o)))


def gated_contract_bf16_backward(x, wg, wu, gate, up, dh, ctx=None):
    """(dx, dwg, dwu) from dh and what gated_contract_bf16 returned."""
    what = "gated_contract_bf16_backward"
    m, n, k, operands = _gated_operands(x, wg, wu, what)
    operands += [_operand(v, np.uint16, (m, n), what) for v in (gate, up, dh)]
    return tuple(_run(ctx, operands, [(np.uint16, (m, k)), (np.uint16, (n, k)), (np.uint16, (n, k))],
                      lambda c, i, o: c.gated_contract_bf16_backward(*i, m, n, k, *o)))


def quantize_rows_i8(values, ctx=None):
    """(codes int8, scales float32) of the rows of `values` [rows, extent]."""
    x, code = _storage(values, "quantize_rows_i8")
    rows, extent = x.shape
    return tuple(_run(ctx, [x], [(np.int8, x.shape), (np.float32, (rows,))],
                      lambda c, i, o: c.quantize_rows_i8(code, *i, rows, extent, *o)))


def contract_i8(a, b, a_scales, b_scales, out_dtype=np.float32, ctx=None):
    """int8 a [m, k], b [n, k] with a scale a row each -> [m, n], float32 or
    uint16 (bf16 patterns)."""
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    if a.ndim != 2 or b.ndim != 2 or out_dtype not in (np.float32, np.uint16):
        raise Refusal(L.REFUSE_UNSUPPORTED, "contract_i8", "operands in two dimensions, a float32 or uint16 result")
    (m, k), n = a.shape, b.shape[0]
    operands = [_operand(a, np.int8, (m, k), "contract_i8"), _operand(b, np.int8, (n, k), "contract_i8"),
                _operand(a_scales, np.float32, (m,), "contract_i8"), _operand(b_scales, np.float32, (n,), "contract_i8")]
    code = L.F32 if out_dtype == np.float32 else L.BF16
    return _run(ctx, operands, [(out_dtype, (m, n))], lambda c, i, o: c.contract_i8(*i, m, n, k, code, *o))[0]


# --- the attention sublayer (no reference counterpart) --------------------------

def _int32(values, what: str):
    """Whole numbers as i32; refused where that would change one."""
    a = np.asarray(values)
    with np.errstate(invalid="ignore"):
        b = np.ascontiguousarray(a.astype(np.int32)) if a.dtype.kind in "biuf" else None
    if b is None or not np.array_equal(a, b):
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, what, "a list holds more than whole numbers of 32 bits")
    return b


def _counts(what: str, **values):
    """Sizes that are passed on as unsigned numbers of 32 bits."""
    for name, v in values.items():
        if not 0 <= v < 1 << 32:
            raise Refusal(L.REFUSE_INVALID_ARGUMENT, what, f"{name} is {v}")


def page_slots(kept, fresh, page: int, free_pages, table, tokens: int | None = None, ctx=None):
    """(table, starts, lengths, positions, slots, taken) of a batch whose
    sequences hold `kept` tokens and get `fresh` more; table [sequences, width]
    names the kept tokens' pages, and the new pages come from free_pages.
    `tokens`: rows of the batch (default: the sum of fresh)."""
    kept, fresh, free = (_int32(v, "page_slots").reshape(-1) for v in (kept, fresh, free_pages))
    table = _int32(table, "page_slots")
    if table.ndim != 2 or not len(kept) == len(fresh) == len(table):
        raise Refusal(L.REFUSE_INVALID_ARGUMENT, "page_slots", "a length of each kind and a row of the table for each sequence")
    if tokens is None:
        tokens = int(np.maximum(fresh, 0).sum(dtype=np.int64))
    _counts("page_slots", page=page, tokens=tokens)
    n, i32 = len(kept), np.int32

    def launch(c, i, o):
        if table.size:
            c.copy(o[0], i[3], table.nbytes)
        c.page_slots(i[0], i[1], n, page, i[2], len(free), o[0], table.shape[1], tokens, *o[1:])

    return tuple(_run(ctx, [kept, fresh, free, table],
                      [(i32, table.shape), (i32, (n + 1,)), (i32, (n,)), (i32, (tokens,)), (i32, (tokens,)), (i32, (1,))], launch))


def _heads(q, k, rotary, pairing, eps_bits, frequencies, positions, what: str):
    q, k = np.ascontiguousarray(q), np.ascontiguousarray(k)
    if q.ndim != 3 or k.ndim != 3 or q.dtype != k.dtype or q.dtype not in (np.float32, np.uint16) or \
            q.shape[::2] != k.shape[::2] or pairing not in ("halves", "neighbours"):
        raise Refusal(L.REFUSE_UNSUPPORTED, what,
                      "q and k [tokens, heads, head_dim], float32 or uint16 (bf16 patterns), pairs as halves or neighbours")
    (tokens, q_heads, dim), kv_heads = q.shape, k.shape[1]
    _counts(what, rotary=rotary, eps_bits=eps_bits)
    positions = _operand(positions, np.int32, (tokens,), what)
    frequencies = _operand(frequencies, np.float64, (rotary // 2,), what)
    layout = L.HeadLayout(tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=dim, rotary=rotary,
                          pairing=L.ROTATE_HALVES if pairing == "halves" else L.ROTATE_NEIGHBOURS, eps_bits=eps_bits,
                          q_stride=q_heads * dim, k_stride=kv_heads * dim, q_out_stride=q_heads * dim, k_out_stride=kv_heads * dim)
    return q, k, layout, L.F32 if q.dtype == np.float32 else L.BF16, [positions, frequencies]


def norm_rotate(q, k, wq, wk, positions, frequencies, rotary: int, pairing: str = "halves", eps_bits: int = 0x358637BD, ctx=None):
    """(q_out, k_out): each head normed (eps_bits 0: not) and its first `rotary`
    elements turned by positions [tokens] times frequencies [rotary / 2]; wq and
    wk [head_dim] or None."""
    q, k, layout, code, turn = _heads(q, k, rotary, pairing, eps_bits, frequencies, positions, "norm_rotate")
    w = [None if v is None else _operand(v, q.dtype, q.shape[2:], "norm_rotate") for v in (wq, wk)]
    return tuple(_run(ctx, [q, k, *w, *turn], [(q.dtype, q.shape), (k.dtype, k.shape)],
                      lambda c, i, o: c.norm_rotate(code, layout, i[0], i[1], None, *i[2:], *o)))


def norm_rotate_backward(dq_out, dk_out, q, k, wq, wk, positions, frequencies, rotary: int, pairing: str = "halves",
                         eps_bits: int = 0x358637BD, ctx=None):
    """(dq, dk, dwq, dwk) of norm_rotate; without a norm dwq and dwk are None."""
    what = "norm_rotate_backward"
    q, k, layout, code, turn = _heads(q, k, rotary, pairing, eps_bits, frequencies, positions, what)
    dy = [_operand(d, x.dtype, x.shape, what) for d, x in ((dq_out, q), (dk_out, k))]
    w = [None if v is None else _operand(v, q.dtype, q.shape[2:], what) for v in (wq, wk)]
    outputs = [(q.dtype, q.shape), (k.dtype, k.shape)] + ([(q.dtype, q.shape[2:])] * 2 if eps_bits else [])
    got = _run(ctx, [*dy, q, k, *w, *turn], outputs,
               lambda c, i, o: c.norm_rotate_backward(code, layout, *i, *o))
    return tuple(got) if eps_bits else (*got, None, None)


def paged_attention_bf16(q, k_cache, v_cache, table, starts, lengths, scale: float, window: int = 0, sinks: int = 0, ctx=None):
    """out [tokens, heads, head_dim]: the attention of q's rows over the cache
    [pages, page, kv_heads, head_dim] (bf16 patterns); rows of no sequence are 0."""
    what = "paged_attention_bf16"
    q, k_cache, v_cache = (np.ascontiguousarray(a) for a in (q, k_cache, v_cache))
    table = _int32(table, what)
    _counts(what, window=window, sinks=sinks)
    if q.ndim != 3 or k_cache.ndim != 4 or table.ndim != 2 or q.dtype != np.uint16 or q.shape[2] != k_cache.shape[3]:
        raise Refusal(L.REFUSE_UNSUPPORTED, what, "q [tokens, heads, head_dim] and the cache [pages, page, heads, head_dim], uint16")
    k_cache, v_cache = (_operand(a, np.uint16, k_cache.shape, what) for a in (k_cache, v_cache))
    starts = _operand(starts, np.int32, (len(table) + 1,), what)
    lengths = _operand(lengths, np.int32, (len(table),), what)
    (tokens, heads, dim), (pages, page, kv_heads, _) = q.shape, k_cache.shape
    shape = L.AttentionShape(tokens=tokens, sequences=len(table), q_heads=heads, scale=scale, q_stride=heads * dim,
                             out_stride=heads * dim, table_width=table.shape[1], window=window, sinks=sinks,
                             max_fresh=max(int(np.diff(starts).max(initial=0)), 0), max_length=max(int(lengths.max(initial=0)), 0))

    def launch(c, i, o):
        cache = L.PagedCache(k=i[1].ptr, v=i[2].ptr, pages=pages, page=page, heads=kv_heads, head_dim=dim,
                             page_stride=page * kv_heads * dim, token_stride=kv_heads * dim, head_stride=dim)
        if q.size:
            c.copy(o[0], i[6], q.nbytes)
        c.paged_attention_bf16(shape, i[0], cache, *i[3:6], o[0])

    return _run(ctx, [q, k_cache, v_cache, table, starts, lengths, np.zeros_like(q)], [(np.uint16, q.shape)], launch)[0]


__all__ = [
    "strict_sum", "strict_partitioned_sum", "cooperative_grouped_sum", "tree_sum",
    "rms_norm_f32", "rms_norm_bf16", "softmax_f32", "silu_f32", "gather",
    "contract_strict_f32", "contract_bf16", "dequantize_u4", "layer_norm", "layer_norm_backward", "gated_contract_bf16",
    "gated_contract_bf16_backward", "quantize_rows_i8", "contract_i8", "page_slots", "norm_rotate", "norm_rotate_backward",
    "paged_attention_bf16", "default_context", "GatherIndexOutOfBounds",
]
