"""The attention sublayer from its definitions, in 64 bits and plain loops:
page tables and slots, head norms with the rotation and their gradients,
attention over a paged cache; and the bounds that the tests hold the kernels to.

A rounding is off by at most half a step: U32 (binary32) and U16 (bf16) relative
to the value.  Each bound counts the roundings between the operands and the
result, at their worst."""
from __future__ import annotations

import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8


# -- page tables ----------------------------------------------------------------
def page_slots(kept, fresh, page, free, table, tokens):
    """(table, starts, lengths, positions, slots, taken)."""
    top = 2 ** 31 - 1
    table = np.array(table, np.int64)
    width = table.shape[1]
    starts, lengths, positions, slots, taken = [0], [], [0] * tokens, [-1] * tokens, 0
    for s, (have_tokens, new) in enumerate(zip(kept, fresh)):
        have_tokens, new = max(int(have_tokens), 0), max(int(new), 0)
        have = -(-have_tokens // page)
        for j in range(have, min(-(-(have_tokens + new) // page), width)):
            if starts[-1] + max(j * page - have_tokens, 0) < tokens:  # the token that opens the page has a row
                table[s, j] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(new):
            row, position = starts[-1] + i, have_tokens + i
            if row < tokens:
                entry = table[s, position // page] if position // page < width else -1
                slot = entry * page + position % page
                positions[row] = min(position, top)
                slots[row] = slot if 0 <= entry and slot <= top else -1
        starts.append(starts[-1] + new)
        lengths.append(have_tokens + new)
    cut = lambda v: np.minimum(np.array(v, np.int64), top).astype(np.int32)
    return table.astype(np.int32), cut(starts), cut(lengths), cut(positions), cut(slots), min(taken, top)


# -- head norms and rotation ------------------------------------------------------
def pairs(dim, rotary, pairing):
    p = np.arange(rotary // 2)
    return (p, p + rotary // 2) if pairing == "halves" else (2 * p, 2 * p + 1)


def angles(positions, frequencies):
    a = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    return np.cos(a)[:, None, :], np.sin(a)[:, None, :]


def _turned(x, cos, sin, i, j):
    y = x.copy()
    y[..., i] = x[..., i] * cos - x[..., j] * sin
    y[..., j] = x[..., j] * cos + x[..., i] * sin
    return y


def norm_rotate(x, w, positions, frequencies, rotary, pairing, eps):
    """(y, bound) of heads x [tokens, heads, dim]; eps None: no norm.

    bound: the mean of squares is a sum of dim terms in lanes of dim / 64 (at most
    16) and six folds, half of whose error reaches r; the division, the root, two
    products with r and w, the rotation's two products and its sum, and cos and
    sin, off by two roundings and their series' 3e-8 each: below 32 of binary32."""
    x = np.asarray(x, np.float64)
    i, j = pairs(x.shape[-1], rotary, pairing)
    u = x
    if eps is not None:
        u = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            u = u * np.asarray(w, np.float64)
    cos, sin = angles(positions, frequencies)
    size = np.abs(u)
    size[..., i], size[..., j] = size[..., i] + size[..., j], size[..., i] + size[..., j]
    return _turned(u, cos, sin, i, j), 32 * U32 * size


def norm_rotate_backward(dy, x, w, positions, frequencies, rotary, pairing, eps):
    """(dx, dw, bound of dx, bound of dw).  The bounds count as above: g (4
    roundings on |dy_i| + |dy_j|), r and xh (20), the mean over the head (dim / 64 + 6
    and the products), dx's own; dw a sum of tokens * heads terms in some order."""
    dy = np.asarray(dy, np.float64)
    i, j = pairs(dy.shape[-1], rotary, pairing)
    cos, sin = angles(positions, frequencies)
    g = _turned(dy, cos, -sin, i, j)
    size = np.abs(dy)
    size[..., i], size[..., j] = size[..., i] + size[..., j], size[..., i] + size[..., j]
    if eps is None:
        return g, None, 8 * U32 * size, None
    x = np.asarray(x, np.float64)
    wide = np.ones(dy.shape[-1]) if w is None else np.asarray(w, np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * r
    dx = r * (g * wide - xh * (g * wide * xh).mean(-1, keepdims=True))
    of_dx = 64 * U32 * r * (size * np.abs(wide) + np.abs(xh) * (size * np.abs(wide * xh)).mean(-1, keepdims=True))
    terms = dy.shape[0] * dy.shape[1]
    return dx, (g * xh).sum((0, 1)), of_dx, (terms + 64) * U32 * (size * np.abs(xh)).sum((0, 1))


# -- attention ---------------------------------------------------------------------
def paged_attention(q, k, v, table, starts, lengths, scale, window, sinks, out):
    """(out, bound): q [tokens, heads, dim], k and v [pages, page, kv_heads, dim] in
    64 bits; rows of no sequence keep what `out` holds, with a bound of 0.

    bound: the weights are rounded to bf16 for the product with v (U16 of sum w |v|),
    the result to bf16 (U16 of itself); a logit of dim products is off by dim / 16
    + 16 roundings at most in each of the matrix unit's running sums, taken as dim,
    on scale * sum |q k|, twice that where it enters the weight and the weights'
    sum; the sums over the keys (chains of at most keys / 16 + 32 steps, with their
    rescaling) and the exponential add the rest."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, bound = np.array(out, np.float64), np.zeros(np.shape(out))
    pages, page, kv_heads, dim = k.shape
    group = q.shape[1] // kv_heads
    for s in range(len(lengths)):
        fresh = starts[s + 1] - starts[s]
        for i in range(fresh):
            p, row = lengths[s] - fresh + i, starts[s] + i
            j = np.arange(max(min(p + 1, table.shape[1] * page), 0))
            if window:
                j = j[(j > p - window) | (j < sinks)]
            entry = table[s, j // page] if len(j) else j
            there = (entry >= 0) & (entry < pages)
            at = np.where(there, entry, 0)
            for h in range(q.shape[1]):
                kk = np.where(there[:, None], k[at, j % page, h // group], 0.0) if len(j) else np.zeros((0, dim))
                vv = np.where(there[:, None], v[at, j % page, h // group], 0.0) if len(j) else np.zeros((0, dim))
                logits = scale * (kk @ q[row, h])
                if not len(j) or logits.max() == -np.inf:
                    out[row, h] = 0.0
                    continue
                w = np.exp(logits - logits.max())
                w /= w.sum()
                out[row, h] = w @ vv
                sizes = w @ np.abs(vv)
                off = scale * (np.abs(kk) @ np.abs(q[row, h])).max()
                bound[row, h] = (U16 * (np.abs(out[row, h]) * (1 + U16) + sizes)
                                 + U32 * (2 * (dim + 16) * off + len(j) / 8 + 96) * sizes)
    return out, bound
