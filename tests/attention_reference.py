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

    bound: the weights w_j are rounded to bf16, for the product with v and for their
    sum alike: sum w_j (1 + e_j) v_j / sum w_j (1 + e_j) is off by sum w_j e_j (v_j -
    out) / (1 - U16), at most U16 (1 + 2 U16) sum w |v - out|; the result to bf16 (U16
    of itself); a logit of dim products is off by dim / 16 + 16 roundings at most in
    each of the matrix unit's running sums, taken as dim, on scale * sum |q k|, twice
    that where it enters the weight and the weights' sum; the sums over the keys
    (chains of at most keys / 16 + 32 steps, with their rescaling) and the exponential
    add the rest."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, bound = np.array(out, np.float64), np.zeros(np.shape(out))
    pages, page, kv_heads, dim = k.shape
    group = q.shape[1] // kv_heads
    for s in range(len(lengths)):
        fresh = int(starts[s + 1] - starts[s])
        most = max(min(int(lengths[s]), table.shape[1] * page), 0)
        keys = np.arange(most)
        entry = table[s, keys // page] if most else keys
        there = (entry >= 0) & (entry < pages)
        at = np.where(there, entry, 0)
        for h in range(kv_heads):
            kk = np.where(there[:, None], k[at, keys % page, h], 0.0) if most else np.zeros((0, dim))
            vv = np.where(there[:, None], v[at, keys % page, h], 0.0) if most else np.zeros((0, dim))
            k_size, v_size, v_square = np.abs(kk), np.abs(vv), vv * vv
            for i in range(fresh):
                p, row = int(lengths[s]) - fresh + i, starts[s] + i
                j = keys[:max(p + 1, 0)]
                if window:
                    j = j[(j > p - window) | (j < sinks)]
                rows = (row, slice(h * group, (h + 1) * group))
                if not len(j):
                    out[rows] = 0.0
                    continue
                of_j = slice(j[0], j[-1] + 1) if len(j) == j[-1] - j[0] + 1 else j  # no copy where nothing lies between
                kj, vj = kk[of_j], vv[of_j]
                logits = scale * (q[rows] @ kj.T)
                top = logits.max(1, keepdims=True)
                w = np.exp(logits - np.where(top == -np.inf, 0.0, top))
                total = w.sum(1, keepdims=True)
                w /= np.where(total == 0.0, 1.0, total)
                o = w @ vj
                sizes = w @ v_size[of_j]
                # sum w |v - out| by Cauchy's inequality: no term for each key, element and row
                spread = np.sqrt(np.maximum(w @ v_square[of_j] - o * o * (2 - w.sum(1, keepdims=True)), 0.0))
                off = scale * (np.abs(q[rows]) @ k_size[of_j].T).max(1, keepdims=True)
                out[rows] = o
                bound[rows] = (U16 * (np.abs(o) * (1 + U16) + (1 + 2 * U16) * np.minimum(spread, sizes + np.abs(o)))
                               + U32 * (2 * (dim + 16) * off + len(j) / 8 + 96) * sizes)
                dead = np.nonzero(total[:, 0] == 0.0)[0]  # every logit -infinity
                out[row, h * group + dead], bound[row, h * group + dead] = 0.0, 0.0
    return out, bound
