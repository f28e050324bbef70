"""Plain 64-bit forms of the feed-forward sublayer's operators, with bounds on
what binary32 arithmetic and one rounding of each result may add.

u is binary32's half step 2^-24; `half(bf16)` 2^-8, `half(f32)` 2^-24, relative
to the value rounded."""
from __future__ import annotations

import numpy as np

import oracle

U = 2.0 ** -24
EPS_BITS = 0x3727C5AC
EPS = float(np.uint32(EPS_BITS).view(np.float32))


def half(dtype: str) -> float:
    return 2.0 ** -8 if dtype == "bf16" else U


def store(dtype: str, values) -> np.ndarray:
    """Values as the operator's storage (bf16 bits, or f32)."""
    v = np.ascontiguousarray(values, dtype=np.float32)
    return oracle.bf16_narrow(v).reshape(v.shape) if dtype == "bf16" else v


def wide(dtype: str, stored) -> np.ndarray:
    a = np.asarray(stored)
    if dtype == "bf16":
        return oracle.bf16_widen(np.ascontiguousarray(a)).reshape(a.shape).astype(np.float64)
    return a.astype(np.float64)


def layer_norm(x, w, b, eps=EPS):
    mu = x.mean(-1, keepdims=True)
    d = x - mu
    r = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    xh = d * r
    return (xh if w is None else xh * w) + (0.0 if b is None else b), mu[..., 0], r[..., 0]


def layer_norm_bounds(dtype, x, w, b, eps=EPS):
    """A lane adds at most 40 values one after another (longer runs are summed
    in 64 bits), then at most 10 pairwise levels: a sum is within 50 u of the
    sum of magnitudes.  mu: that, over the count, and one rounding.  The
    differences carry mu's error and a rounding, r half the variance's (102 u
    of the squares' and mu's) and 4 u of its own, y five roundings more."""
    y, mu, r = layer_norm(x, w, b, eps)
    mag = np.abs(x).mean(-1, keepdims=True)
    e_mu = 52 * U * mag
    xh = np.abs((x - mu[:, None]) * r[:, None])
    # relative error of r: |d var| / (2 var) <= 60 u + e_mu^2 r^2, plus its own rounding
    e_r = 60 * U + (e_mu * r[:, None]) ** 2 + 4 * U
    e_xh = e_mu * r[:, None] + U * (np.abs(x) + np.abs(mu[:, None])) * r[:, None] + xh * (e_r + 4 * U)
    scale = 1.0 if w is None else np.abs(w)
    e_y = e_xh * scale + 2 * U * (xh * scale + (0.0 if b is None else np.abs(b)))
    return e_y + half(dtype) * (np.abs(y) + e_y), e_mu[:, 0], e_r[:, 0] * r


def layer_norm_backward(dy, x, w, mean, rstd):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy if w is None else dy * w
    c1, c2 = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    return rstd[:, None] * (g - c1 - xh * c2), (dy * xh).sum(0), dy.sum(0)


def layer_norm_backward_bounds(dtype, dy, x, w, mean, rstd):
    """xh: two roundings.  The row means: 50 u of the magnitudes, and the
    terms' own 4 u.  The column sums: a thread adds its rows one after
    another, then the partials: no more additions than rows + 600."""
    rows = x.shape[0]
    dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd)
    xh = np.abs((x - mean[:, None]) * rstd[:, None])
    e_xh = (np.abs(x) + np.abs(mean[:, None])) * rstd[:, None] * U + 2 * U * xh
    g = np.abs(dy if w is None else dy * w)
    m1, m2 = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    e_c1 = 52 * U * m1
    e_c2 = 56 * U * m2 + (g * e_xh).mean(-1, keepdims=True)
    c2 = np.abs((g * xh)).mean(-1, keepdims=True)
    e_dx = rstd[:, None] * (4 * U * g + e_c1 + 4 * U * m1 + xh * e_c2 + e_xh * c2 + 6 * U * xh * c2)
    n = min(rows, 1200) + 600
    e_dw = n * U * (np.abs(dy) * xh).sum(0) + (np.abs(dy) * e_xh).sum(0)
    e_db = n * U * np.abs(dy).sum(0)
    h = half(dtype)
    return (e_dx + h * (np.abs(dx) + e_dx), e_dw + h * (np.abs(dw) + e_dw), e_db + h * (np.abs(db) + e_db))


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def gated(x, wg, wu):
    g, u = x @ wg.T, x @ wu.T
    return g * sigmoid(g) * u, g, u


def gated_bounds(x, wg, wu):
    """A product of bf16 values is exact in binary32; k additions are within
    k u of the sum of magnitudes.  The activation: a slope of at most 1.1, and
    |G| log2(e) u of the exponent, three approximations of 2 u and two products."""
    k = x.shape[1]
    h, g, u = gated(x, wg, wu)
    e_g, e_u = k * U * (np.abs(x) @ np.abs(wg).T), k * U * (np.abs(x) @ np.abs(wu).T)
    e_h = 1.1 * e_g * (np.abs(u) + e_u) + np.abs(g * sigmoid(g)) * e_u + np.abs(h) * (12 + 2 * np.abs(g)) * U
    b = half("bf16")
    return e_h + b * (np.abs(h) + e_h), e_g + b * (np.abs(g) + e_g), e_u + b * (np.abs(u) + e_u)


def gated_backward(x, wg, wu, gate, up, dh):
    s = sigmoid(gate)
    du = dh * gate * s
    dg = dh * up * s * (1.0 + gate * (1.0 - s))
    return dg @ wg + du @ wu, dg.T @ x, du.T @ x


def gated_backward_bounds(x, wg, wu, gate, up, dh):
    """dG and dU are rounded to bf16 (half a step each) after some 24 + 3 |G|
    roundings of binary32 of their terms' magnitudes; the sums' additions are
    within their count of u."""
    s = sigmoid(gate)
    b = half("bf16")
    du = np.abs(dh * gate * s)
    terms = np.abs(dh * up * s) * (1.0 + np.abs(gate) * (1.0 - s))
    dg = np.abs(dh * up * s * (1.0 + gate * (1.0 - s)))
    few = (24 + 3 * np.abs(gate)) * U
    # 1 - s is taken of a rounded s: its absolute error is s's, 4 u
    e_dg = b * dg + few * terms + np.abs(dh * up * s * gate) * 4 * U
    e_du = (b + few) * du
    dx, dwg, dwu = gated_backward(x, wg, wu, gate, up, dh)
    n, m = gate.shape[1], gate.shape[0]
    e_dx = (e_dg + 2 * n * U * dg) @ np.abs(wg) + (e_du + 2 * n * U * du) @ np.abs(wu)
    e_dwg, e_dwu = (e_dg + m * U * dg).T @ np.abs(x), (e_du + m * U * du).T @ np.abs(x)
    return (e_dx + b * (np.abs(dx) + e_dx), e_dwg + b * (np.abs(dwg) + e_dwg), e_dwu + b * (np.abs(dwu) + e_dwu))


def quantize_rows(x):
    """(codes, scales) of f32 rows, exactly: quotients of binary32 numbers in
    64 bits never round onto a tie or off one."""
    x = np.asarray(x, dtype=np.float32)
    finite = np.isfinite(x).all(-1)
    top = np.abs(np.where(np.isfinite(x), x, 0)).max(-1)
    scale = np.maximum((top.astype(np.float64) / 127.0).astype(np.float32), np.float32(2.0 ** -126))
    with np.errstate(invalid="ignore"):
        q = np.rint(x.astype(np.float64) / scale.astype(np.float64)[:, None])
    q = np.where(finite[:, None], q, 0)
    return q.astype(np.int8), np.where(finite, scale, np.float32(np.nan)).astype(np.float32)


def contract_i8(a, b, sa, sb):
    """The f32 result, bit for bit."""
    total = a.astype(np.float64) @ b.astype(np.float64).T  # whole numbers below 2^31: exact
    with np.errstate(over="ignore", invalid="ignore"):
        return (total.astype(np.float32) * sa[:, None].astype(np.float32)) * sb[None, :].astype(np.float32)
