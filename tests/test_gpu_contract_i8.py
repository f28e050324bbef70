"""The 8-bit linear layer on the device: codes, scales and products bit for
bit with the exact definitions."""
from __future__ import annotations

import numpy as np
import pytest

import feed_forward_reference as ref
import oracle
from tiler_amd import _lib as L
from tiler_amd.realize import realize
from test_gpu_layer_norm import CODE, ROW_FORMS, Buffers, storage

pytestmark = pytest.mark.gpu


@pytest.fixture
def mem(ctx):
    m = Buffers(ctx)
    yield m
    m.free()


def quantize(ctx, mem, dtype, x, shift=0):
    rows, extent = x.shape
    q, s = mem.out(np.int8, rows * extent, shift), mem.out(np.float32, rows)
    ctx.quantize_rows_i8(CODE[dtype], mem.put(x, shift), rows, extent, q, s)
    ctx.synchronize()
    return mem.get(q, np.int8, (rows, extent)), mem.get(s, np.float32, (rows,))


def check_quantize(ctx, mem, dtype, x, shift=0):
    q, s = quantize(ctx, mem, dtype, x, shift)
    wq, ws = ref.quantize_rows(ref.wide(dtype, x))
    assert np.array_equal(s, ws, equal_nan=True), np.flatnonzero(s != ws)[:4]
    assert np.array_equal(q, wq), np.argwhere(q != wq)[:4]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("extent", [1, 3, 16, 63, 64, 100, 512, 1000, 1111, 2048, 4096, 5001, 8192, 8193, 16400, 40000])
def test_quantize(ctx, mem, dtype, extent):
    rng = np.random.default_rng(extent)
    for rows in (1, 6, 130):
        x = rng.standard_normal((rows, extent)) * np.exp(rng.normal(0, 3, (rows, 1)))
        for shift in (0, 1):
            check_quantize(ctx, mem, dtype, ref.store(dtype, x), shift)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("form,rows,extent", ROW_FORMS)
def test_quantize_forms(ctx, mem, dtype, form, rows, extent):
    extent = extent if dtype == "bf16" else extent // 2
    if dtype == "bf16" and form == "w1c4":
        form = "w4c1"  # more than two pieces a thread
    rz = realize(L.PROGRAM_QUANTIZE_ROWS_I8, (rows, extent), dtype=CODE[dtype], permissions=L.PERMITS_REASSOCIATION)
    assert rz.symbols == [f"tiler_quantize_rows_i8_{dtype}_{form}"]
    check_quantize(ctx, mem, dtype, ref.store(dtype, np.random.default_rng(extent).standard_normal((rows, extent))))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_ties(ctx, mem, dtype):
    """Quotients that are exactly half-way, and a step of binary32 to each side."""
    rows = []
    for top in (127.0, 254.0, 127.0 * 2.0 ** -100, 127.0 * 2.0 ** 90, 127.0 * 3.0, 63.5):
        s = np.float32(top) / np.float32(127.0)
        half = (np.arange(-126, 126) + 0.5).astype(np.float32) * s
        v = np.concatenate([[top], half, np.nextafter(half, np.float32(np.inf)), np.nextafter(half, np.float32(-np.inf)),
                            np.arange(-127, 128).astype(np.float32) * s])
        rows.append(np.resize(v, 1100).astype(np.float32))
    x = np.stack(rows)
    check_quantize(ctx, mem, dtype, ref.store(dtype, x))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_special_rows(ctx, mem, dtype):
    n = 600
    x = np.ones((9, n), np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 17] = np.nan
    x[3, 599] = np.inf
    x[4, 0] = -np.inf
    x[5] = 2.0 ** -133 * np.arange(n)  # the scale at its floor, subnormal values
    x[6] = 3e38
    x[6, 3] = -3e38
    x[7] = 2.0 ** -126 * np.arange(n)
    check_quantize(ctx, mem, dtype, ref.store(dtype, x))


def product(ctx, mem, a, b, sa, sb, dtype, shift=0):
    m, k = a.shape
    n = b.shape[0]
    c = mem.out(storage(dtype), m * n, shift)
    ctx.contract_i8(mem.put(a, shift), mem.put(b, shift), mem.put(sa), mem.put(sb), m, n, k, CODE[dtype], c)
    ctx.synchronize()
    return mem.get(c, storage(dtype), (m, n))


def check_product(ctx, mem, m, n, k, dtype, shift=0, codes=None):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a = rng.integers(-128, 128, (m, k)).astype(np.int8) if codes is None else np.full((m, k), codes, np.int8)
    b = rng.integers(-128, 128, (n, k)).astype(np.int8) if codes is None else np.full((n, k), codes, np.int8)
    sa, sb = rng.uniform(1e-3, 1, m).astype(np.float32), rng.uniform(1e-3, 1, n).astype(np.float32)
    got = product(ctx, mem, a, b, sa, sb, dtype, shift)
    want = ref.contract_i8(a, b, sa, sb)
    if dtype == "bf16":
        want = oracle.bf16_narrow(want).reshape(want.shape)
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 1000, 4096), (3, 5, 7), (16, 128, 256), (17, 100, 128), (33, 64, 1000),
          (64, 512, 4096), (65, 200, 512), (128, 128, 128), (129, 257, 144), (200, 96, 2048), (256, 256, 640),
          (300, 513, 1111), (511, 264, 784), (1024, 1024, 1024), (257, 5001, 1111),
          (4100, 4104, 208)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ctx, mem, dtype, m, n, k):
    check_product(ctx, mem, m, n, k, dtype)


# Every form of the product, shallower and deeper than the slices it keeps in LDS
FORMS = [("few1x1", 3, 24, 1040), ("few2x1", 17, 2056, 1040), ("few2x2", 17, 4104, 1040), ("few4x2", 33, 4104, 1040),
         ("few4x4", 33, 8200, 2064), ("t64_d", 33, 8200, 528), ("t64_d", 3, 20008, 1040), ("t96_d", 130, 12008, 2064),
         ("t96", 3, 8200, 80), ("t96", 130, 12008, 1040), ("t128", 301, 8200, 16), ("t128", 200, 12008, 1040),
         ("t192", 520, 14344, 16), ("t192", 400, 20008, 1040), ("t256", 1000, 12008, 16), ("t256", 1500, 8200, 1040),
         ("g64", 70, 200, 333), ("g128", 600, 9000, 65)]


@pytest.mark.parametrize("form,m,n,k", FORMS)
def test_product_forms(ctx, mem, form, m, n, k):
    for dtype in ("bf16", "f32"):
        rz = realize(L.PROGRAM_CONTRACTION_I8, (m, n, k), dtype=CODE[dtype], permissions=L.PERMITS_REASSOCIATION,
                     flags=L.REGION_ALIGNED16)
        assert rz.symbols == [f"tiler_contract_i8_{dtype}_{form}"]
        check_product(ctx, mem, m, n, k, dtype)


@pytest.mark.parametrize("m,n,k", [(16, 128, 256), (100, 96, 512), (300, 264, 1024)])
@pytest.mark.parametrize("shift", [1, 4, 8])
def test_product_unaligned(ctx, mem, m, n, k, shift):
    for dtype in ("bf16", "f32"):
        check_product(ctx, mem, m, n, k, dtype, shift)


@pytest.mark.parametrize("m", [1, 70])
def test_the_longest_sum(ctx, mem, m):
    """131071 products of -128 with itself: the largest sum 32 bits hold."""
    check_product(ctx, mem, m, 40, 131071, "f32", codes=-128)
    check_product(ctx, mem, m, 40, 131056, "f32", codes=-128)


def test_scales_that_are_not_finite(ctx, mem):
    """A NaN scale (a poisoned row) gives a NaN row; an infinite one follows
    the products."""
    a, b = np.ones((4, 32), np.int8), np.ones((3, 32), np.int8)
    a[2] = 0
    sa = np.array([1.0, np.nan, np.inf, np.inf], np.float32)
    sb = np.array([1.0, 2.0, 0.0], np.float32)
    for dtype in ("f32", "bf16"):
        got = ref.wide(dtype, product(ctx, mem, a, b, sa, sb, dtype))
        want = ref.contract_i8(a, b, sa, sb)
        assert np.array_equal(got, want.astype(np.float64), equal_nan=True)


def test_linear_layer(ctx, mem):
    """Quantized rows into the product, on the device throughout."""
    rng = np.random.default_rng(8)
    m, n, k = 37, 300, 500
    x, w = ref.store("bf16", rng.standard_normal((m, k))), rng.standard_normal((n, k)).astype(np.float32)
    q, s, wq, ws = mem.out(np.int8, m * k), mem.out(np.float32, m), mem.out(np.int8, n * k), mem.out(np.float32, n)
    c = mem.out(np.float32, m * n)
    ctx.quantize_rows_i8(L.F32, mem.put(w), n, k, wq, ws)
    ctx.quantize_rows_i8(L.BF16, mem.put(x), m, k, q, s)
    ctx.contract_i8(q, wq, s, ws, m, n, k, L.F32, c)
    ctx.synchronize()
    (eq, es), (ewq, ews) = ref.quantize_rows(ref.wide("bf16", x)), ref.quantize_rows(w)
    got = mem.get(c, np.float32, (m, n))
    assert np.array_equal(got, ref.contract_i8(eq, ewq, es, ews))
    # each code is within half a scale of its value: the sum's error is at most that of its terms
    xf, wf = ref.wide("bf16", x), w.astype(np.float64)
    bound = (0.5 * es[:, None] * np.abs(wf).sum(-1)[None, :] + 0.5 * ews[None, :] * np.abs(xf).sum(-1)[:, None]
             + 0.25 * k * es[:, None] * ews[None, :])
    assert (np.abs(got - xf @ wf.T) <= bound * 1.0001).all()
