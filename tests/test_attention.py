"""The attention sublayer without a GPU: what the workspace queries refuse and
answer, the structs' layout, and the oracle against a second way to the same
results."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import attention_reference as ref
import test_abi_layout
from tiler_amd import _lib as L
from tiler_amd import families
from tiler_amd.realize import propose, realize
from tiler_amd.runtime import Refusal


def test_struct_layouts(tmp_path, monkeypatch):
    monkeypatch.setattr(test_abi_layout, "STRUCTS", {
        L.PagedCache: "tiler_hip_paged_cache",
        L.HeadLayout: "tiler_hip_head_layout",
        L.AttentionShape: "tiler_hip_attention_shape",
    })
    checks = [f for name, f in vars(test_abi_layout).items() if name.startswith("test_")]
    assert checks
    for f in checks:
        f(*(tmp_path for _ in range(f.__code__.co_argcount)))


def cache(**kw):
    a = dict(k=16, v=16, pages=10, page=16, heads=2, head_dim=64, page_stride=16 * 128, token_stride=128, head_stride=64)
    a.update(kw)
    return L.PagedCache(**a)


def shape(**kw):
    a = dict(tokens=4, sequences=4, q_heads=8, scale=0.125, q_stride=512, out_stride=512, table_width=5)
    a.update(kw)
    return L.AttentionShape(**a)


def attention(s, c):
    n = ctypes.c_uint64(1)
    return L.lib().tiler_hip_paged_attention_bf16_workspace(None, ctypes.byref(s), ctypes.byref(c), ctypes.byref(n)), n.value


@pytest.mark.parametrize("s,c,status", [
    (shape(), cache(), L.OK),
    (shape(q_heads=7), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(q_heads=0), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(scale=0.0), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(scale=-1.0), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(scale=float("nan")), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(scale=float("inf")), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(scale=3e38), cache(), L.REFUSE_INVALID_ARGUMENT),  # not finite in steps of log2
    (shape(q_stride=511), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(out_stride=511), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(q_stride=0, out_stride=0, tokens=1), cache(), L.OK),  # one token has no next one
    (shape(reserved=1), cache(), L.REFUSE_INVALID_ARGUMENT),
    (shape(tokens=1 << 29), cache(), L.REFUSE_CAPACITY),  # 2^32 rows
    (shape(table_width=1 << 27), cache(), L.REFUSE_CAPACITY),  # 2^31 positions
    (shape(sequences=1 << 31), cache(), L.REFUSE_CAPACITY),
    (shape(sequences=0), cache(), L.OK),
    (shape(table_width=0), cache(), L.OK),
    (shape(), cache(pages=0), L.OK),
    (shape(), cache(page=0), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(heads=0), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(head_dim=0), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(reserved=1), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(head_dim=60), L.REFUSE_UNSUPPORTED),
    (shape(q_stride=4096, out_stride=4096), cache(head_dim=264, page_stride=16 * 528, token_stride=528, head_stride=264),
     L.REFUSE_UNSUPPORTED),
    (shape(), cache(token_stride=129, page_stride=16 * 130), L.REFUSE_UNSUPPORTED),  # rows off 16 bytes
    (shape(), cache(page_stride=16 * 128 - 8), L.REFUSE_INVALID_ARGUMENT),  # rows overlap
    (shape(), cache(token_stride=120), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(head_stride=56), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(token_stride=64, head_stride=16 * 64), L.OK),  # [pages, heads, page, dim]
    (shape(), cache(token_stride=64, page_stride=16 * 64, head_stride=10 * 16 * 64), L.OK),  # heads outermost
    (shape(), cache(token_stride=64, page_stride=16 * 64, head_stride=9 * 16 * 64), L.REFUSE_INVALID_ARGUMENT),
    (shape(), cache(page=1, token_stride=0, page_stride=128), L.OK),  # one token has no next one
    (shape(q_heads=8), cache(heads=1, head_stride=0), L.OK),
    (shape(), cache(pages=1 << 27), L.REFUSE_CAPACITY),  # 2^31 slots
    (shape(), cache(page_stride=1 << 58), L.REFUSE_CAPACITY),
    (shape(), cache(page_stride=(1 << 64) - 8), L.REFUSE_CAPACITY),
])
def test_attention_requests(s, c, status):
    assert attention(s, c)[0] == status


def test_attention_workspace():
    # enough sequences for the CUs: no parts to join
    assert attention(shape(tokens=1000, sequences=1000), cache()) == (L.OK, 0)
    # few long contexts: parts of the keys
    status, n = attention(shape(tokens=1, sequences=1, table_width=1000, max_length=16000), cache())
    assert status == L.OK and n > 0
    # an unknown length is the table's
    assert attention(shape(tokens=1, sequences=1, table_width=1000), cache()) == (L.OK, n)
    assert attention(shape(tokens=1, sequences=1, table_width=1000, max_length=100), cache()) == (L.OK, 0)
    assert attention(shape(tokens=1, sequences=1, table_width=1000, window=100, sinks=4), cache()) == (L.OK, 0)
    s, c = shape(), cache()
    query = L.lib().tiler_hip_paged_attention_bf16_workspace
    assert query(None, None, ctypes.byref(c), ctypes.byref(ctypes.c_uint64())) == L.REFUSE_INVALID_ARGUMENT
    assert query(None, ctypes.byref(s), None, ctypes.byref(ctypes.c_uint64())) == L.REFUSE_INVALID_ARGUMENT
    assert query(None, ctypes.byref(s), ctypes.byref(c), None) == L.REFUSE_INVALID_ARGUMENT


def heads(**kw):
    a = dict(tokens=4, q_heads=8, kv_heads=2, head_dim=64, rotary=64, pairing=L.ROTATE_HALVES, eps_bits=0x358637BD,
             q_stride=512, k_stride=128, v_stride=128, q_out_stride=512, k_out_stride=128)
    a.update(kw)
    return L.HeadLayout(**a)


@pytest.mark.parametrize("h,dtype,status", [
    (heads(), L.BF16, L.OK),
    (heads(), L.F32, L.OK),
    (heads(), 2, L.REFUSE_UNSUPPORTED),
    (heads(head_dim=0), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(rotary=63), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(rotary=66), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(rotary=0), L.BF16, L.OK),
    (heads(pairing=2), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(eps_bits=0x7F800000), L.BF16, L.REFUSE_INVALID_ARGUMENT),  # infinity
    (heads(eps_bits=0x7FC00000), L.BF16, L.REFUSE_INVALID_ARGUMENT),  # a NaN
    (heads(eps_bits=0x80000000), L.BF16, L.REFUSE_INVALID_ARGUMENT),  # -0
    (heads(eps_bits=0xB58637BD), L.BF16, L.REFUSE_INVALID_ARGUMENT),  # below zero
    (heads(eps_bits=0), L.BF16, L.OK),
    (heads(reserved=1), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(q_stride=511), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(k_stride=127), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(q_out_stride=511), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(k_out_stride=127), L.BF16, L.REFUSE_INVALID_ARGUMENT),
    (heads(tokens=1, q_stride=0, k_stride=0, q_out_stride=0, k_out_stride=0), L.BF16, L.OK),
    (heads(q_heads=0, kv_heads=0), L.BF16, L.OK),
    (heads(head_dim=1026, rotary=2, q_stride=1 << 14, q_out_stride=1 << 14, k_stride=1 << 14, k_out_stride=1 << 14), L.BF16,
     L.REFUSE_CAPACITY),
    (heads(tokens=1 << 41), L.BF16, L.REFUSE_CAPACITY),
    (heads(q_stride=1 << 41), L.BF16, L.REFUSE_CAPACITY),
    (heads(q_heads=1 << 21, q_stride=1 << 30, q_out_stride=1 << 30), L.BF16, L.REFUSE_CAPACITY),
])
def test_head_requests(h, dtype, status):
    n = ctypes.c_uint64(1)
    got = L.lib().tiler_hip_norm_rotate_backward_workspace(None, dtype, ctypes.byref(h), ctypes.byref(n))
    assert got == status
    if status == L.OK:  # partial sums of the weights' gradients, where there is a norm
        assert (n.value > 0) == bool(h.eps_bits and (h.q_heads or h.kv_heads))


def test_head_query_arguments():
    query, h = L.lib().tiler_hip_norm_rotate_backward_workspace, heads()
    assert query(None, L.BF16, None, ctypes.byref(ctypes.c_uint64())) == L.REFUSE_INVALID_ARGUMENT
    assert query(None, L.BF16, ctypes.byref(h), None) == L.REFUSE_INVALID_ARGUMENT


# -- the oracle -------------------------------------------------------------------
def test_oracle_of_the_rotation_by_complex_numbers():
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((5, 3, 12)), rng.standard_normal(12)
    positions, frequencies = rng.integers(0, 100, 5), rng.uniform(0, 1, 4)
    for pairing in ("halves", "neighbours"):
        y, _ = ref.norm_rotate(x, w, positions, frequencies, 8, pairing, 1e-3)
        u = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-3) * w
        z = u[..., :4] + 1j * u[..., 4:8] if pairing == "halves" else u[..., 0:8:2] + 1j * u[..., 1:8:2]
        z = z * np.exp(1j * positions[:, None] * frequencies)[:, None, :]
        if pairing == "halves":
            np.testing.assert_allclose(y[..., :8], np.concatenate([z.real, z.imag], -1), rtol=1e-12)
        else:
            np.testing.assert_allclose(y[..., :8], np.stack([z.real, z.imag], -1).reshape(5, 3, 8), rtol=1e-12)
        np.testing.assert_allclose(y[..., 8:], u[..., 8:], rtol=1e-12)


@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("eps", [1e-3, None])
def test_oracle_of_the_gradients_by_differences(pairing, eps):
    rng = np.random.default_rng(1)
    x, w, dy = rng.standard_normal((2, 2, 10)), rng.standard_normal(10), rng.standard_normal((2, 2, 10))
    positions, frequencies = rng.integers(0, 100, 2), rng.uniform(0, 1, 3)

    def loss(x, w):
        return (ref.norm_rotate(x, w, positions, frequencies, 6, pairing, eps)[0] * dy).sum()

    dx, dw, _, _ = ref.norm_rotate_backward(dy, x, w, positions, frequencies, 6, pairing, eps)
    step = 1e-5
    for index in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[index] = step
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * step) - dx[index]) < 1e-8
    if eps is not None:
        for i in range(10):
            d = np.zeros(10)
            d[i] = step
            assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * step) - dw[i]) < 1e-8


def test_oracle_of_attention_by_a_dense_mask():
    rng = np.random.default_rng(2)
    k, v, q = (rng.standard_normal(s) for s in ((6, 4, 2, 8), (6, 4, 2, 8), (5, 6, 8)))
    table = np.array([[4, 1, 0, -1], [3, 5, 2, -1]])
    starts, lengths = [0, 3, 5], [11, 9]
    for window, sinks in ((0, 0), (4, 2), (1, 0), (100, 5)):
        out, _ = ref.paged_attention(q, k, v, table, starts, lengths, 0.3, window, sinks, np.zeros((5, 6, 8)))
        for s in range(2):
            keys, vals = k[table[s, :3]].reshape(12, 2, 8), v[table[s, :3]].reshape(12, 2, 8)
            n = starts[s + 1] - starts[s]
            p = np.arange(lengths[s] - n, lengths[s])[:, None]
            j = np.arange(12)
            mask = (j <= p) & ((j > p - window) | (j < sinks) if window else True)
            for h in range(6):
                logits = np.where(mask, 0.3 * q[starts[s]:starts[s + 1], h] @ keys[:, h // 3].T, -np.inf)
                e = np.exp(logits)
                np.testing.assert_allclose(out[starts[s]:starts[s + 1], h], e @ vals[:, h // 3] / e.sum(-1, keepdims=True),
                                           rtol=1e-12)


def test_oracle_of_page_slots_on_a_batch_written_out():
    table, starts, lengths, positions, slots, taken = ref.page_slots([5, 0, 8], [2, 0, 5], 4, [7, 9], [[1, 2, -1], [-1] * 3,
                                                                                                     [3, 4, -1]], 8)
    assert table.tolist() == [[1, 2, -1], [-1, -1, -1], [3, 4, 7]]
    assert starts.tolist() == [0, 2, 2, 7] and lengths.tolist() == [7, 0, 13]
    assert positions.tolist() == [5, 6, 8, 9, 10, 11, 12, 0]
    assert slots.tolist() == [9, 10, 28, 29, 30, 31, -1, -1]  # position 12 lies past the table's width
    assert taken == 1


# -- the recognizer ---------------------------------------------------------------
RE = L.PERMITS_REASSOCIATION
EPS = 0x358637BD


def bits(x):
    return int(np.float32(x).view(np.uint32))


def rotate_region(backward=False, extents=(5, 8, 2, 64, 64), variant=0, dtype=L.BF16, pairing=0, eps=EPS, **kw):
    q, k = extents[1] * extents[3], extents[2] * extents[3]
    kw = {"permissions": RE, "strides": (q, k, q, k), "grouping": (pairing,), "scalars": (eps,), **kw}
    return realize(L.PROGRAM_NORM_ROTATE_BACKWARD if backward else L.PROGRAM_NORM_ROTATE, extents, dtype=dtype,
                   variant=variant, **kw)


def attention_region(tokens=4, sequences=4, width=5, pages=10, page=16, kv_heads=2, heads=8, dim=64, window=0, sinks=0,
                     fresh=0, scale=0.125, **kw):
    row = kv_heads * dim
    kw = {"permissions": RE, "dtype": L.BF16, "strides": (heads * dim, heads * dim, page * row, row, dim), **kw}
    return realize(L.PROGRAM_PAGED_ATTENTION, (tokens, sequences, width, pages, page, kv_heads, heads, dim),
                   grouping=(window, sinks, fresh), scalars=(bits(scale),), **kw)


def counted(rz):
    roles = [role for role, _ in rz.slots]
    return tuple(roles.count(r) for r in (L.SLOT_INPUT, L.SLOT_OUTPUT, L.SLOT_SCRATCH))


ALL_GRADS = L.ROTATE_DQ | L.ROTATE_DK | L.ROTATE_DWQ | L.ROTATE_DWK


@pytest.mark.parametrize("rz,counts", [
    (lambda: rotate_region(variant=L.ROTATE_K_OUT), (4, 2, 0)),
    (lambda: rotate_region(variant=L.ROTATE_WQ | L.ROTATE_WK | L.ROTATE_K_OUT), (6, 2, 0)),
    (lambda: rotate_region(extents=(5, 8, 0, 64, 0)), (1, 1, 0)),
    (lambda: rotate_region(True, variant=L.ROTATE_WQ | L.ROTATE_WK | ALL_GRADS), (8, 4, 2)),
    (lambda: rotate_region(True, variant=L.ROTATE_DQ, eps=0), (3, 1, 0)),
    (lambda: rotate_region(True, variant=L.ROTATE_DK | L.ROTATE_DWK), (4, 2, 1)),
    (lambda: attention_region(), (6, 1, 0)),
    (lambda: attention_region(width=1000, tokens=1, sequences=1), (6, 1, 2)),
    (lambda: attention_region(width=0), (5, 1, 0)),
])
def test_slots(rz, counts):
    rz = rz()
    assert counted(rz) == counts and rz.symbols
    for i, (role, _) in enumerate(rz.slots):
        assert rz.slot_alignment(i) == 16


@pytest.mark.parametrize("rz,status", [
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, permissions=0), L.REFUSE_UNSUPPORTED),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, dtype=2), L.REFUSE_UNSUPPORTED),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, input_subnormals=L.SUBNORMALS_FLUSH_SIGN), L.REFUSE_UNSUPPORTED),
    (lambda: rotate_region(variant=0), L.REFUSE_INVALID_ARGUMENT),  # the keys go nowhere
    (lambda: rotate_region(variant=L.ROTATE_K_OUT | L.ROTATE_DQ), L.REFUSE_INVALID_ARGUMENT),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT | L.ROTATE_WQ, eps=0), L.REFUSE_INVALID_ARGUMENT),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, pairing=2), L.REFUSE_INVALID_ARGUMENT),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, pairing=1 << 32), L.REFUSE_CAPACITY),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, extents=(5, (1 << 32) + 8, 2, 64, 64)), L.REFUSE_CAPACITY),
    (lambda: rotate_region(True, variant=L.ROTATE_K_OUT), L.REFUSE_INVALID_ARGUMENT),
    (lambda: rotate_region(True, variant=L.ROTATE_DWQ, eps=0), L.REFUSE_INVALID_ARGUMENT),
    (lambda: rotate_region(True, variant=L.ROTATE_DQ, permissions=0), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(permissions=0), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(dtype=L.F32), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(form=L.FORM_CONTRACT_SKINNY), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(form=10), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(dim=136, form=L.FORM_ATTENTION_TILE_256), L.REFUSE_UNSUPPORTED),
    (lambda: rotate_region(variant=L.ROTATE_K_OUT, form=L.FORM_ATTENTION_FEW), L.REFUSE_UNSUPPORTED),
    (lambda: attention_region(variant=1), L.REFUSE_INVALID_ARGUMENT),
    (lambda: attention_region(window=1 << 32), L.REFUSE_CAPACITY),
    (lambda: attention_region(page=1 << 32), L.REFUSE_CAPACITY),
    (lambda: attention_region(scale=0.0), L.REFUSE_INVALID_ARGUMENT),
    (lambda: attention_region(heads=7), L.REFUSE_INVALID_ARGUMENT),
    (lambda: attention_region(flags=0), L.REFUSE_UNSUPPORTED),  # the cache's rows start on 16 bytes
    (lambda: attention_region(strides=(512, 512, 1 << 33, 128, 64)), L.REFUSE_CAPACITY),
    (lambda: attention_region(pages=1, strides=(512, 512, 1 << 33, 128, 64)), None),  # one page has no next one
    (lambda: attention_region(pages=1, strides=(512, 512, 7, 128, 64)), None),
    (lambda: attention_region(kv_heads=1, strides=(512, 512, 1024, 64, 3)), None),
    (lambda: attention_region(page=1, strides=(512, 512, 128, 5, 64)), None),
    (lambda: attention_region(pages=1, page=1 << 26, width=1, strides=(512, 512, 0, 128, 64)), L.REFUSE_CAPACITY),
])
def test_refused_regions(rz, status):
    if status is None:
        assert rz().symbols
        return
    with pytest.raises(Refusal) as e:
        rz()
    assert e.value.status == status, str(e.value)


def test_proposals():
    for rz, program, kw in ((rotate_region(variant=L.ROTATE_K_OUT), L.PROGRAM_NORM_ROTATE,
                             dict(extents=(5, 8, 2, 64, 64), variant=L.ROTATE_K_OUT, strides=(512, 128, 512, 128),
                                  scalars=(EPS,), dtype=L.BF16)),
                            (attention_region(), L.PROGRAM_PAGED_ATTENTION,
                             dict(extents=(4, 4, 5, 10, 16, 2, 8, 64), strides=(512, 512, 16 * 128, 128, 64),
                                  scalars=(bits(0.125),), dtype=L.BF16))):
        offer = propose(program, permissions=RE, **kw)
        assert offer.proposals[offer.chosen].symbols == rz.symbols
        strict = propose(program, **kw)
        assert not strict.proposals and strict.declined


@pytest.mark.parametrize("kw,symbol", [
    (dict(dim=64, eps=EPS), "tiler_norm_rotate_bf16_h4"), (dict(dim=128, pairing=1), "tiler_norm_rotate_bf16_n8"),
    (dict(dim=256), "tiler_norm_rotate_bf16_h16"), (dict(dim=512), "tiler_norm_rotate_bf16_h32"),
    (dict(dim=1024), "tiler_norm_rotate_bf16_h64"), (dict(dim=90, rotary=34), "tiler_norm_rotate_bf16_any"),
    (dict(dim=128, dtype=L.F32), "tiler_norm_rotate_f32_h16"), (dict(dim=1024, dtype=L.F32), "tiler_norm_rotate_f32_any"),
    (dict(dim=64, rotary=24), "tiler_norm_rotate_bf16_any")])
def test_rotation_forms(kw, symbol):
    kw = dict(kw)
    dim = kw.pop("dim")
    rotary = kw.pop("rotary", dim)
    assert rotate_region(extents=(5, 8, 2, dim, rotary), variant=L.ROTATE_K_OUT, **kw).symbols == [symbol]


@pytest.mark.parametrize("kw,symbols", [
    (dict(tokens=4, fresh=1), ["few64"]),
    (dict(tokens=4, fresh=1, dim=72), ["few128"]),
    (dict(tokens=4, fresh=1, dim=136), ["few256"]),
    (dict(tokens=1, sequences=1, width=1000), ["few64", "join"]),
    (dict(tokens=40, sequences=1), ["t128_d64"]),
    (dict(tokens=40, sequences=1, dim=72), ["t128_d96"]),
    (dict(tokens=40, sequences=1, dim=104), ["t128_d128"]),
    (dict(tokens=40, sequences=1, dim=136), ["t128_d192"]),
    (dict(tokens=40, sequences=1, dim=200), ["t128_d256"]),
    (dict(tokens=40, sequences=1, width=1000), ["t128_d64", "join"]),
    (dict(tokens=1 << 14, sequences=1, width=1 << 10), ["t256_d64"]),
    (dict(tokens=1 << 14, sequences=1, width=1 << 10, dim=256), ["t128_d256"]),
])
def test_attention_forms(kw, symbols):
    assert attention_region(**kw).symbols == ["tiler_paged_attention_bf16_" + s for s in symbols]


# -- the host functions' checks ------------------------------------------------------
def test_host_functions_refuse():
    q, k = np.zeros((3, 4, 64), np.uint16), np.zeros((3, 2, 64), np.uint16)
    at, f = np.zeros(3, np.int32), np.ones(32)
    cache, table, starts, lengths = (np.zeros((6, 4, 2, 64), np.uint16), np.zeros((2, 3), np.int32), np.zeros(3, np.int32),
                                     np.zeros(2, np.int32))
    for call, status in (
            (lambda: families.page_slots([1], [1, 2], 4, [0], np.zeros((1, 2))), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.page_slots([1], [1], 4, [0], np.zeros((2, 2))), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.norm_rotate(q, k[:, :, :32], None, None, at, f, 64), L.REFUSE_UNSUPPORTED),
            (lambda: families.norm_rotate(q, k.astype(np.float32), None, None, at, f, 64), L.REFUSE_UNSUPPORTED),
            (lambda: families.norm_rotate(q, k, None, None, at, f, 64, "pairs"), L.REFUSE_UNSUPPORTED),
            (lambda: families.norm_rotate(q, k, None, None, at[:2], f, 64), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.norm_rotate(q, k, None, None, at, f[:4], 64), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.norm_rotate(q, k, np.zeros(8, np.uint16), None, at, f, 64), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.norm_rotate_backward(q, q, q, k, None, None, at, f, 64), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.paged_attention_bf16(q[0], cache, cache, table, starts, lengths, 1.0), L.REFUSE_UNSUPPORTED),
            (lambda: families.paged_attention_bf16(q, cache, cache[:5], table, starts, lengths, 1.0), L.REFUSE_INVALID_ARGUMENT),
            (lambda: families.paged_attention_bf16(q, cache, cache, table, starts[:2], lengths, 1.0), L.REFUSE_INVALID_ARGUMENT)):
        with pytest.raises(Refusal) as e:
            call()
        assert e.value.status == status, str(e.value)
