"""The attention sublayer's requests at their ends, without a GPU: what the
workspace queries and the recognizer answer for the largest, the widest and the
unusual."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from test_attention import ALL_GRADS, RE, attention, bits, cache, rotate_region, shape
from tiler_amd import _lib as L
from tiler_amd import families
from tiler_amd.realize import propose, realize
from tiler_amd.runtime import Refusal

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def need(tokens, sequences, heads, kv_heads, dim, **kw):
    row = kv_heads * dim
    status, n = attention(shape(tokens=tokens, sequences=sequences, q_heads=heads, q_stride=heads * dim, out_stride=heads * dim,
                                table_width=64, **kw),
                          cache(page=1024, heads=kv_heads, head_dim=dim, page_stride=1024 * row, token_stride=row, head_stride=dim))
    assert status == L.OK
    return n


def most(tokens, heads, dim):
    """Bytes that parts may take: eight of every row or 256 MB, or two rounds of workgroups
    (512 of 128 rows, 256 from heads of more than 128 on) of the tiles behind whole ones."""
    part = 4 * dim + 8  # results, maximum and sum in binary32
    return max(8 * tokens * heads * part, 256 << 20, 2 * 512 * 128 * part) + 512


@pytest.mark.parametrize("tokens,sequences,heads,kv_heads,dim,window,fresh", [
    (814, 128, 32, 8, 256, 32768, 7), (6629, 256, 8, 8, 128, 16384, 0), (814, 128, 32, 8, 256, 32768, 0),
    (30000, 1000, 16, 8, 64, 32768, 0), (3000, 1000, 8, 8, 128, 4096, 0)])
def test_workspace_of_many_windowed_sequences(tokens, sequences, heads, kv_heads, dim, window, fresh):
    assert need(tokens, sequences, heads, kv_heads, dim, window=window, max_fresh=fresh) <= most(tokens, heads, dim)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (8, 8, 128), (32, 8, 256), (16, 1, 64), (64, 8, 64), (40, 1, 8)])
def test_workspace_is_bounded(heads, kv_heads, dim):
    for sequences in (1, 2, 7, 24, 128, 256, 1000):
        for each in (1, 3, 7, 30, 100, 512, 2048):
            for tokens in {sequences * each, sequences * each * 3 // 5 + 1, sequences * each * 9}:
                if tokens > 40000:
                    continue
                for window in (0, 300, 4096, 32768):
                    for longest in (500, 8000, 65536):
                        for fresh in (min(each, tokens), 0):
                            n = need(tokens, sequences, heads, kv_heads, dim, window=window, max_fresh=fresh, max_length=longest)
                            assert n <= most(tokens, heads, dim), (tokens, sequences, window, longest, fresh)


def test_every_rotation_kernel_is_tested():
    """The heads that the GPU tests run reach each kernel that a request can be sent to."""
    from test_gpu_attention_ends import WIDE_FORMS
    from test_gpu_norm_rotate import FORMS

    reached = set()
    for heads, kv_heads, dim, rotary in FORMS + WIDE_FORMS:
        for dtype in (L.BF16, L.F32):
            for pairing in (L.ROTATE_HALVES, L.ROTATE_NEIGHBOURS):
                kw = dict(extents=(5, heads, kv_heads, dim, rotary), dtype=dtype, pairing=pairing)
                reached.update(rotate_region(variant=L.ROTATE_K_OUT, **kw).symbols)
                reached.update(rotate_region(True, variant=ALL_GRADS, **kw).symbols)
    info, registered, i = L.EntryInfo(), set(), 0
    while L.lib().tiler_hip_payload_entry(i, ctypes.byref(info)) == L.OK:
        registered.add(info.symbol.decode())
        i += 1
    assert reached == {s for s in registered if s.startswith("tiler_norm_rotate")}


@pytest.mark.parametrize("pairing", [L.ROTATE_HALVES, L.ROTATE_NEIGHBOURS])
@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
def test_rotation_without_a_norm_under_the_strict_contract(dtype, pairing):
    """Without a norm nothing is summed: no order to permit."""
    kw = dict(dtype=dtype, pairing=pairing, eps=0)
    for backward, variant in ((False, L.ROTATE_K_OUT), (True, L.ROTATE_DQ | L.ROTATE_DK), (True, L.ROTATE_DK)):
        strict = rotate_region(backward, variant=variant, permissions=0, **kw)
        assert strict.symbols and strict.symbols == rotate_region(backward, variant=variant, **kw).symbols
        with pytest.raises(Refusal) as e:
            rotate_region(backward, variant=variant, permissions=0, dtype=dtype, pairing=pairing)
        assert e.value.status == L.REFUSE_UNSUPPORTED
    offer = propose(L.PROGRAM_NORM_ROTATE, (5, 8, 2, 64, 64), dtype=dtype, variant=L.ROTATE_K_OUT, strides=(512, 128, 512, 128),
                    grouping=(pairing,))
    assert len(offer.proposals) == 1 and not offer.declined


def test_a_region_says_its_longest_sequence():
    """The parts of the keys go by the longest sequence, as the direct call's do by
    max_length, not by the table's room."""
    def region(longest):
        return realize(L.PROGRAM_PAGED_ATTENTION, (1, 1, 1000, 10, 16, 2, 8, 64), dtype=L.BF16, permissions=RE,
                       strides=(512, 512, 16 * 128, 128, 64), grouping=(0, 0, 1), scalars=(bits(0.125), longest))

    def direct(longest):
        return attention(shape(tokens=1, sequences=1, table_width=1000, max_fresh=1, max_length=longest), cache())[1]

    for longest in (0, 100, 600, 5000, 15999, 16000, 1 << 31):
        scratch = sum(-(-n // 256) * 256 for role, n in region(longest).slots if role == L.SLOT_SCRATCH)
        assert scratch == direct(longest), longest
    assert len(region(100).symbols) == 1 and len(region(0).symbols) == 2


def test_host_functions_keep_their_numbers():
    """Numbers that do not fit what the call takes are refused, not cut: a window of -1
    would be one of 2^32 - 1, a length of 2^31 one of nothing."""
    q, k = np.zeros((3, 4, 64), np.uint16), np.zeros((3, 2, 64), np.uint16)
    at, f = np.zeros(3, np.int32), np.ones(32)
    pages, table, starts, lengths = (np.zeros((6, 4, 2, 64), np.uint16), np.zeros((2, 3), np.int32), np.zeros(3, np.int32),
                                     np.zeros(2, np.int32))
    wide, none = np.array([1 << 31]), np.zeros((1, 2), np.int32)
    for call in (
            lambda: families.paged_attention_bf16(q, pages, pages, table, starts, lengths, 1.0, window=-1),
            lambda: families.paged_attention_bf16(q, pages, pages, table, starts, lengths, 1.0, window=1 << 32),
            lambda: families.paged_attention_bf16(q, pages, pages, table, starts, lengths, 1.0, window=4, sinks=-1),
            lambda: families.paged_attention_bf16(q, pages, pages, table + 0.5, starts, lengths, 1.0),
            lambda: families.paged_attention_bf16(q, pages, pages, table.astype(np.int64) + (1 << 32), starts, lengths, 1.0),
            lambda: families.page_slots(wide, [1], 4, [0], none),
            lambda: families.page_slots([1], wide, 4, [0], none),
            lambda: families.page_slots([1.5], [1], 4, [0], none),
            lambda: families.page_slots([float("nan")], [1], 4, [0], none),
            lambda: families.page_slots([1], [1], 4, wide, none),
            lambda: families.page_slots([1], [1], 4, [0], none.astype(np.int64) + (1 << 33)),
            lambda: families.page_slots([1], [1], 4, ["a"], none),
            lambda: families.page_slots([1], [1], -4, [0], none),
            lambda: families.page_slots([1], [1], 4, [0], none, tokens=-1),
            lambda: families.norm_rotate(q, k, None, None, at, f, 64, eps_bits=1 << 32),
            lambda: families.norm_rotate(q, k, None, None, at, f, -64)):
        with pytest.raises(Refusal) as e:
            call()
        assert e.value.status == L.REFUSE_INVALID_ARGUMENT, str(e.value)


def test_gradients_of_one_side_ask_nothing_of_the_other():
    """Without dk and dwk (dq and dwq) the strides of the keys (queries) do not matter."""
    for norm in (0x358637BD, 0):
        for variant, strides in ((L.ROTATE_DQ, (512, 0, 512, 0)), (L.ROTATE_DK, (0, 128, 0, 128))):
            assert rotate_region(True, variant=variant, strides=strides, eps=norm).symbols
            for i in (0, 1, 2, 3):
                if strides[i]:
                    cut = tuple(s - (n == i) for n, s in enumerate(strides))
                    with pytest.raises(Refusal) as e:
                        rotate_region(True, variant=variant, strides=cut, eps=norm)
                    assert e.value.status == L.REFUSE_INVALID_ARGUMENT
    for variant in (L.ROTATE_DQ | L.ROTATE_DK, L.ROTATE_DQ | L.ROTATE_DWK):
        for strides in ((511, 128, 512, 128), (512, 127, 512, 128), (512, 128, 511, 128), (512, 128, 512, 127)):
            with pytest.raises(Refusal):
                rotate_region(True, variant=variant, strides=strides)
    for strides in ((511, 128, 512, 128), (512, 127, 512, 128)):
        with pytest.raises(Refusal):
            rotate_region(variant=L.ROTATE_K_OUT, strides=strides)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_planners_are_sanitizer_clean(tmp_path):
    """tests/native/attention_planner_sanitize.cpp: 400000 requests, ordinary and extreme,
    under the address and undefined-behaviour sanitizers; grids, parts, tiles and scratch of
    each plan are what the kernels take them for."""
    exe, runtime = tmp_path / "attention_planner_sanitize", os.path.join(ROOT, "tiler_amd", "csrc", "runtime")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined,float-cast-overflow,float-divide-by-zero",
                    "-fno-sanitize-recover=all", f"-I{os.path.join(ROOT, 'include')}", f"-I{runtime}",
                    os.path.join(ROOT, "tests", "native", "attention_planner_sanitize.cpp"),
                    os.path.join(runtime, "attention.cpp"), os.path.join(runtime, "program.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "attention-planner-sanitize ok" in r.stdout and "runtime error" not in r.stderr


@pytest.mark.parametrize("sequences,kv_heads,keys,parts", [
    (1, 1, 2000, 8), (1, 1, 4000, 16), (1, 1, 8000, 31), (1, 1, 32000, 63), (1, 2, 32000, 63), (1, 1, 60000, 86), (1, 8, 32000, 63),
    (1, 8, 60000, 64), (8, 8, 32000, 8), (16, 8, 1000, 4), (64, 8, 32000, 1)])
def test_parts_of_few_rows(sequences, kv_heads, keys, parts):
    """256 keys to a part at least, sqrt(keys / 8) parts at most, and the CUs' share."""
    for group, dim in ((1, 64), (4, 128), (4, 256)):
        n = need(sequences, sequences, group * kv_heads, kv_heads, dim, max_fresh=1, max_length=keys)
        rows = sequences * group * kv_heads
        up = lambda b: -(-b // 256) * 256
        assert n == (up(4 * dim * rows * parts) + up(8 * rows * parts) if parts > 1 else 0)


def test_more_workgroups_than_a_launch_has():
    for sequences, status in (((1 << 22) - 1, L.OK), (1 << 22, L.REFUSE_CAPACITY), (1 << 23, L.REFUSE_CAPACITY)):
        assert attention(shape(tokens=sequences, sequences=sequences, max_fresh=1), cache())[0] == status
