"""Page tables, positions and cache slots of a batch's new tokens, against the
definition in plain loops: whole numbers, all of them equal."""
from __future__ import annotations

import numpy as np
import pytest

from attention_reference import page_slots as expected

pytestmark = pytest.mark.gpu


def run(ctx, kept, fresh, page, free, table, tokens, stream=None):
    kept, fresh, free, table = (np.asarray(a, np.int32) for a in (kept, fresh, free, table))
    n, width = table.shape
    ins = [ctx.to_device(a) for a in (kept, fresh, free, table)]
    outs = [ctx.to_device(np.full(max(c, 1), 12345, np.int32)) for c in (n + 1, n, tokens, tokens, 1)]
    ctx.page_slots(ins[0], ins[1], n, page, ins[2], len(free), ins[3], width, tokens, *outs, stream=stream)
    ctx.synchronize()
    got = [ins[3].download(np.int32, (n, width))] + [b.download(np.int32, (c,)) for b, c in
                                                     zip(outs, (n + 1, n, tokens, tokens, 1))]
    for b in ins + outs:
        b.free()
    return got


def check(ctx, kept, fresh, page, free, table, tokens):
    table = np.asarray(table, np.int32)
    got = run(ctx, kept, fresh, page, free, table, tokens)
    want = expected(kept, fresh, page, list(free), table, tokens)
    for name, a, b in zip(("table", "starts", "lengths", "positions", "slots", "taken"), got, want):
        np.testing.assert_array_equal(a, np.atleast_1d(b) if name == "taken" else b, err_msg=name)


def batch(seed, sequences, most_kept, most_fresh, page, spare=3, short=0):
    rng = np.random.default_rng(seed)
    kept, fresh = rng.integers(0, most_kept + 1, sequences), rng.integers(0, most_fresh + 1, sequences)
    have, need = -(-kept // page), -(-(kept + fresh) // page)
    width = int(need.max(initial=0)) + spare
    pool = rng.permutation(int(have.sum() + need.sum()) + 10)
    table = np.full((sequences, width), -7, np.int64)
    at = 0
    for s in range(sequences):
        table[s, :have[s]] = pool[at:at + have[s]]
        at += have[s]
    taken = int((need - have).sum())
    return kept, fresh, pool[at:at + max(taken - short, 0)], table, int(fresh.sum())


@pytest.mark.parametrize("page", [1, 3, 16, 64, 1000])
@pytest.mark.parametrize("sequences,most_kept,most_fresh", [(1, 0, 1), (1, 500, 700), (5, 40, 1), (64, 300, 1), (33, 70, 130)])
def test_batches(ctx, sequences, most_kept, most_fresh, page):
    kept, fresh, free, table, tokens = batch(sequences + page, sequences, most_kept, most_fresh, page)
    check(ctx, kept, fresh, page, free, table, tokens)
    check(ctx, kept, fresh, page, free, table, tokens + 17)  # rows that pad the batch


@pytest.mark.parametrize("sequences", [1023, 1024, 1025, 2600])
def test_more_sequences_than_a_workgroup_sums_at_once(ctx, sequences):
    kept, fresh, free, table, tokens = batch(sequences, sequences, 50, 3, 8)
    check(ctx, kept, fresh, 8, free, table, tokens + 1100)


def test_more_tokens_than_a_workgroup_places(ctx):
    kept, fresh, free, table, tokens = batch(5, 40, 100, 900, 24)
    assert tokens > 4096
    check(ctx, kept, fresh, 24, free, table, tokens)


def test_sequences_without_new_tokens_and_below_zero(ctx):
    table = np.arange(4 * 6).reshape(4, 6)
    check(ctx, [5, 0, 9, 3], [0, 0, 0, 0], 4, [50, 51], table, 3)
    check(ctx, [-5, 4, -1, 3], [2, -7, 1, -1], 4, [50, 51, 52], table, 5)


def test_a_short_list_and_a_narrow_table(ctx):
    for short in (1, 4, 1000):
        kept, fresh, free, table, tokens = batch(short, 9, 30, 25, 4, short=short)
        check(ctx, kept, fresh, 4, free, table, tokens)
    kept, fresh, free, table, tokens = batch(8, 9, 30, 25, 4)
    check(ctx, kept, fresh, 4, free, table[:, :3], tokens)  # tokens beyond the table's width
    check(ctx, kept, fresh, 4, free, table[:, :1], tokens)


def test_fewer_rows_than_new_tokens(ctx):
    kept, fresh, free, table, tokens = batch(11, 7, 30, 25, 4)
    check(ctx, kept, fresh, 4, free, table, tokens // 2)


def test_far_lengths(ctx):
    """Positions next to 2^31, and sums past it."""
    check(ctx, [2 ** 31 - 5, 3], [3, 2], 64, [7], [[1, 2], [3, 4]], 5)
    check(ctx, [2 ** 31 - 5, 2 ** 31 - 1], [9, 1], 1 << 30, [9, 8], [[1, 1], [0, 1]], 10)
    got = run(ctx, [0, 0, 5], [2 ** 31 - 1, 2 ** 31 - 1, 2], 16, [4], [[0], [0], [6]], 4)
    np.testing.assert_array_equal(got[1], [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1])
    np.testing.assert_array_equal(got[3], [0, 1, 2, 3])


def test_no_sequences(ctx):
    got = run(ctx, [], [], 16, [], np.zeros((0, 4)), 3)
    assert got[1].tolist() == [0] and got[3].tolist() == [0, 0, 0] and got[4].tolist() == [-1] * 3 and got[5].tolist() == [0]
