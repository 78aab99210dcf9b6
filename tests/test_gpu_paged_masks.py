"""A key that a token does not see has no part in its result, however large its value: weights of masked keys are exactly 0.

The values of the masked rows are 2^126, finite in both cache types; a weight of 2^-126 in place of 0 would add 1 a key where the
results are of the size of 1. Bounds: those of test_gpu_paged.py for the rows that see ordinary values only, in which the
masked rows do not appear."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged import EPS24, IDS, KINDS, BF16, U, Batch, attention64, queries

pytestmark = pytest.mark.gpu

LARGE = 2.0 ** 126


def check_rows(got, want, mag, big, act, cache, longest, keep):
    got = got.double().cpu().view(want.shape)[keep]
    want, mag = want[keep], mag[keep]
    if act == BF16 and cache == BF16:
        tol = mag * (2 * 128 * EPS24 * big + 2 * U) + U * want.abs()
    else:
        tol = mag * (2 * 12 * EPS24 * big + 2.0 ** -22 + (longest / 4 + 64) * EPS24) + (U * want.abs() if act == BF16 else 0)
    assert bool(((got - want).abs() <= tol + 1e-30).all()), float((got - want).abs().max())


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,kv", [(100, 100), (100, 333), (4, 60)], ids=["prompt", "continued", "few"])
def test_values_of_later_rows_do_not_leak(vox, act, cache, hd, n, kv):
    """The last rows of a sequence hold large values: the tokens in front of them do not see them."""
    late = 30 if n > 30 else 2
    bt = Batch([(n, kv)], 2, hd, 16, cache, seed=n)
    p, r = bt.rows(bt.table[0], kv)
    bt.v[p[kv - late:], r[kv - late:]] = LARGE
    q = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=n, max_kv=kv)
    want, mag, big = attention64(bt, q, 4, hd ** -0.5)
    check_rows(got, want, mag, big, act, cache, kv, slice(0, n - late))


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [1, 100])
def test_values_behind_a_window_do_not_leak(vox, act, cache, n):
    """The first rows hold large values: a window hides them from every token."""
    kv, window = 300, 40
    first = kv - n + 1 - window  # the first row that some token sees
    bt = Batch([(n, kv)], 2, 64, 16, cache, seed=n)
    p, r = bt.rows(bt.table[0], kv)
    bt.v[p[:first], r[:first]] = LARGE
    q = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=n, max_kv=kv, window=window)
    want, mag, big = attention64(bt, q, 4, 64 ** -0.5, window)
    check_rows(got, want, mag, big, act, cache, kv, slice(0, n))


@pytest.mark.parametrize("hd", [64, 128])
def test_values_of_later_rows_do_not_leak_in_one_tile_blocks(vox, hd):
    """The same in a batch of so many short prompts that blocks of one row tile take them, behind a prefix and without one."""
    n, late = 60, 20
    for prefix in (0, 70):
        bt = Batch([(n, n)] * 40, 4, hd, 16, BF16, seed=hd, prefix=prefix)
        for b in range(40):
            p, r = bt.rows(bt.table[b], n)
            bt.v[p[n - late:], r[n - late:]] = LARGE
        q = queries(bt, 8, BF16)
        table, kv_len, q_start = bt.dev()
        h = bt.handle(vox)
        kw = dict(q_start=q_start, max_q=n, max_kv=n)
        got = h.attend_prefix(q.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, **kw) if prefix else h.attend(q.cuda(), table, kv_len, **kw)
        want, mag, big = attention64(bt, q, 8, hd ** -0.5)
        keep = [b * n + i for b in range(40) for i in range(n - late)]
        check_rows(got, want, mag, big, BF16, BF16, n + prefix, keep)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,seqs", [(1, 2), (1, 200), (5, 3), (70, 3), (200, 2), (30, 40)])
def test_pages_far_in_front_of_a_window_are_given_away(vox, act, cache, hd, n, seqs):
    """Rows 128 and more in front of the first row that a sequence's tokens see are never read: their page table entries name no
    page, and nothing is reported. (The 127 rows between hold finite values that no token sees.)"""
    window, page = 50, 16
    lens = [(n, n + 600 + 37 * b % 300) for b in range(seqs)]
    bt = Batch(lens, 4, hd, page, cache, seed=n + hd)
    q = queries(bt, 8, act)
    want, mag, big = attention64(bt, q, 8, hd ** -0.5, window)
    kv = bt.handle(vox)
    for b, (_, k) in enumerate(lens):
        gone = max(k - n + 1 - window - 127, 0) // page  # whole pages of such rows
        assert gone > 0
        bt.table[b, :gone] = -1
    table, kv_len, q_start = bt.dev(uniform=True)
    for qs, mq, mkv in ((None, 0, 0), (bt.q_start.cuda(), n, max(k for _, k in lens)), (bt.q_start.cuda(), 0, 0)):
        got = kv.attend(q.cuda(), table, kv_len, q_start=qs, max_q=mq, max_kv=mkv, window=window)
        check_rows(got, want, mag, big, act, cache, 1100, slice(None))
    assert vox.device_error() == 0
