"""Lengths, offsets and page numbers that are out of range, in every kernel family: none is followed, each is reported by
vox_cuda_device_error(), and the batch's other sequences keep their results. Every value is held inside its range on the device
before it forms an address."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged import IDS, KINDS, Batch, queries

pytestmark = pytest.mark.gpu

HEADS, KVH, HD = 4, 2, 64


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [1, 40])
def test_bad_pages_and_lengths(vox, act, cache, n):
    bt = Batch([(n, 60), (n, 60)], KVH, HD, 16, cache, seed=1, fill=0.0)
    kv = bt.handle(vox)
    table, kv_len, _ = bt.dev()
    q = queries(bt, HEADS, act).cuda()
    good = kv.attend(q, table, kv_len)
    assert vox.device_error() == 0
    second = table[1].tolist()
    width = table.shape[1]
    for t, ln in ((i32([[10 ** 6] * width, second]), kv_len), (i32([[-5] * width, second]), kv_len),
                  (i32([table[0, :3].tolist() + [2 ** 31 - 1] * (width - 3), second]), kv_len),  # the last page alone
                  (table, i32([-3, 60])), (table, i32([-2 ** 31, 60])), (table, i32([2 ** 31 - 1, 60]))):
        out = kv.attend(q, t, ln)
        assert vox.device_error() == 2
        assert torch.equal(out[n:], good[n:])
    assert torch.equal(kv.attend(q, table, kv_len), good) and vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("starts", [[0, 9000, 2], [-7, 1, 2], [0, 2 ** 31 - 1, 2 ** 31 - 1], [5, 0, 2]])
def test_bad_offsets(vox, act, cache, n, starts):
    bt = Batch([(n, 60), (n, 60)], KVH, HD, 16, cache, seed=1, fill=0.0)
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev()
    q = queries(bt, HEADS, act).cuda()
    good = kv.attend(q, table, kv_len, q_start=q_start, max_q=n)
    assert vox.device_error() == 0
    kv.attend(q, table, kv_len, q_start=i32(starts), max_q=n)
    assert vox.device_error() == 2
    assert torch.equal(kv.attend(q, table, kv_len, q_start=q_start, max_q=n), good) and vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("n,seqs", [(1, 2), (1, 60), (40, 2)])
def test_bad_prefix_page(vox, act, cache, n, seqs):
    """A prefix page out of range, where the call's own blocks read the prefix, where a launch of its own does, and in prompts."""
    bt = Batch([(n, 60)] * seqs, KVH, HD, 16, cache, seed=1, fill=0.0, prefix=200)
    kv = bt.handle(vox)
    table, kv_len, _ = bt.dev()
    pre = bt.prefix_pages.cuda()
    q = queries(bt, HEADS, act).cuda()
    good = kv.attend_prefix(q, pre, 200, table, kv_len)
    assert vox.device_error() == 0
    for at, bad in ((0, -1), (5, 10 ** 6), (12, 2 ** 31 - 1)):
        p = pre.clone()
        p[at] = bad
        kv.attend_prefix(q, p, 200, table, kv_len)
        assert vox.device_error() == 2
    assert torch.equal(kv.attend_prefix(q, pre, 200, table, kv_len), good) and vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
def test_bad_pages_among_many_sequences(vox, act, cache):
    """One bad page of one of many sequences, whose tiles all blocks share: reported, and every other sequence as before (the split
    does not depend on page numbers)."""
    lens = [(1, 30 + 7 * b % 400) for b in range(200)]
    lens[0] = (1, 3000)
    bt = Batch(lens, KVH, HD, 16, cache, seed=2, fill=0.0)
    kv = bt.handle(vox)
    table, kv_len, _ = bt.dev()
    q = queries(bt, HEADS, act).cuda()
    good = kv.attend(q, table, kv_len, max_kv=3000)
    assert vox.device_error() == 0
    t = table.clone()
    t[17, 0] = -1
    out = kv.attend(q, t, kv_len, max_kv=3000)
    assert vox.device_error() == 2
    keep = [b for b in range(200) if b != 17]
    assert torch.equal(out[keep], good[keep])
