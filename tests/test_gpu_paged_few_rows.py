"""The few-row kernels at every number of rows that they are built for: 1, 2, 4 and 8 on the CUDA cores, 8 and 16 on the tensor cores, in
heads of 64 and 128, in the frames that a small call (clusters) and a large one (equal runs of all tiles) take, with and
without a shared prefix.

Bounds: those of test_gpu_paged.py's check, 2 * 12 eps d + 2^-22 + (n / 4 + 64) eps of the sum of p |v| (eps = 2^-24, d = sum |q k| scale of a
row's largest key, twice because a score's error reaches the weight and the sum). What the kernels at f32 accuracy compute:
  CUDA cores: q times the scale 2 eps, a product and a fused add, one add of the halves, at most 5 exchanged adds: 9 eps d.
  bf16 cache, q in three bf16 parts: the parts hold q to 2^-27 and their products are exact; six chains of hd / 32 tensor-core steps, each
    cut within 2 eps of its partial sum, then 5 adds and the scale: 14 eps d if every partial sum were d and every error had one sign.
    Partial sums of products of random signs are near d / sqrt(hd): 6 adds and cuts of d / 8 stay below 2 eps d.
  TF32, operands cut in two: what is cut off a product is at most 2^-21 for each lo part and 2^-22 for lo lo, 20 eps of |q k|, with the
    random sign of the part that it is cut off: a sum of hd of them has a standard deviation below 20 eps d / sqrt(hd) = 2.5 eps d, four of
    which are 10; hd / 8 chained steps cut within 2 eps of a partial sum near d / sqrt(hd) add less than 2 eps d (hd 64: 8 * 2 / 8).
  The weights carry the 2^-22 of 2^x; a sum over n keys rounds once a key of its chain, of which a warp holds a part.
So 12 eps d is a bound for the first and, for inputs of random signs as here, more than four standard deviations for the others."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_paged import IDS, KINDS, Batch, attention64, check, queries

pytestmark = pytest.mark.gpu

# (heads, kv heads, head width, new tokens a sequence): rows a key/value head = heads / kv heads * tokens
ROWS = [(2, 2, 128, 1), (3, 1, 128, 1), (8, 2, 128, 1), (4, 2, 128, 1), (6, 1, 128, 1), (2, 2, 64, 1), (4, 2, 64, 1), (6, 2, 64, 1),
        (4, 1, 64, 1), (7, 1, 64, 1), (14, 2, 64, 2), (12, 1, 64, 1), (3, 1, 64, 4), (6, 2, 128, 5)]


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd,n", ROWS)
@pytest.mark.parametrize("prefix", [0, 140])
@pytest.mark.parametrize("seqs", [3, 150])
def test_rows_of_every_kernel(vox, act, cache, heads, kvh, hd, n, prefix, seqs):
    r = np.random.default_rng(heads + hd)
    kv = [int(x) for x in r.integers(n, 260, seqs)]
    kv[0], kv[1], kv[2] = 700 if seqs == 3 else 1500, 0, n
    bt = Batch([(n, x) for x in kv], kvh, hd, 16, cache, seed=heads, prefix=prefix)
    q = queries(bt, heads, act)
    table, kv_len, _ = bt.dev(uniform=True)
    h = bt.handle(vox)
    kw = dict(max_kv=max(kv))
    got = h.attend_prefix(q.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, **kw) if prefix else h.attend(q.cuda(), table, kv_len, **kw)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, max(kv) + prefix)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd,n", [(2, 2, 128, 1), (4, 1, 128, 1), (7, 1, 64, 2)])
def test_more_tokens_than_the_bound(vox, act, cache, heads, kvh, hd, n):
    """Sequences with more new tokens than max_q says, so that a kernel of few rows takes several row tiles."""
    lens = [(n, 300), (9 * n, 40), (0, 5), (5 * n + 1, 700)]
    bt = Batch(lens, kvh, hd, 16, cache, seed=7)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=n, max_kv=700)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, 700)
    assert vox.device_error() == 0
