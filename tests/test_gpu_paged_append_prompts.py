"""The append of many tokens (vox_cuda_kv_append from 64 warp loads an SM on: four pairs of loads an item, two items a warp, several
tokens a block), against the 64-bit form and the bounds of test_gpu_paged.py's test_append."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged import BF16, EPS24, F32, IDS, KINDS, U, Batch, append64

pytestmark = pytest.mark.gpu

GEOM = [(16, 8, 128), (14, 2, 64), (5, 1, 128), (3, 3, 64)]


def ragged(act, heads, kvh, hd):
    """Sequences of together just more tokens than the many-token form starts at, of lengths that divide nothing; one of them
    without new tokens, two continued."""
    per = 32 // (hd // (32 // (4 if act == F32 else 2)))  # heads a warp load takes
    loads = -(-(heads + 2 * kvh) // per)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = sms * 64 // loads + 37
    cut = [n // 3 + 1, n // 5, 0, n // 4 + 3]
    cut.append(n - sum(cut))
    return [(q, q + e) for q, e in zip(cut, (0, 130, 9, 0, 61))]


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", GEOM)
@pytest.mark.parametrize("norms", [True, False], ids=["norms", "plain"])
def test_append_of_many_tokens(vox, act, cache, heads, kvh, hd, norms):
    lens = ragged(act, heads, kvh, hd)
    bt = Batch(lens, kvh, hd, 16, cache, seed=hd + heads)
    g = torch.Generator().manual_seed(11)
    units = heads + 2 * kvh
    wide = (torch.randn((bt.tokens, units * hd + 16), generator=g) * 2).to(act)  # rows of a wider projection
    qkv = wide[:, :units * hd]
    qn, kn = (1 + 0.3 * torch.randn(hd, generator=g) for _ in range(2)) if norms else (None, None)
    longest = max(n for _, n in lens)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e6), 0, longest)
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev()
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got_q = kv.append(wide.cuda()[:, :units * hd], cs, table, kv_len, heads, q_start=q_start, q_norm_w=dev(qn), k_norm_w=dev(kn), eps=1e-6)
    wq, wk, wv, qm, km = append64(bt, qkv.contiguous(), cs.cpu(), heads, qn, kn, 1e-6)
    seq = torch.tensor([b for b, (n, _) in enumerate(lens) for _ in range(n)])
    pos = torch.tensor([n_ - n + i for n, n_ in lens for i in range(n)])
    page, row = bt.table[seq, pos // 16].long(), pos % 16
    k2, v2 = kv.k.cpu(), kv.v.cpu()
    got_q, got_k, got_v = got_q.cpu().view(wq.shape), k2[page, row], v2[page, row]
    assert torch.equal(got_v, wv.to(act).to(cache))
    if norms:
        for got, want, m, dt in ((got_q, wq, qm, act), (got_k, wk, km, cache)):
            tol = 24 * EPS24 * m + (U * want.abs() * (1 + 2.0 ** -8) if dt == BF16 else 0)
            assert bool(((got.double() - want).abs() <= tol).all())
    else:
        x = qkv.float().reshape(bt.tokens, units, hd)
        c, s = cs.cpu()[pos, :, 0][:, None], cs.cpu()[pos, :, 1][:, None]
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
        assert torch.equal(got_q, y[:, :heads].to(act)) and torch.equal(got_k, y[:, heads:heads + kvh].to(cache))
    # nothing else of the cache has changed
    k2[page, row], v2[page, row] = bt.k[page, row], bt.v[page, row]
    bits = torch.int32 if cache == F32 else torch.int16
    assert torch.equal(k2.view(bits), bt.k.view(bits)) and torch.equal(v2.view(bits), bt.v.view(bits))
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", GEOM[:2])
def test_tokens_without_a_page_or_a_table_row_are_skipped_among_many(vox, act, cache, heads, kvh, hd):
    """Sixteen tokens whose page number is out of range, in the middle of a sequence and of blocks, and the last ones, whose
    positions have no row of the rotation table: their q rows and the cache stay, all others are as without them."""
    lens = ragged(act, heads, kvh, hd)
    bt = Batch(lens, kvh, hd, 16, cache, seed=5)
    units = heads + 2 * kvh
    qkv = (torch.randn((bt.tokens, units * hd), generator=torch.Generator().manual_seed(3)) * 2).to("cuda", act)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e6), 0, max(n for _, n in lens))
    table, kv_len, q_start = bt.dev()
    good = bt.handle(vox)
    want = good.append(qkv, cs, table, kv_len, heads, q_start=q_start)
    assert vox.device_error() == 0
    bad_table = table.clone()
    bad_table[0, 3] = 10 ** 6
    rows = lens[3][1] - 5  # of the fourth sequence, the last five positions and more of longer ones
    kv = bt.handle(vox)
    q = torch.full((bt.tokens, heads * hd), 7.0, dtype=act, device="cuda")
    kv.append(qkv, cs[:rows], bad_table, kv_len, heads, q_start=q_start, q=q)
    assert vox.device_error() == 2
    at = [(b, n_ - n + i) for b, (n, n_) in enumerate(lens) for i in range(n)]
    skipped = torch.tensor([p >= rows or (b == 0 and 48 <= p < 64) for b, p in at], device="cuda")
    assert 16 < int(skipped.sum()) < bt.tokens // 2
    assert bool((q[skipped] == 7.0).all()) and torch.equal(q[~skipped], want[~skipped])
    seq, pos = (torch.tensor(x) for x in zip(*at))
    page, row = bt.table[seq, pos // 16].long(), pos % 16
    bits = torch.int32 if cache == F32 else torch.int16
    for got, full, old in ((kv.k, good.k, bt.k), (kv.v, good.v, bt.v)):
        expect = full.cpu().clone()
        gone = skipped.cpu()
        expect[page[gone], row[gone]] = old[page[gone], row[gone]]
        assert torch.equal(got.cpu().view(bits), expect.view(bits))
