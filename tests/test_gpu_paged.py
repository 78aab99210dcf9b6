"""The paged key/value cache operators (PagedKV: append, attend, attend_prefix) against plain 64-bit implementations.

Tolerances (eps = 2^-24, the unit roundoff of f32 with its 24 significant bits; u = 2^-8, that of bf16 with 8), derived from the arithmetic of the kernels:
  append, no head norm: bit-exact against f32 products and sums rounded one by one (one more rounding for bf16 rows);
  append, head norm: the mean square is a sum of head_dim squares over at most 8 fused adds a lane and 5 butterfly adds,
    then rsqrt (2 ulp) and two products: < 16 eps relative; the rotation adds 3 roundings of terms |a| + |b| at most;
  attend, f32: a score is a chain of at most 4 fused adds, 1 add and 5 butterfly adds of products with a scaled q: its
    error is below 12 eps * sum |q k| scale =: d, doubled in a softmax weight relative to the sum; 2^x adds 2^-22; a
    weighted sum adds one rounding a key of its chain: (n / 4 + 64) eps. Together times the sum of p |v|;
  attend, bf16 on the tensor cores: products of bf16 are exact in f32; sums of up to 128 of them, aligned to the largest
    term: 128 eps * sum |q k| scale; each weight is rounded to bf16 (u relative), and the result once more.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS24, U = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16
KINDS = [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)]  # activations, cache
IDS = ["f32", "f32-bf16", "bf16", "bf16-f32"]


class Batch:
    """A pool of pages in shuffled order, NaN in every row that belongs to no sequence, and a ragged batch over it."""

    def __init__(self, lens, kvh, hd, page, cache, seed=0, prefix=0, spare=3, head_major=False, fill=math.nan):
        g = torch.Generator().manual_seed(seed)
        need = [-(-kv // page) for _, kv in lens]
        npre = -(-prefix // page)
        total = sum(need) + npre + spare
        order = torch.randperm(total, generator=g).tolist()
        self.lens, self.page, self.kvh, self.hd, self.prefix = lens, page, kvh, hd, prefix
        self.tokens = sum(q for q, _ in lens)
        self.table = torch.zeros((len(lens), max(need + [1]) + 1), dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.prefix_pages = torch.tensor(order[at:at + npre], dtype=torch.int32)
        self.k = torch.full((total, page, kvh, hd), fill)
        self.v = torch.full((total, page, kvh, hd), fill)
        self.seq_k, self.seq_v = [], []
        for b, (_, kv) in enumerate(lens):
            self._put(self.table[b], kv, g)
        if prefix:
            self._put(self.prefix_pages, prefix, g)
        self.k, self.v = self.k.to(cache), self.v.to(cache)
        self.head_major = head_major
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32)
        self.q_start = torch.tensor(np.concatenate([[0], np.cumsum([q for q, _ in lens])]), dtype=torch.int32)

    def rows(self, pages, n):
        r = torch.arange(n)
        return pages[r // self.page].long(), r % self.page

    def _put(self, pages, n, g):
        p, r = self.rows(pages, n)
        self.k[p, r] = torch.randn((n, self.kvh, self.hd), generator=g) * 1.5
        self.v[p, r] = torch.randn((n, self.kvh, self.hd), generator=g)

    def handle(self, vox):
        k, v = self.k.cuda(), self.v.cuda()
        if self.head_major:  # memory order [pages][kv_heads][page_size][head_dim]
            k, v = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v))
        return vox.PagedKV(k, v)

    def dev(self, uniform=False):
        return self.table.cuda(), self.kv_len.cuda(), None if uniform else self.q_start.cuda()


def attention64(bt, q, heads, scale, window=0):
    """(out, sum p |v|, largest sum |q k| scale) in 64 bits, token by token as the definition says."""
    grp = heads // bt.kvh
    out = torch.zeros((bt.tokens, heads, bt.hd), dtype=torch.float64)
    mag, big, at = torch.zeros_like(out), 0.0, 0
    for b, (n, kv) in enumerate(bt.lens):
        p, r = bt.rows(bt.table[b], kv)
        k, v = bt.k[p, r].double(), bt.v[p, r].double()
        if bt.prefix:
            p, r = bt.rows(bt.prefix_pages, bt.prefix)
            k, v = torch.cat((bt.k[p, r].double(), k)), torch.cat((bt.v[p, r].double(), v))
        for i in range(n):
            pos = kv - n + i
            lo = max(0, pos + 1 - window) if window else 0
            seen = torch.arange(max(k.shape[0], 0))
            keep = (seen < bt.prefix) | ((seen - bt.prefix <= pos) & (seen - bt.prefix >= lo))
            kk, vv = k[keep], v[keep]
            if kk.shape[0] == 0:
                continue
            qi = q[at + i].double().view(bt.kvh, grp, bt.hd)
            s = torch.einsum("hgd,nhd->hgn", qi, kk) * scale
            big = max(big, float((torch.einsum("hgd,nhd->hgn", qi.abs(), kk.abs()) * abs(scale)).max()))
            w = torch.softmax(s, -1)
            out[at + i] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(heads, bt.hd)
            mag[at + i] = torch.einsum("hgn,nhd->hgd", w, vv.abs()).reshape(heads, bt.hd)
        at += n
    return out, mag, big


def check(got, want, mag, big, act, cache, longest):
    got = got.double().cpu().view(want.shape)
    assert torch.isfinite(got).all()
    if act == BF16 and cache == BF16:
        tol = mag * (2 * 128 * EPS24 * big + 2 * U) + U * want.abs()
    else:
        tol = mag * (2 * 12 * EPS24 * big + 2.0 ** -22 + (longest / 4 + 64) * EPS24)
        if act == BF16:
            tol = tol + U * want.abs()
    bad = (got - want).abs() > tol + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside: worst {((got - want).abs() / (tol + 1e-30)).max():.2f} of the bound"


def queries(bt, heads, act, seed=1):
    return (torch.randn((bt.tokens, heads, bt.hd), generator=torch.Generator().manual_seed(seed)) * 1.5).to(act)


# the shapes where it can go wrong: empty and one-row sequences, lengths at, one below and one above a page and a tile of
# 128 keys, a sequence without new tokens, more new tokens than rows (the first see nothing)
TOKENS = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 0), (1, 127), (1, 128), (1, 129), (1, 700)]
MIXED = [(5, 5), (0, 33), (1, 200), (130, 130), (3, 2), (0, 0), (64, 129), (17, 300)]


@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (14, 2, 64), (4, 4, 64), (12, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("lens,page", [(TOKENS, 16), (MIXED, 32)], ids=["tokens", "mixed"])
def test_attend(vox, heads, kvh, hd, act, cache, lens, page):
    bt = Batch(lens, kvh, hd, page, cache, seed=heads)
    q = queries(bt, heads, act)
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev(uniform=lens is TOKENS)
    got = kv.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=max(n for n, _ in lens), max_kv=max(n for _, n in lens))
    assert got.dtype == act and got.shape == q.shape
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, 700)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("window", [1, 16, 77, 1000])
def test_attend_window(vox, act, cache, window):
    lens = [(1, 300), (40, 90), (129, 200), (1, 5), (2, 1)]
    bt = Batch(lens, 2, 64, 16, cache, seed=window)
    q = queries(bt, 6, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, window=window)
    want, mag, big = attention64(bt, q, 6, 64 ** -0.5, window)
    check(got, want, mag, big, act, cache, 300)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.5])
def test_attend_scale(vox, act, cache, scale):
    """Any scale: negative, zero (the mean of the values seen), large."""
    lens = [(1, 200), (50, 150), (3, 3)]
    bt = Batch(lens, 2, 64, 16, cache, seed=8)
    q = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, scale=scale)
    want, mag, big = attention64(bt, q, 4, scale)
    check(got, want, mag, big, act, cache, 200)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("prefix", [1, 64, 251, 600])
def test_attend_prefix(vox, act, cache, heads, kvh, hd, prefix):
    """A prefix that ends inside a page, own parts of no, one and many rows, one and several new tokens."""
    for lens in ([(1, 1), (1, 40), (1, 0), (1, 129)], [(3, 3), (0, 7), (60, 60), (1, 20), (9, 4)]):
        bt = Batch(lens, kvh, hd, 16, cache, seed=prefix, prefix=prefix)
        q = queries(bt, heads, act)
        table, kv_len, q_start = bt.dev()
        got = bt.handle(vox).attend_prefix(q.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, q_start=q_start)
        want, mag, big = attention64(bt, q, heads, hd ** -0.5)
        check(got, want, mag, big, act, cache, 800)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
def test_prefix_equals_its_rows_in_front(vox, act, cache):
    """A shared prefix of whole pages gives what a page table that starts with those pages gives."""
    heads, kvh, hd, page = 16, 8, 128, 64
    bt = Batch([(1, 100), (2, 31), (1, 64)], kvh, hd, page, cache, seed=4, prefix=192)
    q = queries(bt, heads, act).cuda()
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev()
    a = kv.attend_prefix(q, bt.prefix_pages.cuda(), 192, table, kv_len, q_start=q_start)
    front = bt.prefix_pages.cuda()[None].expand(3, -1)
    b = kv.attend(q, torch.cat((front, table), 1).contiguous(), kv_len + 192, q_start=q_start)
    tol = 2.0 ** -7 if act == BF16 else 2e-5
    assert (a.float() - b.float()).abs().max() <= tol * max(1.0, float(b.float().abs().max()))
    c = kv.attend_prefix(q, torch.empty(0, dtype=torch.int32, device="cuda"), 0, table, kv_len, q_start=q_start)
    d = kv.attend(q, table, kv_len, q_start=q_start)
    assert torch.equal(c, d)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("lens", [[(1, 40), (1, 300)], [(33, 40), (150, 300)]], ids=["tokens", "prompts"])
def test_attend_layouts_and_bounds(vox, act, cache, lens):
    """Head-major caches, q as a slice of a wider projection, a strided out, no host bounds or bounds that are too low, a
    wide page table, another stream: the same values as the plain layout, bit for bit where the split is the same."""
    heads, kvh, hd = 6, 2, 64
    bt = Batch(lens, kvh, hd, 16, cache, seed=9)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    kv = bt.handle(vox)
    base = kv.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=160, max_kv=512)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(base, want, mag, big, act, cache, 300)
    bt.head_major = True
    assert torch.equal(base, bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=160, max_kv=512))
    wide = torch.zeros((bt.tokens, (heads + 2 * kvh) * hd), dtype=act, device="cuda")
    wide[:, :heads * hd] = q.cuda().flatten(1)
    out = torch.full((bt.tokens, heads * hd + 16), 7.0, dtype=act, device="cuda")
    got = kv.attend(wide[:, :heads * hd], table, kv_len, q_start=q_start, max_q=160, max_kv=512, out=out[:, :heads * hd])
    assert torch.equal(got, base.flatten(1)) and bool((out[:, heads * hd:] == 7.0).all())
    for mq, mkv in ((0, 0), (1, 1), (7, 130)):
        got = kv.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=mq, max_kv=mkv)
        check(got, want, mag, big, act, cache, 300)
    big_table = torch.full((len(lens), 4000), -1, dtype=torch.int32, device="cuda")
    big_table[:, :table.shape[1]] = table
    got = kv.attend(q.cuda(), big_table, kv_len, q_start=q_start)
    check(got, want, mag, big, act, cache, 300)
    st = torch.cuda.Stream()
    qc = q.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        got = kv.attend(qc, table, kv_len, q_start=q_start, max_q=160, max_kv=512)
    st.synchronize()
    assert torch.equal(got, base)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", [(F32, BF16), (BF16, BF16)], ids=["f32-bf16", "bf16"])
def test_one_page_a_sequence_is_a_linear_cache(vox, act, cache):
    heads, kvh, hd = 14, 2, 64
    bt = Batch([(1, 500), (30, 480), (1, 3)], kvh, hd, 512, cache, seed=2, spare=0)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, 500)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
def test_runs_repeat_bit_for_bit(vox, act, cache):
    bt = Batch([(1, 900), (1, 3), (1, 450)], 8, 128, 16, cache, seed=3, prefix=333)
    q = queries(bt, 16, act).cuda()
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev()
    pre = bt.prefix_pages.cuda()
    a, b = kv.attend(q, table, kv_len), kv.attend_prefix(q, pre, 333, table, kv_len)
    for _ in range(5):
        assert torch.equal(a, kv.attend(q, table, kv_len))
        assert torch.equal(b, kv.attend_prefix(q, pre, 333, table, kv_len))


def test_graph_replay_sees_new_lengths(vox):
    """Lengths live on the device: a captured decode step serves later steps."""
    heads, kvh, hd = 16, 8, 128
    bt = Batch([(1, 200), (1, 90)], kvh, hd, 16, BF16, seed=5)
    q = queries(bt, heads, BF16)
    kv = bt.handle(vox)
    table, kv_len, _ = bt.dev()
    qc = q.cuda()
    kv.attend(qc, table, kv_len, max_kv=256)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv.attend(qc, table, kv_len, max_kv=256)
    for lens in ([(1, 200), (1, 90)], [(1, 31), (1, 1)], [(1, 150), (1, 0)]):
        bt.lens = lens
        kv_len.copy_(torch.tensor([n for _, n in lens], dtype=torch.int32))
        graph.replay()
        want, mag, big = attention64(bt, q, heads, hd ** -0.5)
        check(out, want, mag, big, BF16, BF16, 200)


@pytest.mark.parametrize("act,cache", [(F32, F32), (BF16, BF16)], ids=["f32", "bf16"])
def test_rows_past_2_to_31_elements(vox, act, cache):
    """Pages whose offsets need more than 32 bits, for the append and the attention that reads its rows."""
    kvh, hd, page, heads = 8, 128, 64, 16
    per = page * kvh * hd
    pages = (1 << 31) // per + 70
    k = torch.empty((pages, page, kvh, hd), dtype=cache, device="cuda")
    v = torch.empty_like(k)
    bt = Batch([(1, 100), (70, 100)], kvh, hd, page, cache, seed=6, spare=0)
    shift = pages - bt.k.shape[0]
    k[shift:], v[shift:] = bt.k.cuda(), bt.v.cuda()
    kv = vox.PagedKV(k, v)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    table = table + shift
    got = kv.attend(q.cuda(), table, kv_len, q_start=q_start)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, 100)
    qkv = torch.randn((2, (heads + 2 * kvh) * hd), device="cuda").to(act)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e6), 0, 128)
    kv.append(qkv, cs, table, kv_len, heads)
    for b in range(2):
        assert torch.equal(v[int(table[b, 99 // page]), 99 % page], qkv[b].view(-1, hd)[heads + kvh:].to(cache))
    assert vox.device_error() == 0


# ------------------------------------------------------------------ append

def append64(bt, qkv, cs, heads, qn, kn, eps):
    """(q, k rows, v rows, |a| + |b| of q and k) in 64 bits, by token."""
    kvh, hd = bt.kvh, bt.hd
    x = qkv.double().view(bt.tokens, heads + 2 * kvh, hd)
    pos = torch.tensor([kv - n + i for n, kv in bt.lens for i in range(n)])
    c, s = cs.double()[pos, :, 0][:, None], cs.double()[pos, :, 1][:, None]

    def turn(t, w):
        if w is not None:
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w.double()
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1), torch.cat((a.abs() + b.abs(),) * 2, -1)

    (q, qm), (k, km) = turn(x[:, :heads], qn), turn(x[:, heads:heads + kvh], kn)
    return q, k, x[:, heads + kvh:], qm, km


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (14, 2, 64), (3, 3, 64), (5, 1, 128)])
@pytest.mark.parametrize("lens", [[(1, 1), (1, 16), (1, 17), (1, 400)], [(3, 3), (0, 0), (40, 90), (1, 20), (0, 5), (300, 300)]],
                         ids=["tokens", "prompts"])
@pytest.mark.parametrize("norms", [True, False], ids=["norms", "plain"])
def test_append(vox, act, cache, heads, kvh, hd, lens, norms):
    bt = Batch(lens, kvh, hd, 16, cache, seed=hd)
    g = torch.Generator().manual_seed(11)
    qkv = (torch.randn((bt.tokens, (heads + 2 * kvh) * hd), generator=g) * 2).to(act)
    qn, kn = (1 + 0.3 * torch.randn(hd, generator=g) for _ in range(2)) if norms else (None, None)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e6), 0, 512)
    kv = bt.handle(vox)
    table, kv_len, q_start = bt.dev(uniform=all(n == 1 for n, _ in lens))
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    q = kv.append(qkv.cuda(), cs, table, kv_len, heads, q_start=q_start, q_norm_w=dev(qn), k_norm_w=dev(kn), eps=1e-6)
    assert q.dtype == act
    wq, wk, wv, qm, km = append64(bt, qkv, cs.cpu(), heads, qn, kn, 1e-6)
    seq = [b for b, (n, _) in enumerate(lens) for _ in range(n)]
    pos = [kv_ - n + i for n, kv_ in lens for i in range(n)]
    page = torch.tensor([int(bt.table[b, p // 16]) for b, p in zip(seq, pos)])
    row = torch.tensor(pos) % 16
    k2, v2 = kv.k.cpu(), kv.v.cpu()
    got_q, got_k, got_v = q.cpu().view(wq.shape), k2[page, row], v2[page, row]
    assert torch.equal(got_v, wv.to(act).to(cache))  # v heads are copied
    if norms:
        for got, want, m, dt in ((got_q, wq, qm, act), (got_k, wk, km, cache)):
            tol = 24 * EPS24 * m + (U * want.abs() * (1 + 2.0 ** -8) if dt == BF16 else 0)
            assert bool(((got.double() - want).abs() <= tol).all())
    else:  # the CPU's arithmetic: every product and sum rounded by itself, then once to the destination
        x = qkv.float().view(bt.tokens, heads + 2 * kvh, hd)
        c, s = cs.cpu()[pos, :, 0][:, None], cs.cpu()[pos, :, 1][:, None]
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
        assert torch.equal(got_q, y[:, :heads].to(act)) and torch.equal(got_k, y[:, heads:heads + kvh].to(cache))
    # nothing else of the cache has changed
    k2[page, row], v2[page, row] = bt.k[page, row], bt.v[page, row]
    assert torch.equal(k2.view(torch.int32 if cache == F32 else torch.int16), bt.k.view(torch.int32 if cache == F32 else torch.int16))
    assert torch.equal(v2.view(torch.int32 if cache == F32 else torch.int16), bt.v.view(torch.int32 if cache == F32 else torch.int16))
    assert vox.device_error() == 0


def test_append_matches_the_linear_cache_operator(vox):
    """One sequence, one page: the same bits as qkv_rope writes into a linear cache."""
    heads, kvh, hd, m, pos0 = 16, 8, 128, 37, 5
    qkv = torch.randn((m, (heads + 2 * kvh) * hd), device="cuda")
    qn, kn = torch.rand(hd, device="cuda") + 0.5, torch.rand(hd, device="cuda") + 0.5
    inv = vox.rope_inv_freq(hd, 1e6)
    kc, vc = (torch.zeros((64, kvh * hd), device="cuda") for _ in range(2))
    want = vox.qkv_rope(qkv, vox.rope_table(inv, pos0, m), heads, kvh, hd, kc, vc, pos0, q_norm_w=qn, k_norm_w=kn)
    kv = vox.PagedKV(torch.zeros((1, 64, kvh, hd), device="cuda"), torch.zeros((1, 64, kvh, hd), device="cuda"))
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    got = kv.append(qkv, vox.rope_table(inv, 0, 64), table, torch.tensor([pos0 + m], dtype=torch.int32, device="cuda"), heads, q_norm_w=qn,
                    k_norm_w=kn)
    assert torch.equal(got, want)
    assert torch.equal(kv.k.view(64, -1), kc) and torch.equal(kv.v.view(64, -1), vc)


# ------------------------------------------------------------------ what is out of range, and refusals

def test_out_of_range_lengths_and_pages_are_reported(vox):
    heads, kvh, hd = 4, 2, 64
    bt = Batch([(1, 20), (1, 20)], kvh, hd, 16, F32, seed=1, fill=0.0)
    kv = bt.handle(vox)
    table, kv_len, _ = bt.dev()
    q = queries(bt, heads, F32).cuda()
    good = kv.attend(q, table, kv_len)
    assert vox.device_error() == 0
    for t, n in ((torch.tensor([[10 ** 6, 1, 0], table[1].tolist()], dtype=torch.int32).cuda(), kv_len),
                 (torch.tensor([[-5, 1, 0], table[1].tolist()], dtype=torch.int32).cuda(), kv_len),
                 (table, torch.tensor([-3, 20], dtype=torch.int32).cuda()),
                 (table, torch.tensor([2 ** 31 - 1, 20], dtype=torch.int32).cuda())):
        out = kv.attend(q, t, n)
        assert vox.device_error() == 2
        assert torch.equal(out[1], good[1])  # the other sequence is not touched by it
    starts = torch.tensor([0, 9, 2], dtype=torch.int32).cuda()
    kv.attend(q, table, kv_len, q_start=starts)
    assert vox.device_error() == 2
    # append: tokens without a page or a table row are skipped
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e4), 0, 19)  # position 19 has no row
    before = kv.k.clone()
    qkv = torch.randn((2, (heads + 2 * kvh) * hd), device="cuda")
    kv.append(qkv, cs, table, kv_len, heads)
    assert vox.device_error() == 2 and torch.equal(before, kv.k)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e4), 0, 64)
    kv.append(qkv, cs, torch.full_like(table, 10 ** 6), kv_len, heads)
    assert vox.device_error() == 2 and torch.equal(before, kv.k)
    kv.append(qkv, cs, table, torch.tensor([0, 49], dtype=torch.int32).cuda(), heads)
    assert vox.device_error() == 2 and torch.equal(before, kv.k)


def test_refusals(vox):
    E = vox.VoxCudaError
    z = lambda *s, dt=F32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    for bad in ((z(2, 16, 2, 96), "head_dim"), (z(2, 24, 2, 64), "page_size"), (z(2, 8, 2, 64), "page_size")):
        kv = vox.PagedKV(bad[0], bad[0].clone())
        with pytest.raises(E, match=bad[1]):
            kv.attend(z(1, 2 * bad[0].shape[3]), z(1, 2, dt=torch.int32), z(1, dt=torch.int32))
    with pytest.raises(E):
        vox.PagedKV(z(2, 16, 2, 64), z(2, 16, 2, 64).cpu())
    with pytest.raises(E):
        vox.PagedKV(z(2, 16, 2, 64), z(2, 16, 1, 64))
    with pytest.raises(E):
        vox.PagedKV(z(2, 16, 2, 64, dt=torch.float16), z(2, 16, 2, 64, dt=torch.float16))
    kv = vox.PagedKV(z(2, 16, 2, 64), z(2, 16, 2, 64))
    table, n1 = z(1, 2, dt=torch.int32), z(1, dt=torch.int32)
    with pytest.raises(E, match="multiple of kv_heads"):
        kv.attend(z(1, 3 * 64), table, n1)
    with pytest.raises(E, match="whole heads"):
        kv.attend(z(1, 100), table, n1)
    with pytest.raises(E, match="page_table"):
        kv.attend(z(1, 128), table.long(), n1)
    with pytest.raises(E, match="agree"):
        kv.attend(z(1, 128), table, z(2, dt=torch.int32))
    with pytest.raises(E, match="multiple of seqs"):
        kv.attend(z(3, 128), z(2, 2, dt=torch.int32), z(2, dt=torch.int32))
    with pytest.raises(E, match="float32 or bfloat16"):
        kv.attend(z(1, 128, dt=torch.float16), table, n1)
    with pytest.raises(E, match="out must have"):
        kv.attend(z(1, 128), table, n1, out=z(1, 128, dt=BF16))
    with pytest.raises(E, match="window"):
        kv.attend(z(1, 128), table, n1, window=-1)
    with pytest.raises(E, match="prefix_len"):
        kv.attend_prefix(z(1, 128), table[0], 33, table, n1)
    with pytest.raises(E, match="aligned"):
        kv.attend(z(129)[1:].view(1, 128), table, n1)
    cs = z(8, 32, 2)
    with pytest.raises(E, match="qkv"):
        kv.append(z(1, 128), cs, table, n1, 2)
    with pytest.raises(E, match="cs"):
        kv.append(z(1, 6 * 64), z(8, 64, 2), table, n1, 2)
    with pytest.raises(E, match="q_norm_w"):
        kv.append(z(1, 6 * 64), cs, table, n1, 2, q_norm_w=z(32))
    # nothing to do is no error
    assert kv.attend(z(0, 128), table, n1, q_start=z(2, dt=torch.int32)).shape == (0, 128)
    assert kv.append(z(0, 6 * 64), cs, table, n1, 2, q_start=z(2, dt=torch.int32)).shape == (0, 128)
    # no page listed: no key, zeros
    out = kv.attend(torch.ones((1, 128), device="cuda"), z(1, 0, dt=torch.int32), n1)
    assert bool((out == 0).all())


# ------------------------------------------------------------------ the ways a call is cut

@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("prefix", [0, 140])
def test_many_sequences_share_the_blocks(vox, act, cache, heads, kvh, hd, prefix):
    """More sequences than a block has threads, lengths from 0 to several tiles: equal runs of all sequences' tiles, with and
    without offsets of the tokens, sequences without new tokens and without keys among them."""
    rng = np.random.default_rng(5)
    kv = [int(x) for x in rng.integers(0, 260, 300)]
    kv[0], kv[7], kv[8], kv[299] = 1500, 0, 0, 1
    bt = Batch([(1, n) for n in kv], kvh, hd, 16, cache, seed=1, prefix=prefix)
    q = queries(bt, heads, act)
    table, kv_len, _ = bt.dev(uniform=True)
    h = bt.handle(vox)
    call = (lambda **k: h.attend_prefix(q.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, max_kv=1500, **k)) if prefix else \
        (lambda **k: h.attend(q.cuda(), table, kv_len, max_kv=1500, **k))
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(call(), want, mag, big, act, cache, 1700)
    got = call(q_start=bt.q_start.cuda(), max_q=1)
    check(got, want, mag, big, act, cache, 1700)
    # some sequences have no new token, one has more than the host says (of rows for two blocks of the few-row kernels)
    lens = [(int(x), n) for x, n in zip(rng.integers(0, 2, 300), kv)]
    lens[0], lens[7], lens[40] = (21, 1500), (3, 0), (5, 3)
    bt = Batch(lens, kvh, hd, 16, cache, seed=2, prefix=prefix)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    h = bt.handle(vox)
    got = call(q_start=q_start, max_q=1)
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    check(got, want, mag, big, act, cache, 1700)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("window", [1, 50, 300])
def test_window_over_many_sequences(vox, act, cache, window):
    lens = [(1, int(n)) for n in np.random.default_rng(6).integers(1, 900, 90)]
    bt = Batch(lens, 4, 128, 16, cache, seed=window)
    q = queries(bt, 8, act)
    table, kv_len, _ = bt.dev(uniform=True)
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, max_kv=3000, window=window)
    want, mag, big = attention64(bt, q, 8, 128 ** -0.5, window)
    check(got, want, mag, big, act, cache, 900)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("page", [16, 64, 128, 512])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_of_several_row_blocks(vox, act, cache, page, hd):
    """Prompts that continue cached rows, of several blocks of rows and tiles of keys, that end one row before, at and past
    the ends of tiles, steps and pages."""
    lens = [(257, 640), (128, 128), (129, 513), (64, 65), (1, 511), (300, 301)]
    bt = Batch(lens, 2, hd, page, cache, seed=page)
    q = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev()
    h = bt.handle(vox)
    want, mag, big = attention64(bt, q, 4, hd ** -0.5)
    for mq, mkv in ((300, 640), (0, 0)):
        check(h.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=mq, max_kv=mkv), want, mag, big, act, cache, 640)
    want, mag, big = attention64(bt, q, 4, hd ** -0.5, window=100)
    check(h.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=300, window=100), want, mag, big, act, cache, 640)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("q", [1, 9, 70])
def test_prefix_of_many_tiles(vox, act, cache, q):
    """A prefix cut into several key ranges, against single tokens, short continuations and prompts."""
    bt = Batch([(q, q), (q, q + 150)] * 9, 2, 128, 64, cache, seed=q, prefix=1000)
    x = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev(uniform=True)
    got = bt.handle(vox).attend_prefix(x.cuda(), bt.prefix_pages.cuda(), 1000, table, kv_len, max_kv=q + 150)
    want, mag, big = attention64(bt, x, 4, 128 ** -0.5)
    check(got, want, mag, big, act, cache, 1200)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("prefix", [1, 17, 300, 1500])
def test_prefix_of_few_short_sequences(vox, act, cache, heads, kvh, hd, prefix):
    """Single tokens of few sequences, so that a call's blocks take the prefix and the own rows side by side: prefixes of one
    row to several blocks, own rows of one to more than max_kv said, a sequence without new tokens."""
    bt = Batch([(1, 1), (1, 130), (0, 9), (1, 511), (1, 16)], kvh, hd, 16, cache, seed=prefix, prefix=prefix)
    q = queries(bt, heads, act)
    table, kv_len, q_start = bt.dev()
    want, mag, big = attention64(bt, q, heads, hd ** -0.5)
    h, pre = bt.handle(vox), bt.prefix_pages.cuda()
    for max_kv in (511, 40, 0):
        got = h.attend_prefix(q.cuda(), pre, prefix, table, kv_len, q_start=q_start, max_q=1, max_kv=max_kv)
        check(got, want, mag, big, act, cache, 2100)
        assert torch.equal(got, h.attend_prefix(q.cuda(), pre, prefix, table, kv_len, q_start=q_start, max_q=1, max_kv=max_kv))
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("seqs,longest,prefix", [(24, 4, 700), (48, 36, 1000)])
def test_prefix_of_many_texts(vox, act, cache, seqs, longest, prefix):
    """Texts that fill little of a row tile each behind a long prefix, counted together and apart."""
    r = np.random.default_rng(seqs)
    lens = [(int(n), int(n) + int(e)) for n, e in zip(r.integers(1, longest + 1, seqs), r.integers(0, 30, seqs))]
    lens[3], lens[7] = (longest, longest), (0, 5)
    bt = Batch(lens, 8, 64, 16, cache, seed=seqs, prefix=prefix)
    q = queries(bt, 56, act)
    table, kv_len, q_start = bt.dev()
    want, mag, big = attention64(bt, q, 56, 64 ** -0.5)
    h = bt.handle(vox)
    for mq, mkv in ((longest, longest + 30), (1, 1), (0, 0)):
        got = h.attend_prefix(q.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, q_start=q_start, max_q=mq, max_kv=mkv)
        check(got, want, mag, big, act, cache, prefix + longest + 30)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("q", [4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("prefix", [0, 200])
def test_rows_where_the_kernels_change(vox, act, cache, q, prefix):
    """Two query heads a key/value head: 8, 10, 16, 18, 32 and 34 rows a sequence."""
    bt = Batch([(q, q), (q, 150), (q, q + 1), (q, 333), (q, 0), (q, 2)], 2, 128, 32, cache, seed=q, prefix=prefix)
    x = queries(bt, 4, act)
    table, kv_len, _ = bt.dev(uniform=True)
    h = bt.handle(vox)
    got = h.attend_prefix(x.cuda(), bt.prefix_pages.cuda(), prefix, table, kv_len, max_kv=333) if prefix else \
        h.attend(x.cuda(), table, kv_len, max_kv=333)
    want, mag, big = attention64(bt, x, 4, 128 ** -0.5)
    check(got, want, mag, big, act, cache, 540)
    assert vox.device_error() == 0


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hd,prefix", [(64, 0), (128, 0), (128, 333), (64, 70)])
def test_many_short_prompts(vox, page, hd, prefix):
    """Prompts of at most 128 rows, more of them than the device has room for at once: with and without cached rows in front,
    ends before, at and past steps of 64 keys, a window, sequences longer than max_q and max_kv say."""
    r = np.random.default_rng(page)
    lens = [(int(n), int(n) + int(e)) for n, e in zip(r.integers(1, 65, 30), r.integers(0, 300, 30))]
    lens[:6] = [(64, 64), (63, 65), (64, 128), (1, 129), (0, 70), (64, 513)]
    bt = Batch(lens, 8, hd, page, BF16, seed=page, prefix=prefix)
    q = queries(bt, 16, BF16)
    table, kv_len, q_start = bt.dev()
    h, pre = bt.handle(vox), bt.prefix_pages.cuda()
    want, mag, big = attention64(bt, q, 16, hd ** -0.5)
    for mq, mkv in ((64, 513), (20, 100), (40, 0)):
        kw = dict(q_start=q_start, max_q=mq, max_kv=mkv)
        got = h.attend_prefix(q.cuda(), pre, prefix, table, kv_len, **kw) if prefix else h.attend(q.cuda(), table, kv_len, **kw)
        check(got, want, mag, big, BF16, BF16, 900)
    if not prefix:
        want, mag, big = attention64(bt, q, 16, hd ** -0.5, window=90)
        check(h.attend(q.cuda(), table, kv_len, q_start=q_start, max_q=64, window=90), want, mag, big, BF16, BF16, 900)
    assert vox.device_error() == 0


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
def test_scores_that_keep_rising(vox, act, cache):
    """Every step's largest score is far above the last one's, so the running maximum moves at each; and far below, so it
    never does."""
    for sign in (1.0, -1.0):
        bt = Batch([(1, 700), (150, 700)], 2, 64, 16, cache, seed=7)
        ramp = (torch.arange(700) / 700.0 * 40.0 * sign)[:, None, None]
        for b in range(2):
            p, r = bt.rows(bt.table[b], 700)
            bt.k[p, r] = (torch.ones(700, 2, 64) * ramp / 8).to(cache)
        q = torch.ones((bt.tokens, 4, 64)).to(act)
        table, kv_len, q_start = bt.dev()
        got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=150)
        want, mag, big = attention64(bt, q, 4, 64 ** -0.5)
        check(got, want, mag, big, act, cache, 700)


@pytest.mark.parametrize("act,cache", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [1, 80])
def test_nan_in_a_query_or_key_reaches_its_rows_only(vox, act, cache, n):
    """A query that holds NaN gives NaN in its own row; a key that holds NaN, in the rows that see it."""
    bt = Batch([(n, 200), (n, 150)], 2, 64, 16, cache, seed=3)
    q = queries(bt, 4, act)
    table, kv_len, q_start = bt.dev()
    clean = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=n)
    bad = q.clone()
    bad[n - 1, 2, 5] = math.nan
    got = bt.handle(vox).attend(bad.cuda(), table, kv_len, q_start=q_start, max_q=n)
    assert bool(torch.isnan(got[n - 1, 2]).all())
    keep = torch.ones((2 * n, 4), dtype=torch.bool)
    keep[n - 1, 2] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
    p, r = bt.rows(bt.table[1], 150)
    bt.k[p[149], r[149], 0, 3] = math.nan  # the last key of the second sequence, key/value head 0: its last token alone sees it
    got = bt.handle(vox).attend(q.cuda(), table, kv_len, q_start=q_start, max_q=n)
    assert bool(torch.isnan(got[2 * n - 1, :2]).all())
    keep = torch.ones((2 * n, 4), dtype=torch.bool)
    keep[2 * n - 1, :2] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
