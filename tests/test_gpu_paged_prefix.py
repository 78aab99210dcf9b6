"""The calls that put a text behind a shared prefix, in the order in which they are documented: the prefix appended once, the text
with the rotation table from row prefix_len on, attend_prefix. Together they are one sequence of prefix and text."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("voice,text", [(1, 1), (33, 7), (100, 60)])
def test_prefix_and_text_are_one_sequence(vox, dtype, voice, text):
    heads, kvh, hd, page, n = 4, 2, 64, 16, voice + text
    g = torch.Generator().manual_seed(voice)
    qkv = torch.randn((n, (heads + 2 * kvh) * hd), generator=g).to("cuda", dtype)
    cs = vox.rope_table(vox.rope_inv_freq(hd, 1e4), 0, n)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    new = lambda pages: vox.PagedKV(*(torch.zeros((pages, page, kvh, hd), dtype=dtype, device="cuda") for _ in range(2)))  # noqa: E731
    pages = -(-n // page)
    one = new(pages)
    table = dev([list(range(pages))])
    q = one.append(qkv, cs, table, dev([n]), heads)
    want = one.attend(q, table, dev([n]))
    front, own = -(-voice // page), -(-text // page)
    two = new(front + own)
    pre, table = dev(list(range(front))), dev([list(range(front, front + own))])
    qv = two.append(qkv[:voice], cs, pre[None], dev([voice]), heads)
    qt = two.append(qkv[voice:], cs[voice:], table, dev([text]), heads)
    # the same positions: the same bits of q and of every key
    assert torch.equal(torch.cat((qv, qt)), q)
    rows = lambda kv, p0, m: kv.k.flatten(0, 1)[p0 * page:p0 * page + m]  # noqa: E731
    assert torch.equal(torch.cat((rows(two, 0, voice), rows(two, front, text))), rows(one, 0, n))
    got = two.attend_prefix(qt, pre, voice, table, dev([text]))
    # two orders of the same sums over at most 160 values of size 1: bf16 weights and results 2^-8 each, on both sides; f32 as in
    # test_gpu_paged.py's comparison of a prefix with its rows in front
    tol = 2.0 ** -6 if dtype == torch.bfloat16 else 2e-5
    assert (got.float() - want[voice:].float()).abs().max() <= tol * max(1.0, float(want.float().abs().max()))
    assert vox.device_error() == 0
