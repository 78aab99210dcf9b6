"""examples/paged_talker.py (a batch of streams behind one voice prompt on a paged cache) against the same model computed in
64 bits, each stream by itself over its whole sequence: voice prompt, own text, decoded tokens.

The products of the example run in bf16 (2^-8 a rounding). A layer rounds, on the way of a value: the normed input, the
projection, q or k, the attention's weights and result, the output projection, the second norm, gate and up, their product
and the down projection, and the residual twice: 12 roundings, each an independent relative error of at most 2^-8 of values
of the hidden state's size, whose root mean square is a third of that; two layers: 24 of them, of a hidden state that grows
to about 3 times its input. sqrt(24) / 3 * 3 * 2^-8 = 0.02 expected, four times that allowed as root mean square."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def example():
    spec = importlib.util.spec_from_file_location("paged_talker", ROOT / "examples" / "paged_talker.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def talk64(t, h):
    """The talker over one whole sequence h [n][dim], causal, in 64 bits."""
    n, hd, kvh, grp = h.shape[0], t.hd, t.kv_heads, t.heads // t.kv_heads
    inv = torch.tensor([1e6 ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    norm = lambda x, w: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731

    def turn(x):
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    mask = torch.ones(n, n, dtype=torch.bool).tril()
    for w in t.host:
        w = {k: (v.to(torch.bfloat16) if v.dim() == 2 else v).double() for k, v in w.items()}
        x = (norm(h, w["ln1"]) @ w["qkv"].T).view(n, -1, hd)
        q, k, v = turn(norm(x[:, :t.heads], w["qn"])), turn(norm(x[:, t.heads:t.heads + kvh], w["kn"])), x[:, t.heads + kvh:]
        z = torch.einsum("nhgd,mhd->hgnm", q.view(n, kvh, grp, hd), k) * hd ** -0.5
        o = torch.einsum("hgnm,mhd->nhgd", torch.softmax(z.masked_fill(~mask, -torch.inf), -1), v).reshape(n, -1)
        h = h + o @ w["o"].T
        g, u = (norm(h, w["ln2"]) @ w["gu"].T).chunk(2, -1)
        h = h + (g * torch.sigmoid(g) * u) @ w["down"].T
    return h


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_streams_behind_one_voice(vox, dtype):
    r = example().run(streams=5, steps=20, layers=2, dtype=dtype, voice=100)
    t = r["talker"]
    close = lambda got, want: (got.double().cpu() - want).pow(2).mean().sqrt() <= 0.08 * want.pow(2).mean().sqrt()  # noqa: E731
    voice = r["voice"][0].double()
    assert close(r["voice"][1], talk64(t, voice))
    at = 0
    for b, n in enumerate(r["texts"]):
        h = torch.cat([voice, r["text"][0][at:at + n].double()] + [x[b:b + 1].double().cpu() for x, _ in r["steps"]])
        want = talk64(t, h)[100:]
        assert close(r["text"][1][at:at + n], want[:n])
        for i, (_, y) in enumerate(r["steps"]):
            assert close(y[b:b + 1], want[n + i:n + i + 1])
        at += n
    assert vox.device_error() == 0
