"""A batch of streams that speak with one voice: a small talker (a Qwen3-style transformer with random weights) decodes them
together on a paged key/value cache.

The voice prompt's keys and values are computed once and stand behind all streams as a shared prefix; every stream then
brings its own text (ragged lengths) and goes on token by token. One layer is: RMSNorm, the fused projection (PagedKV's
append splits, normalises, rotates and stores it), attention behind the shared prefix, the output projection with the
residual and the next norm, and the SwiGLU pair. Pages come from one pool; a stream takes a new page when its last is full.

    python examples/paged_talker.py [--streams 8] [--steps 16] [--layers 2] [--dtype bf16|f32]
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import vox_b200 as vox  # noqa: E402

EPS = 1e-6


class Pool:
    """Free pages of the cache, and the pages of every stream."""

    def __init__(self, pages: int, page: int, streams: int, width: int):
        self.free, self.page = list(range(pages))[::-1], page
        self.of = [[] for _ in range(streams)]
        self.table = torch.zeros((streams, width), dtype=torch.int32)

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise RuntimeError(f"the pool has {len(self.free)} free pages, {n} are needed")
        return [self.free.pop() for _ in range(n)]

    def grow(self, lens) -> None:
        for b, n in enumerate(lens):
            if n > self.table.shape[1] * self.page:
                raise RuntimeError(f"stream {b} has {n} rows, its page table holds {self.table.shape[1]} pages of {self.page}")
            while len(self.of[b]) * self.page < n:
                self.of[b] += self.take(1)
                self.table[b, len(self.of[b]) - 1] = self.of[b][-1]


def sizes(texts, steps: int, voice: int, page: int) -> tuple[int, int, int]:
    """(pages of the pool, pages of a stream's table, positions) that texts of these lengths need with `steps` more tokens each
    behind a voice prompt."""
    need = [-(-(n + steps) // page) for n in texts]
    return sum(need) + -(-voice // page), max(need), voice + max(texts) + steps


class Talker:
    """`layers` layers of `heads` query and `kv_heads` key/value heads of width `hd`, hidden size `dim`, on one pool of pages."""

    def __init__(self, layers=2, dim=256, heads=4, kv_heads=2, hd=64, ff=512, pages=256, page=16, positions=2048,
                 dtype=torch.bfloat16, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: (torch.randn(s, generator=g) / s[-1] ** 0.5)  # noqa: E731
        self.dim, self.heads, self.kv_heads, self.hd, self.dtype = dim, heads, kv_heads, hd, dtype
        self.host = [dict(qkv=rnd((heads + 2 * kv_heads) * hd, dim), o=rnd(dim, heads * hd), gu=rnd(2 * ff, dim), down=rnd(dim, ff),
                          ln1=1 + 0.1 * rnd(1, dim)[0], ln2=1 + 0.1 * rnd(1, dim)[0], qn=1 + 0.1 * rnd(1, hd)[0], kn=1 + 0.1 * rnd(1, hd)[0])
                     for _ in range(layers)]
        self.w = [{k: (t.to(device, torch.bfloat16) if t.dim() == 2 else t.to(device)) for k, t in w.items()} for w in self.host]
        z = lambda: torch.zeros((pages, page, kv_heads, hd), dtype=dtype, device=device)  # noqa: E731
        self.cache = [vox.PagedKV(z(), z()) for _ in range(layers)]
        self.cs = vox.rope_table(vox.rope_inv_freq(hd, 1e6, device), 0, positions)

    def _mm(self, x, w):
        return vox.gemm_bf16(x.to(torch.bfloat16), w, out_dtype=self.dtype)

    def forward(self, h, table, kv_len, q_start=None, max_q=0, max_kv=0, prefix=None):
        """h [tokens][dim] (updated in place, as the residual stream) -> hidden states. kv_len: rows of each stream's own pages with
        the new tokens. prefix: (pages, length) that all streams share, or None; it comes first in position."""
        delta = None
        own = dict(q_start=q_start, max_q=max_q, max_kv=max_kv)
        for w, kv in zip(self.w, self.cache):
            x = vox.rmsnorm(h, w["ln1"], EPS) if delta is None else vox.add_rmsnorm(h, delta, w["ln1"], EPS)
            # the cache row comes from kv_len, the rotation from the position: shift the table's rows by the prefix
            shift = 0 if prefix is None else prefix[1]
            q = kv.append(self._mm(x, w["qkv"]), self.cs[shift:], table, kv_len, self.heads, q_start=q_start, q_norm_w=w["qn"],
                          k_norm_w=w["kn"], eps=EPS)
            o = kv.attend(q, table, kv_len, **own) if prefix is None else kv.attend_prefix(q, prefix[0], prefix[1], table, kv_len, **own)
            x = vox.add_rmsnorm(h, self._mm(o, w["o"]), w["ln2"], EPS)
            delta = self._mm(vox.swiglu_fused(self._mm(x, w["gu"])), w["down"])
        return vox.add(h, delta)


def run(streams=8, steps=16, layers=2, dtype=torch.bfloat16, voice=100, page=16, seed=0):
    """Decodes `steps` tokens of every stream; returns the hidden states of the voice prompt, of the texts and of each step,
    with the inputs that led to them (the model's own output is the next input: a stand-in for sampling)."""
    g = torch.Generator().manual_seed(seed + 1)
    texts = [5 + int(x) for x in torch.randint(0, 40, (streams,), generator=g)]
    pages, width, positions = sizes(texts, steps, voice, page)
    t = Talker(layers=layers, dtype=dtype, seed=seed, page=page, pages=pages, positions=positions)
    pool = Pool(pages, page, streams, width)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    hidden = lambda n: torch.randn((n, t.dim), generator=g).to(dtype)  # noqa: E731
    # the voice prompt, once
    vp = pool.take(-(-voice // page))
    prefix = (dev(vp), voice)
    h_voice = hidden(voice)
    out_voice = t.forward(h_voice.cuda(), prefix[0][None].contiguous(), dev([voice]), max_q=voice, max_kv=voice)
    # the texts, ragged, behind it
    lens = list(texts)
    pool.grow(lens)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    h_text = hidden(starts[-1])
    out_text = t.forward(h_text.cuda(), pool.table.cuda(), dev(lens), q_start=dev(starts), max_q=max(lens), max_kv=max(lens),
                         prefix=prefix)
    x = out_text[torch.tensor(starts[1:], device="cuda") - 1]
    seen = []
    torch.cuda.synchronize()  # the voice and the texts are not part of a step
    t0 = time.perf_counter()
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        pool.grow(lens)
        x_in = x / x.float().pow(2).mean(-1, keepdim=True).sqrt().to(dtype)
        x = t.forward(x_in.clone(), pool.table.cuda(), dev(lens), max_q=1, max_kv=max(lens), prefix=prefix)
        seen.append((x_in, x))
    torch.cuda.synchronize()
    return dict(talker=t, texts=texts, voice=(h_voice, out_voice), text=(h_text, out_text), steps=seen, seconds=time.perf_counter() - t0)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--dtype", choices=["bf16", "f32"], default="bf16")
    args = ap.parse_args()
    r = run(args.streams, args.steps, args.layers, torch.bfloat16 if args.dtype == "bf16" else torch.float32)
    print(f"{args.streams} streams x {args.steps} steps behind one voice prompt: {r['seconds'] / max(args.steps, 1) * 1e3:.2f} ms a step")
