"""Measured cases of the paged key/value cache operators: the append (QKV split, head norms, rotation, cache write), the
attention that reads the cache (prompts and single tokens, ragged batches) and the attention of a batch that shares a
long prefix (a voice prompt) and goes on with keys of its own.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits, rounded once at the end)
or, where `own` is true, through vox_b200. `exact` states the same results in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
THETA = 1e6   # rotation base of the 128-wide heads' talker; any base gives the same work
EPS = 1e-6

# (query heads, key/value heads, head width): the repository's prefill chunk (16 q / 8 kv heads of 128), and two of
# 64-wide heads, one with an odd number of query heads to a key/value head and one with a key/value head for each
GEOM = {"16x8x128": (16, 8, 128), "14x2x64": (14, 2, 64), "16x16x64": (16, 16, 64)}


def listed():
    return [
        # one stream's next token in f32 (the CPU engine's own precision): the smallest call, latency only
        {"name": "append_token_f32", "op": "append", "geom": "16x8x128", "act": "f32", "cache": "f32", "page": 16, "seqs": 1, "q_min": 1,
         "q_max": 1, "kv_min": 700, "kv_max": 700, "mix": 1},
        # the prompts of a batch, ragged, bf16
        {"name": "append_prompts_bf16", "op": "append", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 64, "seqs": 7,
         "q_min": 37, "q_max": 2900, "kv_min": 37, "kv_max": 3300, "mix": 3},
        # one stream's next token in f32: 650 keys, latency
        {"name": "token_one_f32", "op": "attend", "geom": "16x8x128", "act": "f32", "cache": "f32", "page": 16, "seqs": 1, "q_min": 1,
         "q_max": 1, "kv_min": 650, "kv_max": 650, "mix": 4},
        # a serving batch in mid-speech with 7 query heads to a key/value head, ragged lengths, small pages
        {"name": "tokens_ragged_bf16", "op": "attend", "geom": "14x2x64", "act": "bf16", "cache": "bf16", "page": 16, "seqs": 96, "q_min": 1,
         "q_max": 1, "kv_min": 1, "kv_max": 6000, "mix": 5},
        # f32 activations on a bf16 cache (the quantized matvec's outputs are f32)
        {"name": "tokens_mixed", "op": "attend", "geom": "16x8x128", "act": "f32", "cache": "bf16", "page": 32, "seqs": 33, "q_min": 1,
         "q_max": 1, "kv_min": 300, "kv_max": 2500, "mix": 6},
        # long-form narration: 16 streams of up to 32768 cached keys
        {"name": "tokens_long_bf16", "op": "attend", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 64, "seqs": 16, "q_min": 1,
         "q_max": 1, "kv_min": 20000, "kv_max": 32768, "mix": 7},
        # prompts of a batch in f32 (the CPU engine's own precision)
        {"name": "prompts_f32", "op": "attend", "geom": "16x16x64", "act": "f32", "cache": "f32", "page": 32, "seqs": 5, "q_min": 90, "q_max": 700,
         "kv_min": 90, "kv_max": 900, "mix": 8},
        # ragged prompts of a batch, some of them continued, bf16
        {"name": "prompts_ragged_bf16", "op": "attend", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 64, "seqs": 7,
         "q_min": 61, "q_max": 2900, "kv_min": 61, "kv_max": 4100, "mix": 9},
        # one long document prompt: the largest
        {"name": "prompt_long_bf16", "op": "attend", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 128, "seqs": 1,
         "q_min": 8191, "q_max": 8191, "kv_min": 8191, "kv_max": 8191, "mix": 10},
        # eight streams with one short voice prompt that ends inside a page, f32 activations on a bf16 cache
        {"name": "prefix_short_mixed", "op": "prefix", "geom": "14x2x64", "act": "f32", "cache": "bf16", "page": 16, "seqs": 8, "q_min": 1,
         "q_max": 1, "kv_min": 1, "kv_max": 400, "prefix": 251, "mix": 11},
        # the texts of a batch, ragged, behind the one voice prompt that they share
        {"name": "prefix_texts_bf16", "op": "prefix", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 32, "seqs": 24,
         "q_min": 7, "q_max": 150, "kv_min": 7, "kv_max": 150, "prefix": 1003, "mix": 2},
        # a full batch with one long voice and style prompt
        {"name": "prefix_long_bf16", "op": "prefix", "geom": "16x8x128", "act": "bf16", "cache": "bf16", "page": 64, "seqs": 128, "q_min": 1,
         "q_max": 1, "kv_min": 1, "kv_max": 1000, "prefix": 8100, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One case of the listed ranges: token and prompt calls of each operator, each geometry and pair of types."""
    most, largest = max(_cost(c) for c in listed()), {c["name"]: c for c in listed()}
    while True:
        kind = rng.choice(["append_token", "append_prompt", "token", "token", "prompt", "prefix", "prefix_text"])
        act, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
        case = {"geom": rng.choice(sorted(GEOM)), "act": act, "cache": cache, "page": rng.choice([16, 32, 64, 128]),
                "mix": rng.randrange(1 << 30)}
        if kind == "append_token":
            hi = _log_int(rng, 20, 3300)
            case.update(op="append", seqs=_log_int(rng, 1, 128), q_min=1, q_max=1, kv_min=_log_int(rng, 1, hi), kv_max=hi)
        elif kind == "append_prompt":
            q = _log_int(rng, 2, 2900)
            case.update(op="append", seqs=_log_int(rng, 1, 16), q_min=_log_int(rng, 1, q), q_max=q, kv_min=q, kv_max=q + _log_int(rng, 1, 1000))
        elif kind == "token":
            hi = _log_int(rng, 64, 32768)
            case.update(op="attend", seqs=_log_int(rng, 1, 128), q_min=1, q_max=1, kv_min=_log_int(rng, 1, hi), kv_max=hi)
        elif kind == "prompt":
            q = _log_int(rng, 2, 8191 if act == "bf16" else 700)
            case.update(op="attend", seqs=_log_int(rng, 1, 8), q_min=_log_int(rng, 1, q), q_max=q, kv_min=q, kv_max=q + _log_int(rng, 1, 1200))
        elif kind == "prefix":
            case.update(op="prefix", seqs=_log_int(rng, 2, 128), q_min=1, q_max=1, kv_min=1, kv_max=_log_int(rng, 2, 1000),
                        prefix=_log_int(rng, 100, 8192 if act == "bf16" else 1003))
        else:
            q = _log_int(rng, 2, 150)
            case.update(op="prefix", seqs=_log_int(rng, 2, 24), q_min=_log_int(rng, 1, q), q_max=q, kv_min=q, kv_max=q,
                        prefix=_log_int(rng, 100, 1003))
        # a drawn case costs no more than the largest listed one; its cache and its plain form fit the card
        cells = _cells(largest["append_prompts_bf16" if case["op"] == "append" else "tokens_long_bf16"])
        if _cost(case) <= most and _cells(case) <= cells and _scores(case) <= _scores(largest["prompt_long_bf16"]):
            return case


# ------------------------------------------------------------------ the shapes of a case

def _lens(case):
    """(new tokens, cached keys with them) of each sequence: spread over the case's ranges, the first at their top."""
    rng = random.Random(case["mix"])
    out = []
    for b in range(case["seqs"]):
        q = case["q_max"] if b == 0 else rng.randint(case["q_min"], case["q_max"])
        kv = case["kv_max"] if b == 0 else rng.randint(case["kv_min"], case["kv_max"])
        out.append((q, max(kv, q)))
    return out


def _pages(case):
    """Pages of each sequence, then those of the shared prefix."""
    p = case["page"]
    return [-(-kv // p) for _, kv in _lens(case)], -(-case.get("prefix", 0) // p)


def _cells(case):
    own_pages, shared = _pages(case)
    _, kvh, hd = GEOM[case["geom"]]
    return (sum(own_pages) + shared) * case["page"] * kvh * hd


def _scores(case):
    """Scores that the plain form holds at once."""
    h = GEOM[case["geom"]][0]
    return h * max(q * (kv + case.get("prefix", 0)) for q, kv in _lens(case)) if case["q_max"] > 1 else \
        h * case["seqs"] * max(kv for _, kv in _lens(case)) + h * case["seqs"] * case.get("prefix", 0)


def _size(kind):
    return 4 if kind == "f32" else 2


def work(case):
    h, kvh, hd = GEOM[case["geom"]]
    lens = _lens(case)
    tokens = sum(q for q, _ in lens)
    sa, sc = _size(case["act"]), _size(case["cache"])
    if case["op"] == "append":
        # the projection read, q and the K and V rows written, a row of the rotation table for each token
        nbytes = tokens * ((2 * h + 2 * kvh) * hd * sa + 2 * kvh * hd * sc + hd * 4)
        return {"bytes": nbytes, "flops": tokens * (h + kvh) * hd * 8}
    keys = sum(kv for _, kv in lens) + case.get("prefix", 0)          # each key and value once
    pairs = sum(q * kv - q * (q - 1) // 2 + q * case.get("prefix", 0) for q, kv in lens)  # scores not masked
    return {"bytes": 2 * tokens * h * hd * sa + 2 * keys * kvh * hd * sc, "flops": 4 * pairs * h * hd}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


# ------------------------------------------------------------------ inputs

def _dtype(kind):
    return torch.float32 if kind == "f32" else torch.bfloat16


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        import vox_b200

        st["cache"] = vox_b200.PagedKV(st["k"], st["v"])  # the handle that a serving program keeps
    return st


def _inputs(case, seed):
    h, kvh, hd = GEOM[case["geom"]]
    lens = _lens(case)
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    host = random.Random(seed * 7919 + 5)

    def normal(shape, std, dtype, mean=0.0):
        t = torch.empty(shape, dtype=torch.float32, device=DEV)
        return t.normal_(mean, std, generator=g).to(dtype)

    own_pages, shared = _pages(case)
    total = sum(own_pages) + shared + 3                      # a few pages of the pool belong to nobody
    order = list(range(total))
    host.shuffle(order)                                      # pages lie where the pool had room
    width = max(own_pages) + 1
    table = torch.zeros((len(lens), width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(own_pages):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    tokens = sum(q for q, _ in lens)
    st = {"case": case, "tokens": tokens, "lens": lens, "h": h, "kvh": kvh, "hd": hd, "max_q": max(q for q, _ in lens),
          "max_kv": max(kv for _, kv in lens), "table": table.to(DEV),
          "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)}
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    # one token to each sequence needs no offsets
    st["q_start"] = None if case["q_max"] == 1 else torch.tensor(starts, dtype=torch.int32, device=DEV)
    ca, ac = _dtype(case["cache"]), _dtype(case["act"])
    # head-normalised keys with a gain, so that the scores spread as a trained model's do
    st["k"] = normal((total, case["page"], kvh, hd), 1.5, ca)
    st["v"] = normal((total, case["page"], kvh, hd), 1.0, ca)
    if case["op"] == "append":
        st["qkv"] = normal((tokens, (h + 2 * kvh) * hd), 2.0, ac)
        st["qn"], st["kn"] = normal((hd,), 0.1, torch.float32, 1.5), normal((hd,), 0.1, torch.float32, 1.5)
        inv = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float32, device=DEV)
        f = torch.arange(st["max_kv"], dtype=torch.float32, device=DEV)[:, None] * inv[None, :]
        st["cs"] = torch.stack((f.cos(), f.sin()), dim=2).contiguous()   # [positions][hd/2][2]
    else:
        st["q"] = normal((tokens, h, hd), 1.5, ac)
    if shared:
        st["prefix_pages"] = torch.tensor(order[at:at + shared], dtype=torch.int32, device=DEV)
    # where each new token stands: its sequence and its position in it
    st["seq_of"] = torch.tensor([b for b, (q, _) in enumerate(lens) for _ in range(q)], dtype=torch.int64, device=DEV)
    st["pos_of"] = torch.tensor([kv - q + i for q, kv in lens for i in range(q)], dtype=torch.int64, device=DEV)
    return st


# ------------------------------------------------------------------ one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    c, kv = s["case"], s["cache"]
    if c["op"] == "append":
        q = kv.append(s["qkv"], s["cs"], s["table"], s["kv_len"], s["h"], q_start=s["q_start"], q_norm_w=s["qn"], k_norm_w=s["kn"], eps=EPS)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "attend":
        return kv.attend(s["q"], s["table"], s["kv_len"], q_start=s["q_start"], max_q=s["max_q"], max_kv=s["max_kv"])
    return kv.attend_prefix(s["q"], s["prefix_pages"], c["prefix"], s["table"], s["kv_len"], q_start=s["q_start"], max_q=s["max_q"],
                            max_kv=s["max_kv"])


def _run_plain(s):
    c = s["case"]
    if c["op"] == "append":
        return _plain_append(s)
    return _plain_prompts(s) if c["q_max"] > 1 else _plain_tokens(s)


def _plain_append(s):
    c, h, kvh, hd = s["case"], s["h"], s["kvh"], s["hd"]
    x = s["qkv"].float().view(s["tokens"], h + 2 * kvh, hd)
    cs = s["cs"][s["pos_of"]]
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]

    def norm_rotate(t, w):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * w
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        return torch.cat((a * co - b * si, b * co + a * si), dim=-1)

    q = norm_rotate(x[:, :h], s["qn"]).reshape(s["tokens"], h * hd).to(s["qkv"].dtype)
    page = s["table"][s["seq_of"], s["pos_of"] // c["page"]].long()
    row = s["pos_of"] % c["page"]
    s["k"][page, row] = norm_rotate(x[:, h:h + kvh], s["kn"]).to(s["k"].dtype)
    s["v"][page, row] = x[:, h + kvh:].to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _rows(cache, pages, n):
    """The first n rows behind a list of pages, in 32 bits: [n][kv heads][hd]."""
    t = cache[pages.long()]
    return t.reshape(-1, *t.shape[-2:])[:n].float()


def _plain_prompts(s):
    h, kvh, hd = s["h"], s["kvh"], s["hd"]
    out, at, shared = [], 0, s["case"].get("prefix", 0)
    for b, (n, kv) in enumerate(s["lens"]):
        k, v = _rows(s["k"], s["table"][b], kv), _rows(s["v"], s["table"][b], kv)
        if shared:  # the prefix stands in front of the sequence's own keys
            k = torch.cat((_rows(s["k"], s["prefix_pages"], shared), k))
            v = torch.cat((_rows(s["v"], s["prefix_pages"], shared), v))
        q = s["q"][at:at + n].float().view(n, kvh, h // kvh, hd)
        x = torch.matmul(q.permute(1, 2, 0, 3).reshape(kvh, -1, hd), k.permute(1, 2, 0)) * (1.0 / math.sqrt(hd))
        x = x.view(kvh, h // kvh, n, shared + kv)
        hidden = torch.arange(shared + kv, device=DEV)[None, :] > shared + s["pos_of"][at:at + n, None]
        x = x.masked_fill(hidden, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(x.view(kvh, -1, shared + kv), v.permute(1, 0, 2)).view(kvh, h // kvh, n, hd) / x.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).reshape(n, h, hd).to(s["q"].dtype))
        at += n
    return torch.cat(out)


def _plain_tokens(s):
    """One token a sequence: the batch padded to its longest, and the shared prefix, where there is one, in front."""
    c, h, kvh, hd, b = s["case"], s["h"], s["kvh"], s["hd"], len(s["lens"])
    n = -(-s["max_kv"] // c["page"])
    q = s["q"].float().view(b, kvh, h // kvh, hd) * (1.0 / math.sqrt(hd))
    t = s["table"][:, :n].long()
    k = s["k"][t].view(b, -1, kvh, hd).permute(0, 2, 3, 1).float()           # [b][kv][hd][n]
    x = torch.matmul(q, k).masked_fill((torch.arange(n * c["page"], device=DEV)[None, :] >= s["kv_len"][:, None])[:, None, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    if "prefix" in c:
        pk = _rows(s["k"], s["prefix_pages"], c["prefix"]).permute(1, 2, 0)  # [kv][hd][n]
        px = torch.matmul(q.permute(1, 0, 2, 3).reshape(kvh, -1, hd), pk).view(kvh, b, h // kvh, -1).permute(1, 0, 2, 3)
        m = torch.maximum(m, px.amax(-1, keepdim=True))
    del k
    x = torch.exp(x - m)
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, s["v"][t].view(b, -1, kvh, hd).permute(0, 2, 1, 3).float())
    if "prefix" in c:
        px = torch.exp(px - m)
        total = total + px.sum(-1, keepdim=True)
        pv = _rows(s["v"], s["prefix_pages"], c["prefix"]).permute(1, 0, 2)
        o = o + torch.matmul(px.permute(1, 0, 2, 3).reshape(kvh, -1, c["prefix"]), pv).view(kvh, b, h // kvh, hd).permute(1, 0, 2, 3)
    return (o / total).reshape(b, h, hd).to(s["q"].dtype)


# ------------------------------------------------------------------ the same results in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    h, kvh, hd, page = s["h"], s["kvh"], s["hd"], case["page"]
    if case["op"] == "append":
        half = hd // 2
        heads = s["qkv"].double().unflatten(1, (h + 2 * kvh, hd))
        ang = s["cs"].double()[s["pos_of"]]                       # the table is an input
        turn = torch.complex(ang[..., 0], ang[..., 1])[:, None, :]

        def spin(x, w):
            rms = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / hd + EPS)
            x = x / rms * w.double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        flat = s["table"].cpu()[s["seq_of"].cpu(), (s["pos_of"] // page).cpu()].long() * page + (s["pos_of"] % page).cpu()
        flat = flat.to(DEV)
        k, v = s["k"].double().flatten(0, 1), s["v"].double().flatten(0, 1)
        k.index_copy_(0, flat, spin(heads[:, h:h + kvh], s["kn"]))
        v.index_copy_(0, flat, heads[:, h + kvh:])
        return {"q": spin(heads[:, :h], s["qn"]).flatten(1), "k": k.view(s["k"].shape), "v": v.view(s["v"].shape)}
    out = torch.empty((s["tokens"], h, hd), dtype=torch.float64, device=DEV)
    table, at = s["table"].cpu(), 0
    rows = lambda pages, n: (torch.as_tensor(pages).long().repeat_interleave(page) * page + torch.arange(page).repeat(len(pages)))[:n]  # noqa: E731
    front = rows(s["prefix_pages"].cpu(), case["prefix"]) if "prefix" in case else torch.empty(0, dtype=torch.int64)
    kf, vf = s["k"].flatten(0, 1), s["v"].flatten(0, 1)
    for b, (n, kv) in enumerate(s["lens"]):
        idx = torch.cat((front, rows(table[b][:-(-kv // page)], kv))).to(DEV)
        seen = torch.arange(kv - n, kv, device=DEV) + 1 + front.numel()          # keys that each token sees
        for j in range(kvh):
            kk, vv = kf[idx, j].double(), vf[idx, j].double()
            for i in range(j * (h // kvh), (j + 1) * (h // kvh)):
                for lo in range(0, n, 2048):
                    z = s["q"][at + lo:at + min(n, lo + 2048), i].double() @ kk.T / math.sqrt(hd)
                    if n > 1:
                        z = torch.where(torch.arange(idx.numel(), device=DEV) < seen[lo:lo + 2048, None], z, -math.inf)
                    out[at + lo:at + min(n, lo + 2048), i] = torch.softmax(z, dim=-1) @ vv
        at += n
    return out
