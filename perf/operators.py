"""The operators of a serving step over a paged key-value cache, as cases to measure.

A case is a dict of plain values; its ``kind`` names the operator and the rest are sizes and options:

* ``append``   rotation of the queries and keys of new tokens, and their keys and values into the cache's pages
               (``ops.paged_rope_append``);
* ``decode``   attention of one new token per sequence over the pages (``ops.paged_decode_attention``);
* ``prompt``   causal attention of packed prompts (``ops.prompt_attention``);
* ``chunk``    causal attention of packed new tokens over what the pages hold of their sequences, the new tokens included
               (``ops.paged_prompt_attention``);
* ``sample``   tokens from logits with temperature, top-k, top-p and min-p at given random numbers (``ops.sample_tokens``).

``heads`` query heads share ``kv`` key-value heads of ``dim`` values.  A sequence's lengths go by the case alone
(``mix`` picks them between nothing and ``context``, ``new``), so that ``work`` can count them; the values go by the seed.
The pages of a sequence lie anywhere in the pool, as they do after a while of serving.
"""
import math
import random

import torch

own = False  # True: the package's operators; False: their plain forms

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # one token of one sequence, 32 heads of their own: the smallest call, latency alone
        {"name": "append-fp16-1", "kind": "append", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 1,
         "new": 1, "context": 512, "mix": 0, "rotary": 128, "pairs": True},
        # prompts of different lengths behind contexts of their own, 70B-shaped heads, rotated by halves
        {"name": "append-bf16-prompts", "kind": "append", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "page": 32, "seqs": 7,
         "new": 2341, "context": 4096, "mix": 3, "rotary": 128, "pairs": False},
        # one sequence early in its answer, 7B-shaped
        {"name": "decode-fp16-1", "kind": "decode", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 1,
         "context": 577, "mix": 0},
        # a serving batch of ragged lengths, 70B-shaped
        {"name": "decode-bf16-64", "kind": "decode", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "page": 16, "seqs": 64,
         "context": 8192, "mix": 1},
        # two long documents: few rows, so the length has to be split
        {"name": "decode-fp16-long", "kind": "decode", "dtype": "fp16", "heads": 64, "kv": 8, "dim": 128, "page": 64, "seqs": 2,
         "context": 131071, "mix": 0},
        # many short chats with small heads, seven queries to a key
        {"name": "decode-bf16-200", "kind": "decode", "dtype": "bf16", "heads": 14, "kv": 2, "dim": 64, "page": 32, "seqs": 200,
         "context": 1500, "mix": 2},
        # one short prompt, 7B-shaped
        {"name": "prompt-fp16-129", "kind": "prompt", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "seqs": 1, "new": 129,
         "mix": 0},
        # packed prompts, 70B-shaped
        {"name": "prompt-bf16-packed", "kind": "prompt", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "seqs": 3, "new": 4096,
         "mix": 4},
        # new chunks behind long contexts, as a server mixes them, 7B-shaped
        {"name": "chunk-fp16-5", "kind": "chunk", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 5,
         "new": 512, "context": 4096, "mix": 5},
        # wide heads, four queries to a key
        {"name": "chunk-bf16-wide", "kind": "chunk", "dtype": "bf16", "heads": 16, "kv": 4, "dim": 256, "page": 32, "seqs": 2,
         "new": 1024, "context": 2048, "mix": 6},
        # one row of a 32000-token vocabulary, every filter at work
        {"name": "sample-fp16-1", "kind": "sample", "dtype": "fp16", "seqs": 1, "vocab": 32000, "filters": "kpm"},
        # a batch over a large vocabulary, each row with its request's own settings, some of them off
        {"name": "sample-bf16-256", "kind": "sample", "dtype": "bf16", "seqs": 256, "vocab": 128256, "filters": "mixed"},
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    """One more case of the same ranges: any operator, type and head layout, sizes over their logarithm."""
    kind = rng.choice(("append", "decode", "prompt", "chunk", "sample"))
    c = {"kind": kind, "dtype": rng.choice(("fp16", "bf16"))}
    if kind == "sample":
        c["dtype"] = rng.choice(("fp16", "bf16", "fp32"))
        c["vocab"] = _log(rng, 1000, 160000)
        c["seqs"] = _log(rng, 1, max(1, min(256, 16_000_000 // c["vocab"])))
        c["filters"] = rng.choice(("", "k", "p", "m", "kp", "kpm", "mixed"))
        return c
    group, c["kv"] = rng.choice(((1, 32), (1, 8), (2, 8), (3, 5), (4, 8), (4, 2), (5, 8), (7, 4), (8, 8), (8, 1), (16, 2)))
    c["heads"] = group * c["kv"]
    c["dim"] = rng.choice((64, 128, 128, 256))
    c["mix"] = rng.randrange(1 << 20)
    if kind == "decode":
        c["seqs"] = _log(rng, 1, 256)
        c["context"] = _log(rng, 1, max(64, min(65536, (1 << 28) // (c["seqs"] * c["kv"] * c["dim"]))))
    elif kind == "append":
        c["seqs"] = _log(rng, 1, 64)
        c["new"] = rng.choice((1, _log(rng, 1, max(1, 8192 // c["seqs"]))))
        c["context"] = _log(rng, 1, max(64, min(16384, (1 << 27) // (c["seqs"] * c["kv"] * c["dim"]))))
        c["rotary"] = rng.choice((c["dim"], c["dim"], c["dim"] // 2))
        c["pairs"] = rng.random() < 0.5
    elif kind == "prompt":
        c["seqs"] = _log(rng, 1, 16)
        c["new"] = _log(rng, 1, 4096 // c["seqs"])
    else:
        c["seqs"] = _log(rng, 1, 8)
        c["new"] = _log(rng, 1, 1024 // c["seqs"])
        c["context"] = _log(rng, 1, 4096)
    if kind != "prompt":
        c["page"] = rng.choice((8, 16, 32, 64, 128))
    return c


# ---------------------------------------------------------------- lengths and inputs
def _lengths(case):
    """(new tokens, tokens of context) of each sequence.  The first has the largest of both; ``mix`` 0: so have the
    others; else they lie anywhere below, a few at nothing or one."""
    rng, n, mix = random.Random(case["mix"]), case["seqs"], case["mix"]
    most_new, most_ctx = case.get("new", 1), case.get("context", 0)

    def pick(most, least):
        return max(least, min(most, rng.choice((0, 1, most, *(rng.randint(0, most) for _ in range(12))))))

    news = [most_new if i == 0 or not mix or most_new == 1 else pick(most_new, 0) for i in range(n)]
    ctxs = [most_ctx if i == 0 or not mix else pick(most_ctx, 0) for i in range(n)]
    return news, ctxs


def _totals(case):
    """Positions that each sequence has in the cache once its new tokens are there."""
    news, ctxs = _lengths(case)
    return ctxs if case["kind"] == "decode" else [a + b for a, b in zip(news, ctxs)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(case, gen):
    """The cache of one layer: pools of pages ``[pages, kv, page, dim]``, a table of each sequence's pages in order, and the
    lengths.  The table is as wide as the longest sequence may grow."""
    page, totals, dt = case["page"], _totals(case), DTYPES[case["dtype"]]
    width = -(-max(max(totals), 1) // page) + 1
    need = [-(-t // page) for t in totals]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    at = torch.tensor([0, *need], device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    used = col < _ints(need).unsqueeze(1)
    table = torch.where(used, order[(at[:-1].unsqueeze(1) + col).clamp(max=pool - 1)], 0).contiguous()
    shape = (pool, case["kv"], page, case["dim"])
    return {"k_pages": torch.randn(shape, generator=gen, device="cuda", dtype=dt),
            "v_pages": torch.randn(shape, generator=gen, device="cuda", dtype=dt), "table": table, "lens": _ints(totals)}


def _starts(news):
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"kind": kind}

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if kind == "sample":
        rows, vocab, f = case["seqs"], case["vocab"], case["filters"]
        # a bell of unlikely tokens and a tail of a few that stand out, as a language model's logits are
        x = 1.7 * randn(rows, vocab, dtype=torch.float32)
        stand = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
        x.scatter_add_(1, stand, 8.0 + 2.5 * randn(rows, 12, dtype=torch.float32))
        s["logits"] = x.to(dt)
        s["u"] = torch.rand(rows, generator=gen, device="cuda")
        rand = torch.rand(4, rows, generator=gen, device="cuda")
        off = torch.rand(4, rows, generator=gen, device="cuda") < (0.3 if f == "mixed" else 0.0)
        s["temperature"] = torch.where(off[0], 0.0, 0.5 + rand[0])
        top_k = (10 ** (0.5 + 2.0 * rand[1])).to(torch.int32)
        s["top_k"] = torch.where(off[1], 0, top_k) if "k" in f or f == "mixed" else None
        s["top_p"] = torch.where(off[2], 1.0, 0.7 + 0.29 * rand[2]) if "p" in f or f == "mixed" else None
        s["min_p"] = torch.where(off[3], 0.0, 0.15 * rand[3]) if f in ("m", "kpm", "mixed") else None
        return s
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    s["scale"] = 1.0 / math.sqrt(dim)
    news, _ = _lengths(case)
    starts = _starts(news)
    if kind == "prompt":
        # the fused projection's rows: queries, keys and values are views of them
        qkv = randn(max(1, starts[-1]), heads + 2 * kv, dim)
        s.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv], v=qkv[:, heads + kv:], starts=_ints(starts))
        return s
    s.update(_pages(case, gen))
    if kind == "decode":
        s["q"] = 1.5 * randn(case["seqs"], heads, dim)
        return s
    s["starts"] = _ints(starts)
    if kind == "chunk":
        s["q"] = 1.5 * randn(max(1, starts[-1]), heads, dim)
        return s
    s["qkv"] = randn(max(1, starts[-1]), (heads + 2 * kv) * dim)
    half, reach = case["rotary"] // 2, case["page"] * s["table"].shape[1]
    # angles of far positions need 64 bits
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(reach, device="cuda", dtype=torch.float64).unsqueeze(1) * freq
    s.update(cos=angle.cos().float(), sin=angle.sin().float(), pairs=case["pairs"])
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _operators(state)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "chunk": _plain_chunk,
            "sample": _plain_sample}[state["kind"]](state)


def _operators(s):
    from mindpipe_amd import ops
    if s["kind"] == "append":
        q = ops.paged_rope_append(s["qkv"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"],
                                  s["pairs"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["kind"] == "decode":
        return ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"])
    if s["kind"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["starts"], s["scale"])
    if s["kind"] == "chunk":
        return ops.paged_prompt_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"], s["scale"])
    return list(ops.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"]))


# ---------------------------------------------------------------- the plain forms
def _places(s, rows):
    """Of each packed token: its sequence, and its position in it."""
    t = torch.arange(rows, device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, t, right=True) - 1
    return seq, s["lens"].long()[seq] - (starts[seq + 1] - t)


def _plain_append(s):
    kv, page, dim = s["k_pages"].shape[1:]
    rows = s["qkv"].shape[0]
    x = s["qkv"].view(rows, -1, dim)
    heads = x.shape[1] - 2 * kv
    seq, pos = _places(s, rows)
    cos, sin, f = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1), x[:, :heads + kv].float()
    half = s["cos"].shape[1]
    if s["pairs"]:
        a, b = f[..., 0:2 * half:2], f[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = f[..., :half], f[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    turned = torch.cat((turned, f[..., 2 * half:]), -1).to(x.dtype)
    at, row = s["table"].long()[seq, pos // page], pos % page
    s["k_pages"][at, :, row] = turned[:, heads:]
    s["v_pages"][at, :, row] = x[:, heads + kv:]
    return {"q": turned[:, :heads].contiguous(), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _dense(pages, table):
    """The pages in each sequence's order, in 32 bits: ``[seqs, kv, positions, dim]``."""
    b, w = table.shape
    _, kv, page, dim = pages.shape
    return pages[table.long()].float().transpose(1, 2).reshape(b, kv, w * page, dim)


def _softmax_times(scores, seen, v):
    """softmax over the last axis where ``seen``, times v; nothing seen: zeros."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(e, v) / total, 0.0)


def _plain_decode(s):
    b, heads, dim = s["q"].shape
    k, v = _dense(s["k_pages"], s["table"]), _dense(s["v_pages"], s["table"])
    q = s["q"].float().view(b, k.shape[1], -1, dim)
    seen = torch.arange(k.shape[2], device="cuda") < s["lens"].view(b, 1, 1, 1)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    return _softmax_times(scores, seen, v).view(b, heads, dim).to(s["q"].dtype)


def _plain_prompt(s):
    t, heads, dim = s["q"].shape
    kv = s["k"].shape[1]
    q = s["q"].float().view(t, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
    k, v = s["k"].float().permute(1, 2, 0).contiguous(), s["v"].float().transpose(0, 1).contiguous()
    at = torch.arange(t, device="cuda")
    seq = torch.searchsorted(s["starts"], at.int(), right=True)
    seen = (seq.unsqueeze(1) == seq) & (at <= at.unsqueeze(1))
    scores = torch.matmul(q, k).view(kv, heads // kv, t, t) * s["scale"]
    out = _softmax_times(scores, seen, v.unsqueeze(1))
    return out.permute(2, 0, 1, 3).reshape(t, heads, dim).to(s["q"].dtype)


def _plain_chunk(s):
    t, heads, dim = s["q"].shape
    k, v = _dense(s["k_pages"], s["table"]), _dense(s["v_pages"], s["table"])
    b, kv, reach, _ = k.shape
    starts = s["starts"].long()
    seq, pos = _places(s, t)
    at = torch.arange(t, device="cuda") - starts[seq]
    q = torch.zeros(b, t, heads, dim, device="cuda")
    q[seq, at] = s["q"].float()
    last = torch.full((b, t), -1, device="cuda")
    last[seq, at] = pos
    most = min(t, reach)  # no sequence has more new tokens than the table holds
    q, last = q[:, :most].view(b, most, kv, -1, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim), last[:, :most]
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, kv, -1, most, reach) * s["scale"]
    seen = torch.arange(reach, device="cuda") <= last.view(b, 1, 1, most, 1)
    out = _softmax_times(scores, seen, v.unsqueeze(2))
    return out.permute(0, 3, 1, 2, 4).reshape(b, most, heads, dim)[seq, at].to(s["q"].dtype)


def _plain_sample(s):
    # 64 bits: a token is decided by which side of a border a long sum falls on
    x = s["logits"].double()
    rows, vocab = x.shape
    temperature = s["temperature"].double().unsqueeze(1)
    greedy = ~(temperature > 0)
    top = x.amax(1, keepdim=True)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, temperature)))
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ranked = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    keep = torch.ones_like(ranked, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].unsqueeze(1)
        keep &= (k <= 0) | (rank < k)
    if s["top_p"] is not None:
        p = s["top_p"].double().unsqueeze(1)
        sums = torch.where(keep, ranked, 0.0).cumsum(1)
        keep &= (p >= 1) | (sums - ranked < p * sums[:, -1:]) | (rank == 0)
    if s["min_p"] is not None:
        keep &= (ranked >= s["min_p"].double().unsqueeze(1)) | (rank == 0)
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, ranked, 0.0))
    sums = w.cumsum(1)
    total = sums[:, -1:]
    token = (sums <= s["u"].double().unsqueeze(1) * total).sum(1).clamp(max=vocab - 1)
    token = torch.where(greedy.squeeze(1), order[:, 0], token)
    chance = torch.log(w.gather(1, token.unsqueeze(1)) / total).squeeze(1)
    return [token, torch.where(greedy.squeeze(1), 0.0, chance).float()]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "sample":
        rows = case["seqs"]
        return {"bytes": rows * case["vocab"] * e + rows * (5 * 4 + 8 + 4), "flops": 6 * rows * case["vocab"]}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    news, _ = _lengths(case)
    totals, tokens = _totals(case), sum(news)
    if case["kind"] == "append":
        rotated = 4 * case["rotary"]  # a cosine and a sine in 32 bits for each pair
        return {"bytes": tokens * (2 * (heads + 2 * kv) * dim * e + rotated), "flops": tokens * (heads + kv) * case["rotary"] * 3}
    if case["kind"] == "decode":
        return {"bytes": 2 * case["seqs"] * heads * dim * e + 2 * sum(totals) * kv * dim * e,
                "flops": 4 * sum(totals) * heads * dim}
    seen = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(news, totals))
    held = sum(t for n, t in zip(news, totals) if n)
    return {"bytes": 2 * tokens * heads * dim * e + 2 * held * kv * dim * e, "flops": 4 * seen * heads * dim}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    news, _ = _lengths(case)
    totals, paged = _totals(case), case["kind"] != "prompt"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, t) in enumerate(zip(news, totals)):
        n = 1 if case["kind"] == "decode" else n
        rows = slice(first, first + n)
        first += n
        if n == 0 or t == 0:
            continue
        last = torch.arange(t - n, t, device="cuda").unsqueeze(1)
        hidden = torch.arange(t, device="cuda") > last
        for h in range(kv):
            if paged:
                of = s["table"][i, :-(-t // case["page"])].long()
                k, v = (s[p][of, h].reshape(-1, dim)[:t].double() for p in ("k_pages", "v_pages"))
            else:
                k, v = s["k"][rows, h].double(), s["v"][rows, h].double()
            for j in range(h * (heads // kv), (h + 1) * (heads // kv)):
                a = (s["q"][rows, j].double() @ k.t()) * s["scale"]
                out[rows, j] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v
    return out


def _exact_append(case, s):
    heads, kv, page = case["heads"], case["kv"], case["page"]
    news, ctxs = _lengths(case)
    x = s["qkv"].double().view(s["qkv"].shape[0], -1, case["dim"])
    pos = torch.tensor([c + j for n, c in zip(news, ctxs) for j in range(n)], device="cuda")
    seq = torch.tensor([i for i, n in enumerate(news) for _ in range(n)], device="cuda")
    half = case["rotary"] // 2
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos].unsqueeze(1)
    part = x[:, :heads + kv, :2 * half]
    z = torch.view_as_complex(part.unflatten(-1, (half, 2)) if s["pairs"] else
                              part.unflatten(-1, (2, half)).transpose(-1, -2).contiguous()) * turn
    z = torch.view_as_real(z)
    y = x.clone()
    y[:, :heads + kv, :2 * half] = (z if s["pairs"] else z.transpose(-1, -2)).flatten(-2)
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    flat = s["table"].long()[seq, pos // page] * page + pos % page
    for pages, rows in ((k_pages, y[:, heads:heads + kv]), (v_pages, y[:, heads + kv:])):
        pages.copy_(pages.transpose(1, 2).flatten(0, 1).index_copy(0, flat, rows).unflatten(0, (-1, page)).transpose(1, 2))
    return {"q": y[:, :heads], "k_pages": k_pages, "v_pages": v_pages}


def _exact_sample(s):
    """Row by row, on the values from the largest down, in the extended precision of the host."""
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    if x.size > 1 << 26:
        return None
    get = lambda k, none: np.full(len(x), none) if s[k] is None else s[k].double().cpu().numpy()  # noqa: E731
    u, t, ks, ps, ms = get("u", 0), get("temperature", 1), get("top_k", 0), get("top_p", 1), get("min_p", 0)
    tokens, chances = [], []
    for row, u_, t_, k_, p_, m_ in zip(x, u, t, ks, ps, ms):
        if not t_ > 0:
            tokens.append(int(row.argmax()))
            chances.append(0.0)
            continue
        by = np.argsort(-row, kind="stable")
        by = by[:int(k_)] if k_ > 0 else by
        w = np.exp((row[by].astype(np.longdouble) - row[by[0]]) / np.longdouble(t_))
        if p_ < 1:
            reached = np.cumsum(w) >= np.longdouble(p_) * w.sum()
            n = int(reached.argmax()) + 1
            by, w = by[:n], w[:n]
        fine = w >= m_
        fine[0] = True
        by, w = by[fine], w[fine]
        at = np.argsort(by)
        by, w = by[at], w[at]
        sums = np.cumsum(w)
        n = min(int(np.searchsorted(sums, np.longdouble(u_) * sums[-1], side="right")), len(by) - 1)
        tokens.append(int(by[n]))
        chances.append(float(np.log(w[n] / sums[-1])))
    return [torch.tensor(tokens), torch.tensor(chances, dtype=torch.float64)]
