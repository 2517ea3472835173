"""The operators with which a server of the paged cache verifies drafts, searches with beams and serves windows, as cases to measure.

A case is a dict of plain values; its ``kind`` names the operator and the rest are sizes and options:

* ``tree``     attention of a tree of drafted tokens per sequence over what the pages hold of it and over the token's own
               ancestors (``ops.paged_tree_attention``);
* ``wdecode``  attention of one new token per sequence over the last ``window`` positions and the first ``sinks``
               (``ops.paged_decode_window_attention``);
* ``wchunk``   causal attention of packed new tokens, each over its last ``window`` positions and the first ``sinks``
               (``ops.paged_prompt_window_attention``);
* ``beam``     the best continuations of each request over its beams and the vocabulary (``ops.beam_select``);
* ``copy``     pages of every layer copied to other pages, as a fork of sequences needs it (``ops.paged_copy_pages``);
* ``keep``     the accepted ones of the drafted positions moved to the front, in every layer (``ops.paged_keep_positions``).

``heads`` query heads share ``kv`` key-value heads of ``dim`` values.  Lengths, trees and lists of pages go by the case alone
(``mix`` picks them), so that ``work`` can count them; the values go by the seed.  The pages of a sequence lie anywhere
in the pool, as they do after a while of serving.
"""
import math
import random

import torch

own = False  # True: the package's operators; False: their plain forms

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # the draft of one chat, 26 nodes, 7B-shaped
        {"name": "tree-fp16-1", "kind": "tree", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 1,
         "nodes": 26, "context": 1531, "mix": 1},
        # a serving batch of ragged lengths with drafts of up to 64 nodes, 70B-shaped
        {"name": "tree-bf16-24", "kind": "tree", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "page": 64, "seqs": 24,
         "nodes": 64, "context": 8192, "mix": 2},
        # one token of one sequence past its window, 7B-shaped
        {"name": "wdecode-fp16-1", "kind": "wdecode", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 1,
         "context": 5003, "window": 1024, "sinks": 4, "mix": 0},
        # a serving batch, some sequences still inside their window, 70B-shaped
        {"name": "wdecode-bf16-64", "kind": "wdecode", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "page": 32, "seqs": 64,
         "context": 16384, "window": 4096, "sinks": 4, "mix": 3},
        # chunks of prompts, 7B-shaped, a window that is no multiple of anything
        {"name": "wchunk-fp16-5", "kind": "wchunk", "dtype": "fp16", "heads": 32, "kv": 32, "dim": 128, "page": 16, "seqs": 5,
         "new": 512, "context": 4096, "window": 1000, "sinks": 5, "mix": 4},
        # the next part of a long document, 70B-shaped
        {"name": "wchunk-bf16-long", "kind": "wchunk", "dtype": "bf16", "heads": 64, "kv": 8, "dim": 128, "page": 64, "seqs": 1,
         "new": 2048, "context": 8192, "window": 4096, "sinks": 64, "mix": 0},
        # one request with four beams over a vocabulary of 32000
        {"name": "beam-fp16-1x4", "kind": "beam", "dtype": "fp16", "seqs": 1, "beams": 4, "vocab": 32000, "count": 8, "mix": 0},
        # a batch of requests with eight beams each over a large vocabulary, some of them ended
        {"name": "beam-bf16-48x8", "kind": "beam", "dtype": "bf16", "seqs": 48, "beams": 8, "vocab": 128256, "count": 16, "mix": 5},
        # the last page of one sequence copied for three more beams, 32 layers, 7B-shaped heads: three pages of 131 KB a layer and pool
        {"name": "copy-fp16-3", "kind": "copy", "dtype": "fp16", "kv": 32, "dim": 128, "page": 16, "layers": 32, "pairs": 3,
         "pool": 9, "partial": True, "mix": 6},
        # whole pages moved together, all layers of a model with grouped heads
        {"name": "copy-bf16-40", "kind": "copy", "dtype": "bf16", "kv": 8, "dim": 128, "page": 64, "layers": 32, "pairs": 40,
         "pool": 90, "partial": False, "mix": 7},
        # the accepted path of one draft, 32 layers, 7B-shaped
        {"name": "keep-fp16-1", "kind": "keep", "dtype": "fp16", "kv": 32, "dim": 128, "page": 16, "layers": 32, "seqs": 1,
         "nodes": 26, "kept": 5, "context": 100, "mix": 8},
        # a batch of drafts, 32 layers with grouped heads
        {"name": "keep-bf16-40", "kind": "keep", "dtype": "bf16", "kv": 8, "dim": 128, "page": 64, "layers": 32, "seqs": 40,
         "nodes": 64, "kept": 7, "context": 60, "mix": 9},
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    """One more case of the same ranges: any operator, type and head layout, sizes over their logarithm."""
    kind = rng.choice(("tree", "tree", "wdecode", "wchunk", "beam", "copy", "keep"))
    c = {"kind": kind, "dtype": rng.choice(("fp16", "bf16")), "mix": rng.randrange(1, 1 << 20)}
    if kind == "beam":
        c["dtype"] = rng.choice(("fp16", "bf16", "fp32"))
        c["vocab"] = _log(rng, 1000, 160000)
        c["beams"] = _log(rng, 1, 16)
        c["count"] = rng.choice((c["beams"], 2 * c["beams"], 2 * c["beams"]))
        c["seqs"] = _log(rng, 1, max(1, min(64, 24_000_000 // (c["vocab"] * c["beams"]))))
        return c
    group, c["kv"] = rng.choice(((1, 32), (1, 8), (2, 8), (3, 5), (4, 8), (4, 2), (5, 8), (7, 4), (8, 8), (8, 1), (16, 2)))
    c["dim"], c["page"] = rng.choice((64, 128, 128, 256)), rng.choice((8, 16, 32, 64, 128))
    if kind in ("copy", "keep"):
        c["layers"] = _log(rng, 1, 80)
        position = c["kv"] * c["dim"] * c["layers"] * 4
        if kind == "copy":
            most = max(1, min(64, 200_000_000 // (position * c["page"])))
            c["pairs"] = _log(rng, 1, most)
            c["pool"], c["partial"] = 2 * c["pairs"] + rng.randrange(1, 9), rng.random() < 0.5
        else:
            c["nodes"] = _log(rng, 2, 128)
            c["kept"] = rng.randint(1, min(8, c["nodes"]))
            c["context"] = _log(rng, 1, 100)
            c["seqs"] = _log(rng, 1, max(1, min(64, 400_000_000 // (position * (c["nodes"] + c["context"] + 2 * c["page"])))))
        return c
    c["heads"] = group * c["kv"]
    if kind == "wdecode":
        c["seqs"] = _log(rng, 1, 128)
        c["context"] = _log(rng, 1, max(64, min(32768, (1 << 28) // (c["seqs"] * c["kv"] * c["dim"]))))
    elif kind == "tree":
        c["nodes"] = _log(rng, 1, 128)
        c["seqs"] = _log(rng, 1, 32)
        most = min(200_000_000 // (c["kv"] * c["dim"]), 800_000_000 // (c["nodes"] * c["heads"])) // c["seqs"]
        c["context"] = _log(rng, 1, max(64, min(16384, most)))
    else:
        c["seqs"] = _log(rng, 1, 8)
        c["new"] = _log(rng, 1, max(1, min(1024, (1 << 23) // (c["heads"] * c["dim"])) // c["seqs"]))
        c["context"] = _log(rng, 1, 4096)
    if kind != "tree":
        c["window"], c["sinks"] = _log(rng, 1, 8192), rng.choice((0, 0, 1, 4, 4, 64, 100))
    return c


# ---------------------------------------------------------------- lengths and inputs
def _lengths(case):
    """(new tokens, tokens of context) of each sequence.  The first has the largest of both; ``mix`` 0: so have the
    others; else they lie anywhere below, a few at nothing or one."""
    rng, n, mix = random.Random(case["mix"]), case["seqs"], case["mix"]
    most_new, most_ctx = case.get("new", case.get("nodes", 1)), case["context"]

    def pick(most):
        return min(most, rng.choice((0, 1, most, *(rng.randint(0, most) for _ in range(12)))))

    news = [most_new if i == 0 or not mix or most_new == 1 else pick(most_new) for i in range(n)]
    ctxs = [most_ctx if i == 0 or not mix else pick(most_ctx) for i in range(n)]
    return news, ctxs


def _totals(case):
    """Positions that each sequence has in the cache once its new tokens are there."""
    news, ctxs = _lengths(case)
    return ctxs if case["kind"] == "wdecode" else [a + b for a, b in zip(news, ctxs)]


def _trees(case):
    """Of each sequence the nodes' parents: node 0 is the last token that was taken, the others follow any earlier node, late
    ones more often, as drafts grow level by level."""
    rng = random.Random(case["mix"] + 1)
    trees = []
    for n in _lengths(case)[0]:
        trees.append([-1] + [rng.randrange(i // 3, i) if rng.random() < 0.7 else rng.randrange(0, i) for i in range(1, n)])
    return [t[:n] for t, n in zip(trees, _lengths(case)[0])]


def _ancestors(parents):
    """Of each node the set of itself and its ancestors, as the bits of a whole number."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return seen


def _kept(case):
    """Of each sequence the nodes that were accepted, ascending.  Their new places hold no other node that is accepted (those
    that stay apart), so that a pass over the same cache gives the same again."""
    rng = random.Random(case["mix"] + 2)
    kept = []
    for n in _lengths(case)[0]:
        count = min(n, rng.randint(1, case["kept"])) if kept else min(n, case["kept"])
        stay = rng.randint(0, count)
        rest = list(range(count, n))
        moved = sorted(rng.sample(rest, min(len(rest), count - stay)))
        kept.append(list(range(count - len(moved))) + moved)
    return kept


def _pairs(case):
    """(source, destination, positions in use) of each copy: any pages, a source may serve several."""
    rng = random.Random(case["mix"] + 3)
    pages = list(range(case["pool"]))
    rng.shuffle(pages)
    dst, sources = pages[:case["pairs"]], pages[case["pairs"]:]
    src = [rng.choice(sources) for _ in dst]
    return src, dst, [rng.randint(1, case["page"]) if case["partial"] else case["page"] for _ in dst]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(case, gen, layers=()):
    """The cache of one layer or all: pools of pages ``[layers, pages, kv, page, dim]``, a table of each sequence's pages in
    order, and the lengths.  The table is as wide as the longest sequence may grow."""
    page, totals, dt = case["page"], _totals(case), DTYPES[case["dtype"]]
    width = -(-max(max(totals), 1) // page) + 1
    need = [-(-t // page) for t in totals]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    at = torch.tensor([0, *need], device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    used = col < _ints(need).unsqueeze(1)
    table = torch.where(used, order[(at[:-1].unsqueeze(1) + col).clamp(max=pool - 1)], 0).contiguous()
    shape = (*layers, pool, case["kv"], page, case["dim"])
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

    if kind == "beam":
        rows, vocab = case["seqs"] * case["beams"], case["vocab"]
        # a bell of unlikely tokens and a tail of a few that stand out, as a language model's logits are
        x = 1.7 * randn(rows, vocab, dtype=torch.float32)
        stand = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
        x.scatter_add_(1, stand, 8.0 + 2.5 * randn(rows, 12, dtype=torch.float32))
        s["logits"] = x.to(dt)
        s["scores"] = -12.0 - 3.0 * torch.rand(case["seqs"], case["beams"], generator=gen, device="cuda")
        end = torch.rand(case["seqs"], case["beams"], generator=gen, device="cuda") < 0.15
        s.update(ended=end if case["mix"] else None, count=case["count"], pad=2)
        return s
    if kind == "copy":
        shape = (case["layers"], case["pool"], case["kv"], case["page"], case["dim"])
        src, dst, filled = _pairs(case)
        s.update(k_pages=randn(*shape), v_pages=randn(*shape), src=_ints(src), dst=_ints(dst),
                 filled=_ints(filled) if case["partial"] else None)
        return s
    if kind == "keep":
        s.update(_pages(case, gen, (case["layers"],)))
        kept = _kept(case)
        s.update(first=_ints(_lengths(case)[1]), keep=_ints([i for k in kept for i in k]), starts=_ints(_starts([len(k) for k in kept])))
        return s
    heads, dim = case["heads"], case["dim"]
    news, _ = _lengths(case)
    starts = _starts(news)
    s.update(_pages(case, gen), scale=1.0 / math.sqrt(dim))
    if kind == "wdecode":
        s.update(q=1.5 * randn(case["seqs"], heads, dim), window=case["window"], sinks=case["sinks"])
        return s
    s.update(q=1.5 * randn(max(1, starts[-1]), heads, dim), starts=_ints(starts), most=max(news))
    if kind == "wchunk":
        s.update(window=case["window"], sinks=case["sinks"])
        return s
    words = -(-case["nodes"] // 64)
    seen = [a for t in _trees(case) for a in _ancestors(t)] or [0]
    low = (1 << 64) - 1
    signed = lambda x: x - (1 << 64) if x >> 63 else x  # noqa: E731
    s["masks"] = torch.tensor([[signed(a >> 64 * w & low) for w in range(words)] for a in seen], dtype=torch.int64, device="cuda")
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _operators(state)
    return {"tree": _plain_tree, "wdecode": _plain_wdecode, "wchunk": _plain_wchunk, "beam": _plain_beam, "copy": _plain_copy,
            "keep": _plain_keep}[state["kind"]](state)


def _operators(s):
    from mindpipe_amd import ops
    if s["kind"] == "tree":
        return ops.paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"], s["masks"], s["scale"])
    if s["kind"] == "wdecode":
        return ops.paged_decode_window_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"], s["window"],
                                                 s["sinks"])
    if s["kind"] == "wchunk":
        return ops.paged_prompt_window_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"], s["scale"],
                                                 s["window"], s["sinks"])
    if s["kind"] == "beam":
        return list(ops.beam_select(s["logits"], s["scores"], s["count"], s["ended"], s["pad"]))
    if s["kind"] == "copy":
        ops.paged_copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"], s["filled"])
    else:
        ops.paged_keep_positions(s["k_pages"], s["v_pages"], s["table"], s["first"], s["keep"], s["starts"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---------------------------------------------------------------- the plain forms
def _places(s, rows):
    """Of each packed token: its sequence, its place among the sequence's new tokens, and its position."""
    t = torch.arange(rows, device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, t, right=True) - 1
    return seq, t - starts[seq], s["lens"].long()[seq] - (starts[seq + 1] - t)


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


def _plain_wdecode(s):
    b, heads, dim = s["q"].shape
    k, v = _dense(s["k_pages"], s["table"]), _dense(s["v_pages"], s["table"])
    q = s["q"].float().view(b, k.shape[1], -1, dim)
    at, lens = torch.arange(k.shape[2], device="cuda"), s["lens"].view(b, 1, 1, 1)
    seen = (at < lens) & ((at < s["sinks"]) | (at >= lens - s["window"]))
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    return _softmax_times(scores, seen, v).view(b, heads, dim).to(s["q"].dtype)


def _padded(s, sees):
    """Attention of packed rows over their sequences' pages, the rows padded to the longest sequence's; ``sees`` gives what
    each of the packed rows sees of the positions."""
    t, heads, dim = s["q"].shape
    k, v = _dense(s["k_pages"], s["table"]), _dense(s["v_pages"], s["table"])
    b, kv, reach, _ = k.shape
    seq, at, pos = _places(s, t)
    most = s["most"]
    q = torch.zeros(b, most, heads, dim, device="cuda")
    q[seq, at] = s["q"].float()
    seen = torch.zeros(b, most, reach, device="cuda", dtype=torch.bool)
    seen[seq, at] = sees(seq, pos, torch.arange(reach, device="cuda"))
    q = q.view(b, most, kv, -1, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, kv, -1, most, reach) * s["scale"]
    out = _softmax_times(scores, seen.view(b, 1, 1, most, reach), v.unsqueeze(2))
    return out.permute(0, 3, 1, 2, 4).reshape(b, most, heads, dim)[seq, at].to(s["q"].dtype)


def _plain_wchunk(s):
    def sees(seq, pos, at):
        pos = pos.unsqueeze(1)
        return (at <= pos) & ((at < s["sinks"]) | (at > pos - s["window"]))
    return _padded(s, sees)


def _plain_tree(s):
    def sees(seq, pos, at):
        starts, masks = s["starts"].long(), s["masks"]
        first = (s["lens"].long() - (starts[1:] - starts[:-1]))[seq].unsqueeze(1)  # position of the sequence's node 0
        node = at - first
        bits = masks.gather(1, (node // 64).clamp(0, masks.shape[1] - 1)) >> (node % 64) & 1
        new = (node >= 0) & (at < s["lens"].long()[seq].unsqueeze(1)) & (node < 64 * masks.shape[1])
        return (node < 0) | (new & (bits == 1))
    return _padded(s, sees)


def _plain_beam(s):
    # 64 bits: a token is decided by which of two totals is larger
    x = s["logits"].double()
    batch, beams = s["scores"].shape
    top = x.amax(1, keepdim=True)
    total = s["scores"].double().view(-1, 1) + (x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True))))
    if s["ended"] is not None:
        end = s["ended"].view(-1, 1)
        pad = torch.arange(x.shape[1], device="cuda") == s["pad"]
        total = torch.where(end, torch.where(pad, s["scores"].double().view(-1, 1), -math.inf), total)
    total = total.view(batch, -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :s["count"]], at[:, :s["count"]]
    none = best == -math.inf
    return [best.float(), torch.where(none, -1, at // x.shape[1]), torch.where(none, -1, at % x.shape[1])]


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pages in (s["k_pages"], s["v_pages"]):
        if s["filled"] is None:
            pages[:, dst] = pages[:, src]
        else:
            used = torch.arange(pages.shape[3], device="cuda") < s["filled"].view(-1, 1)
            pages[:, dst] = torch.where(used.view(1, len(src), 1, -1, 1), pages[:, src], pages[:, dst])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_keep(s):
    starts, page = s["starts"].long(), s["k_pages"].shape[3]
    t = torch.arange(len(s["keep"]), device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    first = s["first"].long()[seq]
    to, of = first + t - starts[seq], first + s["keep"]
    table = s["table"].long()
    to_page, of_page = table[seq, to // page], table[seq, of // page]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[:, to_page, :, to % page] = pages[:, of_page, :, of % page]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "beam":
        rows = case["seqs"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * e + 5) + case["seqs"] * case["count"] * 20, "flops": 4 * rows * case["vocab"]}
    position = 2 * case["kv"] * case["dim"] * e  # a key and a value of every head
    if case["kind"] == "copy":
        return {"bytes": 2 * sum(_pairs(case)[2]) * case["layers"] * position, "flops": 0}
    if case["kind"] == "keep":
        moved = sum(i != j for k in _kept(case) for j, i in enumerate(k))
        return {"bytes": 2 * moved * case["layers"] * position, "flops": 0}
    heads, dim = case["heads"], case["dim"]
    news, ctxs = _lengths(case)
    totals = _totals(case)
    if case["kind"] == "wdecode":
        seen = sum(min(t, case["window"] + min(case["sinks"], max(0, t - case["window"]))) for t in totals)
        return {"bytes": 2 * case["seqs"] * heads * dim * e + seen * position, "flops": 4 * seen * heads * dim}
    tokens = sum(news)
    if case["kind"] == "tree":
        held = sum(t for n, t in zip(news, totals) if n)
        seen = sum(n * c for n, c in zip(news, ctxs)) + sum(bin(a).count("1") for t in _trees(case) for a in _ancestors(t))
        return {"bytes": 2 * tokens * heads * dim * e + held * position + 8 * tokens, "flops": 4 * seen * heads * dim}
    w, sinks = case["window"], case["sinks"]
    seen = held = 0
    for n, c in zip(news, ctxs):
        held += min(c + n, w + n - 1 + min(sinks, max(0, c + 1 - w))) if n else 0
        seen += sum(min(p + 1, w + min(sinks, max(0, p + 1 - w))) for p in range(c, c + n))
    return {"bytes": 2 * tokens * heads * dim * e + held * position, "flops": 4 * seen * heads * dim}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "beam":
        return _exact_beam(case, s)
    if case["kind"] in ("copy", "keep"):
        return _exact_moves(case, s)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    news, _ = _lengths(case)
    totals, group = _totals(case), heads // kv
    trees = [_ancestors(t) for t in _trees(case)] if case["kind"] == "tree" else None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, t) in enumerate(zip(news, totals)):
        n = 1 if case["kind"] == "wdecode" else n
        rows = slice(first, first + n)
        first += n
        if n == 0 or t == 0:
            continue
        p = torch.arange(t, device="cuda")
        if trees is not None:
            own_ = torch.tensor([[a >> j & 1 for j in range(n)] for a in trees[i]], dtype=torch.bool, device="cuda")
            seen = torch.cat((torch.ones(n, t - n, dtype=torch.bool, device="cuda"), own_), 1)
        else:
            last = p[t - n:].unsqueeze(1)
            seen = (p <= last) & ((p < case["sinks"]) | (last - p < case["window"]))
        of = s["table"][i, :-(-t // page)].long()
        k, v = (s[x][of].double().transpose(0, 1).reshape(kv, -1, dim)[:, :t] for x in ("k_pages", "v_pages"))
        for h in range(kv):
            for j in range(h * group, (h + 1) * group):
                a = (s["q"][rows, j].double() @ k[h].t()) * s["scale"]
                out[rows, j] = torch.softmax(a.masked_fill(~seen, -math.inf), -1) @ v[h]
    return out


def _exact_moves(case, s):
    """Position by position on the host's lists."""
    pages = [s[x].double() for x in ("k_pages", "v_pages")]
    if case["kind"] == "copy":
        moves = [(a, slice(0, n), b, slice(0, n)) for a, b, n in zip(*_pairs(case))]
    else:
        table, page, moves = s["table"].tolist(), case["page"], []
        for row, c, kept in zip(table, _lengths(case)[1], _kept(case)):
            for j, i in enumerate(kept):
                moves.append((row[(c + i) // page], (c + i) % page, row[(c + j) // page], (c + j) % page))
    for x in pages:
        before = x.clone()
        for a, at, b, to in moves:
            x[:, b, :, to] = before[:, a, :, at]
    return {"k_pages": pages[0], "v_pages": pages[1]}


def _exact_beam(case, s):
    """Row by row in the extended precision of the host: no more than ``count`` of a row can be among the best."""
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    if x.size > 1 << 26:
        return None
    batch, beams, count = case["seqs"], case["beams"], case["count"]
    scores = s["scores"].double().cpu().numpy()
    ended = np.zeros((batch, beams), bool) if s["ended"] is None else s["ended"].cpu().numpy()
    out = [np.full((batch, count), -np.inf), np.full((batch, count), -1), np.full((batch, count), -1)]
    for b in range(batch):
        found = []
        for k in range(beams):
            base, row = np.longdouble(scores[b, k]), x[b * beams + k]
            if ended[b, k]:
                found.append((-base, k, s["pad"]))
                continue
            lse = row.max() + np.log(np.exp(row.astype(np.longdouble) - row.max()).sum())
            least = np.partition(row, -count)[-count]
            found += [(-(base + (np.longdouble(row[v]) - lse)), k, int(v)) for v in np.flatnonzero(row >= least)]
        for i, (t, k, v) in enumerate(sorted(found)[:count]):
            out[0][b, i], out[1][b, i], out[2][b, i] = -t, k, v
    return [torch.tensor(o) for o in out]
