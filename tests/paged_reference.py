"""Plain 64-bit forms of the paged-cache operators and of sampling, on the CPU, and the bounds their kernels are held to."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attention_row(q, k, v, scale):
    """(output, bound of |kernel - output|) of one query over the positions it sees, q [dim], k / v [n, dim] in 64 bits.

    The kernel's scores are fp32 sums of dim products and a scaling: off by at most (dim + 2) 2^-24 sum |q k| scale, a
    relative error of the weights; the exponential adds less than 2^-21.  Weights and outputs are rounded to the type
    (half a step each), fp16 weights below its normal numbers by 2^-32 of the largest.  Sums of n fp32 terms and the joins
    of their parts are off by at most (n + 64) 2^-24 of the sum of magnitudes, numerator and denominator alike."""
    n, dim = k.shape
    if n == 0:
        return torch.zeros(v.shape[1], dtype=torch.float64), torch.zeros(v.shape[1], dtype=torch.float64)
    s = (k @ q) * scale
    w = torch.softmax(s, 0)
    out = w @ v
    size = w @ v.abs()
    rel = 2 * ((dim + 2) * 2.0 ** -24 * ((k.abs() @ q.abs()).max().item() * abs(scale)) + 2.0 ** -21 + (n + 64) * 2.0 ** -24)
    return out, (out.abs(), size, rel, n * 2.0 ** -32 * v.abs().max(0).values)


def allowed(bound, dtype):
    if isinstance(bound, torch.Tensor):
        return bound
    out, size, rel, low = bound
    half = HALF_STEP[dtype]
    # the smallest fp16 numbers are 2^-24 apart
    return half * (out + size) + 1.01 * rel * size + low + (2.0 ** -24 if dtype == torch.float16 else 0.0)


def gather(pages, table, n, head):
    """The first n positions of a sequence's pages and which of them exist, of one head: [n, dim], [n] (64 bits, CPU)."""
    size = pages.shape[2]
    rows, there = [], []
    for p in range(n):
        page = int(table[p // size])
        ok = 0 <= page < pages.shape[0]
        there.append(ok)
        rows.append(pages[page if ok else 0, head, p % size])
    if not rows:
        return torch.zeros(0, pages.shape[3], dtype=torch.float64), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows).double(), torch.tensor(there)


def paged_attention(q, k_pages, v_pages, table, lens, starts, scale):
    """(out, allowed) of packed queries over the pages; starts None: one query per sequence."""
    q, k_pages, v_pages, table, lens = (t.cpu() for t in (q, k_pages, v_pages, table, lens))
    rows, nh, dim = q.shape
    kvh = k_pages.shape[1]
    out, tol = torch.zeros(rows, nh, dim, dtype=torch.float64), torch.zeros(rows, nh, dim, dtype=torch.float64)
    at = list(range(len(lens) + 1)) if starts is None else starts.tolist()
    room = table.shape[1] * k_pages.shape[2]
    for b in range(len(lens)):
        n, length = at[b + 1] - at[b], max(0, min(int(lens[b]), room))
        for h in range(kvh):
            k, there = gather(k_pages, table[b], length, h)
            v, _ = gather(v_pages, table[b], length, h)
            for j in range(n):
                see = max(0, min(room, int(lens[b]) - n + j + 1))
                of = there[:see]
                for g in range(h * nh // kvh, (h + 1) * nh // kvh):
                    row, bound = attention_row(q[at[b] + j, g].double(), k[:see][of], v[:see][of], scale)
                    out[at[b] + j, g], tol[at[b] + j, g] = row, allowed(bound, q.dtype)
    return out, tol


def prompt_attention(q, k, v, starts, scale):
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    rows, nh, dim = q.shape
    kvh = k.shape[1]
    out, tol = torch.zeros(rows, nh, dim, dtype=torch.float64), torch.zeros(rows, nh, dim, dtype=torch.float64)
    at = starts.tolist()
    for a, e in zip(at[:-1], at[1:]):
        for j in range(a, e):
            for g in range(nh):
                h = g * kvh // nh
                row, bound = attention_row(q[j, g].double(), k[a:j + 1, h].double(), v[a:j + 1, h].double(), scale)
                out[j, g], tol[j, g] = row, allowed(bound, q.dtype)
    return out, tol


def check(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN at other places"
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    off = torch.where(odd, 0.0, (got - want).abs())
    worst = (off - torch.where(odd, 0.0, tol)).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {off.max().item():.3g}, {worst:.3g} over the bound"


def rotate(x, cos, sin, pairs):
    """x [rows, heads, dim] in 64 bits, cos / sin [rows, rotary / 2]."""
    half = cos.shape[1]
    c, s, y = cos.double().unsqueeze(1), sin.double().unsqueeze(1), x.clone()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if pairs else (x[..., :half], x[..., half:2 * half])
    u, w = a * c - b * s, a * s + b * c
    if pairs:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = u, w
    else:
        y[..., :half], y[..., half:2 * half] = u, w
    return y


def append(qkv, cos, sin, k_pages, v_pages, table, lens, starts, pairs):
    """(q, k_pages, v_pages) in 64 bits after the append, with True where a value was rotated (a rounding each)."""
    x = qkv.cpu().double()
    pages, kvh, size, dim = k_pages.shape
    x = x.view(x.shape[0], -1, dim)
    nh = x.shape[1] - 2 * kvh
    q = torch.zeros(x.shape[0], nh, dim, dtype=torch.float64)
    k_out, v_out = k_pages.cpu().double().clone(), v_pages.cpu().double().clone()
    at = list(range(len(lens) + 1)) if starts is None else starts.tolist()
    for b in range(len(lens)):
        for t in range(at[b], at[b + 1]):
            pos = int(lens[b]) - (at[b + 1] - t)
            if pos < 0 or pos >= cos.shape[0]:
                continue
            y = rotate(x[t:t + 1, :nh + kvh], cos[pos:pos + 1].cpu(), sin[pos:pos + 1].cpu(), pairs)[0]
            q[t] = y[:nh]
            if pos // size < table.shape[1] and 0 <= int(table[b, pos // size]) < pages:
                k_out[int(table[b, pos // size]), :, pos % size] = y[nh:]
                v_out[int(table[b, pos // size]), :, pos % size] = x[t, nh + kvh:]
    return q, k_out, v_out


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, logprobs) row by row in the host's extended precision."""
    x = logits.detach().cpu().double().numpy()
    rows, vocab = x.shape
    get = lambda t, none: [none] * rows if t is None else t.detach().cpu().double().tolist()  # noqa: E731
    tokens, logprobs = [], []
    for r, (u_, t, k, p, m) in enumerate(zip(get(u, 0), get(temperature, 1), get(top_k, 0), get(top_p, 1), get(min_p, 0))):
        row = np.where(np.isnan(x[r]), -np.inf, x[r])
        top = row.max()
        if top == -np.inf:
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        if not t > 0:
            tokens.append(int(row.argmax()))
            logprobs.append(0.0)
            continue
        by = np.argsort(-row, kind="stable")
        with np.errstate(invalid="ignore"):
            w = np.where(row == top, np.longdouble(1), np.exp((row.astype(np.longdouble) - top) / np.longdouble(t)))
        w[w < 2.0 ** -45] = 0  # less than half of the unit of the sums: never taken
        if k > 0:
            by = by[:int(k)]
        if p < 1:
            sums = np.cumsum(w[by])
            by = by[:max(1, int((sums < np.longdouble(p) * sums[-1]).sum()) + 1)]
        if m > 0:
            by = by[w[by] >= min(m, 1.0)]
        by = np.sort(by)
        sums = np.cumsum(w[by])
        n = min(int(np.searchsorted(sums, np.longdouble(u_) * sums[-1], side="right")), len(by) - 1)
        while w[by[n]] == 0:  # what weighs nothing is never taken
            n -= 1
        tokens.append(int(by[n]))
        logprobs.append(float(np.log(w[by[n]] / sums[-1])))
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)
