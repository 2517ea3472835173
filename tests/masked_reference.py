"""Plain 64-bit forms, on the CPU, of attention with trees and windows over a paged cache, of beam selection and of page moves."""
import math

import numpy as np
import torch

import paged_reference as ref


def masked_attention(q, k_pages, v_pages, table, lens, starts, sees, scale):
    """(out, allowed) of packed queries; ``sees(b, j, n, length)`` lists the positions (any numbers) that row j of sequence b's n
    sees.  ``starts`` None: one query per sequence."""
    q, k_pages, v_pages, table, lens = (t.cpu() for t in (q, k_pages, v_pages, table, lens))
    rows, nh, dim = q.shape
    kvh, room = k_pages.shape[1], table.shape[1] * k_pages.shape[2]
    out, tol = torch.zeros(rows, nh, dim, dtype=torch.float64), torch.zeros(rows, nh, dim, dtype=torch.float64)
    at = list(range(len(lens) + 1)) if starts is None else starts.tolist()
    for b in range(len(lens)):
        n, length = at[b + 1] - at[b], max(0, int(lens[b]))
        for h in range(kvh):
            k, there = ref.gather(k_pages, table[b], min(length, room), h)
            v, _ = ref.gather(v_pages, table[b], min(length, room), h)
            for j in range(n):
                of = [p for p in sorted(set(sees(b, j, n, length))) if 0 <= p < min(length, room) and there[p]]
                for g in range(h * nh // kvh, (h + 1) * nh // kvh):
                    row, bound = ref.attention_row(q[at[b] + j, g].double(), k[of], v[of], scale)
                    out[at[b] + j, g], tol[at[b] + j, g] = row, ref.allowed(bound, q.dtype)
    return out, tol


def in_window(window, sinks):
    def sees(b, j, n, length):
        pos = length - n + j
        return [p for p in range(max(0, pos + 1)) if p < sinks or p > pos - window]
    return sees


def in_tree(sets):
    """``sets[b][j]``: the nodes that node j of sequence b sees."""
    def sees(b, j, n, length):
        return [*range(max(0, length - n)), *(length - n + i for i in sets[b][j] if i < n)]
    return sees


def ancestors(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else []) + [i])
    return seen


def masks(sets, words):
    """The sets of all sequences' nodes as rows of 64-bit words."""
    rows = []
    for s in sets:
        for nodes in s:
            row = [0] * words
            for i in nodes:
                if i < 64 * words:
                    row[i // 64] |= 1 << i % 64
            rows.append([w - (1 << 64) if w >> 63 else w for w in row])
    return torch.tensor(rows, dtype=torch.int64).view(len(rows), words)


def beams(logits, scores, count, ended=None, pad=0):
    """(scores, beams, tokens) row by row in the host's extended precision."""
    x = logits.detach().cpu().double().numpy()
    batch, width = scores.shape
    best = torch.full((batch, count), -math.inf, dtype=torch.float64)
    parent, token = torch.full((batch, count), -1), torch.full((batch, count), -1)
    for b in range(batch):
        found = []
        for k in range(width):
            base = np.longdouble(float(scores[b, k]))
            if ended is not None and bool(ended[b, k]):
                if base > -np.inf:
                    found.append((-base, k, pad))
                continue
            row = np.where(np.isnan(x[b * width + k]), -np.inf, x[b * width + k]).astype(np.longdouble)
            top = row.max()
            if top == -np.inf or not base > -np.inf:
                continue
            if top == np.inf:
                row = np.where(row == top, np.longdouble(0), -np.inf)
                top = np.longdouble(0)
            lse = top + np.log(np.exp(row - top).sum())
            by = np.argsort(-row, kind="stable")[:count]
            found += [(-(base + (row[v] - lse)), k, int(v)) for v in by if row[v] > -np.inf]
        for i, (t, k, v) in enumerate(sorted(found)[:count]):
            best[b, i], parent[b, i], token[b, i] = float(-t), k, v
    return best, parent, token


def copied(pages, src, dst, filled=None):
    """Pools ``[layers, pages, kvh, page, dim]`` after the copies."""
    out = pages.clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        if 0 <= a < pages.shape[1] and 0 <= b < pages.shape[1]:
            n = pages.shape[3] if filled is None else max(0, min(filled[i], pages.shape[3]))
            out[:, b, :, :n] = pages[:, a, :, :n]
    return out


def kept(pages, table, first, keep, starts):
    """Pools after the moves, all of a sequence read before any is written."""
    out, size = pages.clone(), pages.shape[3]

    def place(b, p):
        if not 0 <= p < table.shape[1] * size:
            return None
        page = int(table[b, p // size])
        return (page, p % size) if 0 <= page < pages.shape[1] else None

    for b in range(len(first)):
        for i, e in enumerate(keep[starts[b]:starts[b + 1]]):
            src, dst = place(b, first[b] + e), place(b, first[b] + i)
            if src and dst:
                out[:, dst[0], :, dst[1]] = pages[:, src[0], :, src[1]]
    return out
