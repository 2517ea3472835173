"""Llama-shaped decoder stack with every linear on the W4A16 kernels (measurement harness).

Used to measure prefill and greedy-decode throughput on the shapes of the W4A16
workloads: Llama-2-7B (32 layers, hidden 4096, 32 heads, FFN 11008, vocab 32000)
and Llama-3-70B (80 layers, hidden 8192, 64 q / 8 kv heads, FFN 28672, vocab 128256).
Weights are random W4 g128 codes with fp16 scales / zeros (a random init of the
quantized model; no checkpoint is loaded).  q/k/v and gate/up are fused into one
W4A16 GEMM each (row concatenation of the packed weight is exact).

``decode_step`` runs one greedy step as 7-8 launches per layer: fused residual-add
+ RMSNorm, the W4A16 GEMVs, split-K decode attention with RoPE and the KV append
fused in (plus the split merge), and the gate/up GEMV with SiLU-mul in its epilogue.
With one row (and hidden 2048 / 4096) each add-RMSNorm runs in the prologue of the
GEMV that consumes it: 6 launches per layer.
The KV cache has a fixed capacity ``[L, B, kvh, T, 128]`` and every kernel reads
the current position from device memory, so a step is shape-static and can be
captured into a HIP graph.  ``decode_step_torch`` is the same step in PyTorch ops
(masked attention over the whole cache), kept as the numerical reference.  Prefill
uses PyTorch attention (SDPA) around the same W4A16 linears and fused norm / SiLU-mul kernels.

``PagedKVCache`` holds sequences of different lengths in pages instead.  ``forward_paged`` runs packed
new tokens of any of them (whole prompts, chunks of prompts, one token each) on the paged operators:
append with rotation, decode or prompt attention.  ``generate_paged`` serves prompts with it, the
tokens drawn by ``ops.sample_tokens``.  ``generate_drafted`` has drafted tokens verified, a tree of them per sequence and pass
(``forward_tree``), ``beam_search_paged`` searches with beams that share their pages, and a model whose configuration has a
window keeps only the pages that its tokens still see.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, List, Optional, Sequence, Tuple

import torch

from . import ops


@dataclass
class DecoderConfig:
    layers: int = 32
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 32
    ffn: int = 11008
    vocab: int = 32000
    group: int = 128
    rope_theta: float = 10000.0
    eps: float = 1e-5
    window: int = 0  # positions that a token sees, its own among them (0: all), on a paged cache
    sinks: int = 0   # first positions that stay visible with a window

    @staticmethod
    def llama2_7b():
        return DecoderConfig()

    @staticmethod
    def llama3_70b():
        return DecoderConfig(layers=80, hidden=8192, heads=64, kv_heads=8, ffn=28672, vocab=128256,
                             rope_theta=500000.0)

    @property
    def head_dim(self):
        return self.hidden // self.heads


class _W4:
    """Random W4 g128 linear held as packed codes + fp16 scales / zeros."""

    def __init__(self, n, k, group, gen, device):
        self.n, self.k, self.group = n, k, group
        self.packed = torch.randint(-2**31, 2**31 - 1, (n, k // 8), generator=gen, device=device, dtype=torch.int32)
        # dequantised values (u - z) * s with s ~ 0.0027: weights of std ~0.012 over [-0.02, 0.02]
        self.scales = (torch.rand(n, k // group, generator=gen, device=device) * 0.001 + 0.0022).half()
        self.zeros = torch.full((n, k // group), 8.0, device=device, dtype=torch.float16)

    def __call__(self, x):
        return ops.w4a16_gemm(x, self.packed, self.scales, self.zeros, self.group, None)

    def swiglu(self, x):
        """silu(gate) * up of this fused gate/up linear in one launch."""
        return ops.w4a16_gemm_swiglu(x, self.packed, self.scales, self.zeros, self.group, None)

    def nbytes(self):
        return self.packed.numel() * 4 + self.scales.numel() * 2 + self.zeros.numel() * 2

    def dequantized(self):
        """The pseudo-quantized fp16 weight ``(u - z) * s`` (each op rounded to fp16, as the reference's
        dequantised tensor), unpacked with torch bit operations: the reference path shares no kernel
        with the W4A16 GEMMs it checks.  Cached."""
        w = getattr(self, "_deq", None)
        if w is None:
            shifts = torch.arange(0, 32, 4, device=self.packed.device, dtype=torch.int32)
            u = ((self.packed.unsqueeze(-1) >> shifts) & 0xF).reshape(self.n, self.k).to(torch.float16)
            s = self.scales.repeat_interleave(self.group, dim=1)
            z = self.zeros.repeat_interleave(self.group, dim=1)
            w = (u - z) * s
            self._deq = w
        return w

    def reference(self, x):
        """``F.linear`` on the pseudo-quantized weight with fp32 accumulation, one rounding to fp16."""
        return (x.float() @ self.dequantized().float().t()).half()


def _rms(x, w, eps):
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).half() * w


class PagedKVCache:
    """Keys and values of up to ``sequences`` sequences in pages of ``page`` positions, ``positions`` in all.

    ``k`` / ``v [layers, pages, kv_heads, page, head_dim]`` are the pools; ``table`` (int32, a row of pages for each
    sequence) and ``lens`` (int32) are what the paged operators read, in device memory and updated in place, so a
    captured step goes on working while the sequences grow.  Which pages are free is kept on the host.  Sequences that were
    forked share their pages; one that goes on has a shared page that it would write to copied first (``extend``)."""

    def __init__(self, cfg: DecoderConfig, sequences: int, positions: int, page: int = 64, max_len: Optional[int] = None,
                 device="cuda", dtype=torch.float16):
        if sequences < 1 or positions < 1 or page < 8 or page & (page - 1):
            raise ValueError("sequences and positions must be positive, page a power of two from 8")
        pages = -(-positions // page)
        self.page, self.max_len = page, max_len if max_len is not None else pages * page
        shape = (cfg.layers, pages, cfg.kv_heads, page, cfg.head_dim)
        self.k = torch.zeros(shape, device=device, dtype=dtype)
        self.v = torch.zeros(shape, device=device, dtype=dtype)
        self.table = torch.zeros(sequences, -(-self.max_len // page), device=device, dtype=torch.int32)
        self.lens = torch.zeros(sequences, device=device, dtype=torch.int32)
        self.length = [0] * sequences                      # of lens, on the host
        self._held: List[List[int]] = [[] for _ in range(sequences)]  # -1: a page that was trimmed
        self._least = [0] * sequences                      # below it a next token would look at pages that were trimmed
        self._uses = [0] * pages                           # sequences that hold a page
        self._shared = 0                                   # holds of pages beyond their first
        self._free = list(range(pages - 1, -1, -1))

    def free_positions(self) -> int:
        return len(self._free) * self.page

    def _take(self) -> int:
        page = self._free.pop()
        self._uses[page] = 1
        return page

    def _drop(self, pages: Sequence[int]) -> None:
        for page in pages:
            if page >= 0:
                self._uses[page] -= 1
                if self._uses[page]:
                    self._shared -= 1
                else:
                    self._free.append(page)

    def _set_table(self, rows: List[int], cols: List[int], pages: List[int]) -> None:
        if rows:
            at = torch.tensor([rows, cols], device=self.table.device)
            self.table[at[0], at[1]] = torch.tensor(pages, device=self.table.device, dtype=torch.int32)

    def _set_lens(self) -> None:
        self.lens.copy_(torch.tensor(self.length, dtype=torch.int32))

    @torch.no_grad()
    def extend(self, news: Sequence[int]) -> Optional[torch.Tensor]:
        """Makes room for ``news[b]`` more positions of each sequence b, whose keys and values the next ``forward_paged``
        writes: takes pages, updates ``table`` and ``lens``.  Returns the offsets of the sequences' tokens in their packed
        order (``starts``), or ``None`` where every sequence has one.  Raises, and changes nothing, if a sequence gets too
        long or the pages do not suffice."""
        if len(news) != len(self.length) or any(n < 0 for n in news):
            raise ValueError(f"one count for each of the {len(self.length)} sequences, got {list(news)}")
        want = [-(-(l + n) // self.page) - len(h) for l, n, h in zip(self.length, news, self._held)]
        if any(l + n > self.max_len for l, n in zip(self.length, news)):
            raise RuntimeError(f"a sequence would pass {self.max_len} positions")
        # begun pages that others hold as well: all but the last of their holders that go on have them copied
        uses, copies = {}, []
        for b, (l, n, held) in enumerate(zip(self.length, news, self._held) if self._shared else ()):
            if n and l % self.page:
                page = held[l // self.page]
                uses[page] = uses.get(page, self._uses[page])
                if uses[page] > 1:
                    uses[page] -= 1
                    copies.append((b, page))
        if sum(want) + len(copies) > len(self._free):
            raise RuntimeError(f"{sum(want) + len(copies)} pages are wanted and {len(self._free)} are free")
        device = self.table.device
        rows, cols, pages = [], [], []
        for b, page in copies:
            rows.append(b)
            cols.append(self.length[b] // self.page)
            pages.append(self._take())
            self._held[b][cols[-1]] = pages[-1]
            self._drop([page])
        if copies:
            move = torch.tensor([[page for _, page in copies], pages, [self.length[b] % self.page for b, _ in copies]],
                                device=device, dtype=torch.int32)
            ops.paged_copy_pages(self.k, self.v, move[0], move[1], move[2])
        for b, n in enumerate(want):
            for _ in range(n):
                rows.append(b)
                cols.append(len(self._held[b]))
                pages.append(self._take())
                self._held[b].append(pages[-1])
        self._set_table(rows, cols, pages)
        self.length = [l + n for l, n in zip(self.length, news)]
        self._set_lens()
        if all(n == 1 for n in news):
            return None
        starts = torch.zeros(len(news) + 1, dtype=torch.int32)
        starts[1:] = torch.tensor(news, dtype=torch.int32).cumsum(0)
        return starts.to(device)

    @torch.no_grad()
    def release(self, sequence: int) -> None:
        """Ends a sequence: the pages that it alone held are free again."""
        self._drop(reversed(self._held[sequence]))
        self._held[sequence] = []
        self._least[sequence] = self.length[sequence] = 0
        self.lens[sequence] = 0

    @torch.no_grad()
    def reorder(self, order: Sequence[int]) -> None:
        """Sequence b goes on as what sequence ``order[b]`` was: tables and lengths change, pages are shared and nothing is
        copied before ``extend`` writes.  What no sequence goes on as is released."""
        if len(order) != len(self.length) or not all(0 <= o < len(order) for o in order):
            raise ValueError(f"one of the {len(self.length)} sequences for each of them, got {list(order)}")
        if all(o == b for b, o in enumerate(order)):
            return
        held = [list(self._held[o]) for o in order]
        for pages in held:
            for page in pages:
                if page >= 0:
                    self._uses[page] += 1
                    self._shared += 1
        for pages in self._held:
            self._drop(reversed(pages))
        self._held = held
        self._least = [self._least[o] for o in order]
        self.length = [self.length[o] for o in order]
        self.table.copy_(self.table[torch.tensor(list(order), device=self.table.device)])
        self._set_lens()

    @torch.no_grad()
    def fork(self, source: int, target: int) -> None:
        """The empty sequence ``target`` begins as what ``source`` is."""
        if self.length[target] or source == target:
            raise ValueError(f"sequence {target} must be empty and another than {source}")
        order = list(range(len(self.length)))
        order[target] = source
        self.reorder(order)

    @torch.no_grad()
    def keep(self, drafted: Sequence[int], kept: Sequence[Sequence[int]]) -> None:
        """Of the last ``drafted[b]`` positions of each sequence b those that ``kept[b]`` names stay, ascending from 0, one behind
        the other; pages behind them are free again.  Raises, and changes nothing, where a sequence was forked since its draft, or
        trimmed so far that its next token would look at a page that is gone."""
        if len(drafted) != len(self.length) or len(kept) != len(self.length):
            raise ValueError(f"a count and a list for each of the {len(self.length)} sequences")
        for l, n, at in zip(self.length, drafted, kept):
            if not 0 <= n <= l or any(not 0 <= i < n for i in at) or any(i >= j for i, j in zip(at, at[1:])):
                raise ValueError(f"{list(at)} must ascend below the {n} drafted positions of {l}")
        for l, n, at, held, least in zip(self.length, drafted, kept, self._held, self._least):
            if n and (l - n + len(at) < least or any(page < 0 or self._uses[page] > 1 for page in held[(l - n) // self.page:])):
                raise RuntimeError("a sequence that was forked or trimmed since its draft keeps it as it is")
        if any(i != j for at in kept for j, i in enumerate(at)):
            device, first = self.table.device, [l - n for l, n in zip(self.length, drafted)]
            starts = [0]
            for at in kept:
                starts.append(starts[-1] + len(at))
            ints = torch.tensor([*first, *starts, *(i for at in kept for i in at)], dtype=torch.int32).to(device)
            n = len(first)
            # views of one transfer
            ops.paged_keep_positions(self.k, self.v, self.table, ints[:n], ints[2 * n + 1:], ints[n:2 * n + 1])
        for b, (n, at) in enumerate(zip(drafted, kept)):
            self.length[b] += len(at) - n
            stay = -(-self.length[b] // self.page)
            self._drop(reversed(self._held[b][stay:]))
            del self._held[b][stay:]
        self._set_lens()

    @torch.no_grad()
    def trim(self, window: int, sinks: int = 0) -> int:
        """Frees the pages that no later token sees with a window of ``window`` positions and ``sinks`` first ones; how many."""
        if window < 1 or sinks < 0:
            raise ValueError(f"a window has a position at least, and sinks are not negative: {window}, {sinks}")
        rows, cols = [], []
        for b, held in enumerate(self._held):
            for i in range(-(-sinks // self.page), max(0, self.length[b] - window + 1) // self.page):
                if held[i] >= 0:
                    rows.append(b)
                    cols.append(i)
        for b, i in zip(rows, cols):
            self._drop([self._held[b][i]])
            self._held[b][i] = -1
            self._least[b] = max(self._least[b], (i + 1) * self.page + window - 1)
        self._set_table(rows, cols, [-1] * len(rows))
        return len(rows)


def lookup_draft(match: int = 2, nodes: int = 8, branches: int = 2) -> Callable[[List[int]], Tuple[List[int], List[int]]]:
    """Drafts from the sequence itself for ``W4Decoder.generate_drafted``: what followed the last ``match`` tokens where they
    stood before, the latest places first, up to ``branches`` of them and ``nodes`` tokens in all."""
    def draft(tokens: List[int]) -> Tuple[List[int], List[int]]:
        found: List[int] = []
        parents: List[int] = []
        places = [i for i in range(len(tokens) - match - 1, -1, -1) if tokens[i:i + match] == tokens[-match:]]
        for i in places[:branches]:
            node = -1
            for t in tokens[i + match:i + match + max(1, nodes // branches)]:
                same = [j for j, p in enumerate(parents) if p == node and found[j] == t]
                if not same:
                    found.append(t)
                    parents.append(node)
                node = same[0] if same else len(found) - 1
        return found[:nodes], parents[:nodes]
    return draft


class W4Decoder:
    def __init__(self, cfg: DecoderConfig, max_batch: int, max_len: int, device="cuda", seed: int = 1):
        self.cfg, self.max_batch, self.max_len = cfg, max_batch, max_len
        self.fuse_norm = True  # one-row decode steps: add-RMSNorm inside the next GEMV
        gen = torch.Generator(device=device).manual_seed(seed)
        h, hd, kvh = cfg.hidden, cfg.head_dim, cfg.kv_heads
        self.embed = (torch.randn(cfg.vocab, h, generator=gen, device=device) * 0.02).half()
        self.layers = []
        for _ in range(cfg.layers):
            self.layers.append({
                "ln1": torch.ones(h, device=device, dtype=torch.float16),
                "ln2": torch.ones(h, device=device, dtype=torch.float16),
                "qkv": _W4((cfg.heads + 2 * kvh) * hd, h, cfg.group, gen, device),
                "o": _W4(h, cfg.heads * hd, cfg.group, gen, device),
                "gate_up": _W4(2 * cfg.ffn, h, cfg.group, gen, device),
                "down": _W4(h, cfg.ffn, cfg.group, gen, device),
            })
        self.norm = torch.ones(h, device=device, dtype=torch.float16)
        self.lm_head = _W4(cfg.vocab, h, cfg.group, gen, device)
        # KV cache [L, B, kvh, T, hd]: one 256-byte row per position
        self.k_cache = torch.zeros(cfg.layers, max_batch, kvh, max_len, hd, device=device, dtype=torch.float16)
        self.v_cache = torch.zeros(cfg.layers, max_batch, kvh, max_len, hd, device=device, dtype=torch.float16)
        self.attn_ws = {}
        inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, hd, 2, device=device).float() / hd))
        t = torch.arange(max_len, device=device).float()
        freqs = torch.outer(t, inv)
        self.cos = freqs.cos().half()
        self.sin = freqs.sin().half()

    def _contiguous(self):
        if self.cfg.window:
            raise RuntimeError("a model with a window runs on a paged cache")

    def weight_bytes(self):
        return sum(l[n].nbytes() for l in self.layers for n in ("qkv", "o", "gate_up", "down")) + self.lm_head.nbytes()

    def _rope(self, x, pos):
        # x [B, heads, T, hd]; pos [T] (or [B, T] for decode)
        cos = self.cos[pos].unsqueeze(-3) if pos.dim() == 1 else self.cos[pos].unsqueeze(1)
        sin = self.sin[pos].unsqueeze(-3) if pos.dim() == 1 else self.sin[pos].unsqueeze(1)
        x1, x2 = x[..., 0::2], x[..., 1::2]
        out = torch.empty_like(x)
        out[..., 0::2] = x1 * cos - x2 * sin
        out[..., 1::2] = x1 * sin + x2 * cos
        return out

    @torch.no_grad()
    def prefill(self, tokens, return_logits=False):
        """tokens [B, T] int64; fills the cache at positions [0, T); returns next-token ids [B]
        (or the last position's logits).  The residual adds and RMSNorms run on the fused
        kernels (one launch each), the SiLU-mul in the gate/up GEMM's epilogue, RoPE and the
        cache writes in one launch; attention is PyTorch SDPA."""
        self._contiguous()
        cfg = self.cfg
        b, t = tokens.shape
        hd, nh, kvh = cfg.head_dim, cfg.heads, cfg.kv_heads
        x = self.embed[tokens].reshape(b * t, -1)                  # [B*T, H] residual stream
        delta = None
        for li, l in enumerate(self.layers):
            if delta is None:
                hn = ops.add_rms_norm_quant(x, None, l["ln1"], cfg.eps, quant=False)[0]
            else:
                hn, _, _, x = ops.add_rms_norm_quant(delta, x, l["ln1"], cfg.eps, quant=False)
            # one launch: RoPE on q / k, q to [B, nh, T, hd], k / v into the cache rows 0 .. T-1
            q = ops.prefill_rope_split(l["qkv"](hn), b, nh, kvh, self.cos, self.sin, self.k_cache[li, :b],
                                       self.v_cache[li, :b])
            k, v = self.k_cache[li, :b, :, :t], self.v_cache[li, :b, :, :t]
            kk = k.repeat_interleave(nh // kvh, dim=1) if kvh != nh else k
            vv = v.repeat_interleave(nh // kvh, dim=1) if kvh != nh else v
            att = torch.nn.functional.scaled_dot_product_attention(q, kk.contiguous(), vv.contiguous(), is_causal=True)
            o = l["o"](att.transpose(1, 2).reshape(b * t, nh * hd))
            hn, _, _, x = ops.add_rms_norm_quant(o, x, l["ln2"], cfg.eps, quant=False)
            delta = l["down"](l["gate_up"].swiglu(hn))  # gate/up GEMM with SiLU-mul in its epilogue
        # the last position of each sequence only
        d_last = delta.reshape(b, t, -1)[:, -1].contiguous()
        x_last = x.reshape(b, t, -1)[:, -1].contiguous()
        hn = ops.add_rms_norm_quant(d_last, x_last, self.norm, cfg.eps, quant=False)[0]
        logits = self.lm_head(hn)
        return logits if return_logits else logits.argmax(-1)

    @torch.no_grad()
    def prefill_torch(self, tokens, return_logits=False):
        """The prefill in PyTorch ops (reference path): every linear is F.linear on the
        pseudo-quantized fp16 weight (fp32 accumulation), attention in fp32."""
        self._contiguous()
        cfg = self.cfg
        b, t = tokens.shape
        hd, nh, kvh = cfg.head_dim, cfg.heads, cfg.kv_heads
        x = self.embed[tokens]
        pos = torch.arange(t, device=tokens.device)
        for li, l in enumerate(self.layers):
            hn = _rms(x, l["ln1"], cfg.eps)
            qkv = l["qkv"].reference(hn.reshape(b * t, -1)).reshape(b, t, nh + 2 * kvh, hd).transpose(1, 2)
            q, k, v = qkv[:, :nh], qkv[:, nh:nh + kvh], qkv[:, nh + kvh:]
            q, k = self._rope(q, pos), self._rope(k, pos)
            self.k_cache[li, :b, :, :t] = k
            self.v_cache[li, :b, :, :t] = v
            kk = k.repeat_interleave(nh // kvh, dim=1) if kvh != nh else k
            vv = v.repeat_interleave(nh // kvh, dim=1) if kvh != nh else v
            att = torch.nn.functional.scaled_dot_product_attention(q.float(), kk.float(), vv.float(),
                                                                   is_causal=True).half()
            x = x + l["o"].reference(att.transpose(1, 2).reshape(b * t, nh * hd)).reshape(b, t, -1)
            hn = _rms(x, l["ln2"], cfg.eps)
            gu = l["gate_up"].reference(hn.reshape(b * t, -1))
            act = torch.nn.functional.silu(gu[:, :cfg.ffn]) * gu[:, cfg.ffn:]
            x = x + l["down"].reference(act.contiguous()).reshape(b, t, -1)
        logits = self.lm_head.reference(_rms(x[:, -1], self.norm, cfg.eps).contiguous())
        return logits if return_logits else logits.argmax(-1)

    def attn_splits(self, b):
        """Workgroups per (row, kv head) for the decode attention: ~1024 in all for one head per
        kv head, ~512 (at most 32 splits) for head groups, whose MFMA scoring makes longer
        chunks pay (70B, measured: B = 1 9.38 -> 9.23 ms with 32 splits instead of 64, B = 16
        17.80 -> 17.57 ms with 4 instead of 8), and a score buffer of at most 64 KB per
        workgroup."""
        cfg = self.cfg
        grp = cfg.heads // cfg.kv_heads
        if grp >= 4:
            splits = max(1, min(32, 512 // (b * cfg.kv_heads)))
        else:
            splits = max(1, min(64, 1024 // (b * cfg.kv_heads)))
        while -(-self.max_len // splits) * grp * 4 > 64 * 1024:
            splits += 1
        return splits

    def _attn_workspace(self, b):
        splits = self.attn_splits(b)
        key = (b, splits)
        if key not in self.attn_ws:
            self.attn_ws[key] = ops.decode_attention_workspace(b, self.cfg.heads, splits, self.k_cache.device)
        return splits, self.attn_ws[key]

    @torch.no_grad()
    def decode_step(self, tokens, cur_len, return_logits=False):
        """One greedy step for a batch on the fused kernels.  tokens [B] int64 (the last
        token), cur_len [1] int64 device tensor = position of that token; writes its K/V
        and returns the next ids (or the logits)."""
        self._contiguous()
        cfg = self.cfg
        b = tokens.shape[0]
        hd, nh, kvh = cfg.head_dim, cfg.heads, cfg.kv_heads
        splits, ws = self._attn_workspace(b)
        scale = 1.0 / math.sqrt(hd)
        x = self.embed[tokens]                                    # [B, H] residual stream
        # one row of width <= 4096: each add-RMSNorm runs inside the next GEMV (at 8192 every
        # workgroup's 48 KB prologue costs more than the launch it saves: 70B 9.37 -> 9.80 ms/step)
        fused = self.fuse_norm and b == 1 and cfg.hidden in (2048, 4096) and cfg.group == 128

        def norm_linear(delta, x, w, lin, swiglu=False):
            """(lin(RMSNorm(delta + x) * w), delta + x); delta None: no residual add."""
            if fused:
                src, res = (x, None) if delta is None else (delta, x)
                y, rsum = ops.w4a16_gemv_add_rms_norm(src, res, w, cfg.eps, lin.packed, lin.scales, lin.zeros,
                                                      lin.group, None, swiglu)
                return y, (x if rsum is None else rsum)
            if delta is None:
                hn = ops.add_rms_norm_quant(x, None, w, cfg.eps, quant=False)[0]
            else:
                hn, _, _, x = ops.add_rms_norm_quant(delta, x, w, cfg.eps, quant=False)
            return (lin.swiglu(hn) if swiglu else lin(hn)), x

        delta = None
        for li, l in enumerate(self.layers):
            qkv, x = norm_linear(delta, x, l["ln1"], l["qkv"])
            att = ops.decode_rope_attention(qkv, nh, kvh, self.cos, self.sin, cur_len, self.k_cache[li, :b],
                                            self.v_cache[li, :b], splits, scale, ws)
            act, x = norm_linear(l["o"](att.reshape(b, nh * hd)), x, l["ln2"], l["gate_up"], swiglu=True)
            delta = l["down"](act)
        logits, x = norm_linear(delta, x, self.norm, self.lm_head)
        return logits if return_logits else ops.argmax_rows(logits)

    @torch.no_grad()
    def decode_step_torch(self, tokens, cur_len, return_logits=False):
        """The decode step in PyTorch ops (reference path): RMSNorm on the rounded residual, every
        linear F.linear on the pseudo-quantized fp16 weight (fp32 accumulation), fp32 attention over the
        whole cache masked by the current length."""
        self._contiguous()
        cfg = self.cfg
        b = tokens.shape[0]
        hd, nh, kvh = cfg.head_dim, cfg.heads, cfg.kv_heads
        grp = nh // kvh
        x = self.embed[tokens]                                    # [B, H]
        pos = cur_len.expand(b).unsqueeze(1)                      # [B, 1]
        mask = torch.where(torch.arange(self.max_len, device=tokens.device) > cur_len, float("-inf"), 0.0)
        scale = 1.0 / math.sqrt(hd)
        for li, l in enumerate(self.layers):
            hn = _rms(x, l["ln1"], cfg.eps)
            qkv = l["qkv"].reference(hn).reshape(b, nh + 2 * kvh, 1, hd)
            q, k, v = qkv[:, :nh], qkv[:, nh:nh + kvh], qkv[:, nh + kvh:]
            q, k = self._rope(q, pos), self._rope(k, pos)
            self.k_cache[li, :b].index_copy_(2, cur_len, k.contiguous())
            self.v_cache[li, :b].index_copy_(2, cur_len, v.contiguous())
            qg = q.reshape(b, kvh, grp, hd).float()                # heads grouped by kv head
            kt = self.k_cache[li, :b].float().transpose(-1, -2).contiguous()
            s = torch.matmul(qg, kt) * scale + mask                # [B, kvh, grp, T]
            p = torch.softmax(s, dim=-1)
            att = torch.matmul(p, self.v_cache[li, :b].float()).half()
            x = x + l["o"].reference(att.reshape(b, nh * hd))
            hn = _rms(x, l["ln2"], cfg.eps)
            gu = l["gate_up"].reference(hn)
            act = torch.nn.functional.silu(gu[:, :cfg.ffn]) * gu[:, cfg.ffn:]
            x = x + l["down"].reference(act.contiguous())
        logits = self.lm_head.reference(_rms(x, self.norm, cfg.eps).contiguous())
        return logits if return_logits else logits.argmax(-1)

    def paged_cache(self, sequences: int, positions: int, page: int = 64) -> PagedKVCache:
        """A paged cache for this model: up to ``positions`` in all, ``max_len`` of one sequence."""
        self._angles()  # before a step may be captured
        return PagedKVCache(self.cfg, sequences, positions, page, self.max_len, self.embed.device)

    def _angles(self):
        """cos / sin of every position in fp32, from angles in 64 bits (far positions lose theirs in 32)."""
        if getattr(self, "_cos_sin", None) is None:
            hd, device = self.cfg.head_dim, self.embed.device
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a step has to run, or paged_cache be called, before one is captured")
            inv = self.cfg.rope_theta ** (-torch.arange(0, hd, 2, device=device, dtype=torch.float64) / hd)
            angle = torch.outer(torch.arange(self.max_len, device=device, dtype=torch.float64), inv)
            self._cos_sin = angle.cos().float(), angle.sin().float()
        return self._cos_sin

    @torch.no_grad()
    def forward_paged(self, tokens, cache: PagedKVCache, starts: Optional[torch.Tensor] = None):
        """Logits ``[sequences, vocab]`` after the last of each sequence's new tokens.  ``tokens`` (int64) are the packed new
        tokens and ``starts`` their offsets, both for the positions that ``cache.extend`` has just made room for; without
        ``starts`` each sequence has one.  A sequence without new tokens gets -inf everywhere, from which
        ``ops.sample_tokens`` takes no token (-1).  Reads lengths and pages from device memory: a step without ``starts`` can be
        captured and replayed after each ``extend``."""
        cfg, scale = self.cfg, 1.0 / math.sqrt(self.cfg.head_dim)
        cos, sin = self._paged_checks(tokens, cache)

        def attend(li, qkv):
            k, v = cache.k[li], cache.v[li]
            q = ops.paged_rope_append(qkv, cos, sin, k, v, cache.table, cache.lens, starts)
            if starts is None and cfg.window:
                return ops.paged_decode_window_attention(q, k, v, cache.table, cache.lens, scale, cfg.window, cfg.sinks)
            if starts is None:
                return ops.paged_decode_attention(q, k, v, cache.table, cache.lens, scale)
            if cfg.window:
                return ops.paged_prompt_window_attention(q, k, v, cache.table, cache.lens, starts, scale, cfg.window, cfg.sinks)
            return ops.paged_prompt_attention(q, k, v, cache.table, cache.lens, starts, scale)

        x, delta = self._paged_layers(tokens, attend)
        if starts is not None:  # the last row of each sequence
            last = (starts[1:].long() - 1).clamp(0, len(tokens) - 1)
            delta, x = delta[last], x[last]
        logits = self.lm_head(ops.add_rms_norm_quant(delta, x, self.norm, cfg.eps, quant=False)[0])
        if starts is not None:
            logits.masked_fill_((starts[1:] <= starts[:-1]).unsqueeze(1), -math.inf)
        return logits

    def _paged_checks(self, tokens, cache: PagedKVCache):
        if tokens.dim() != 1 or not tokens.numel():
            raise ValueError(f"tokens must be packed in one dimension and hold one at least, got {tuple(tokens.shape)}")
        if max(cache.length) > self.max_len:
            raise RuntimeError(f"a sequence of {max(cache.length)} positions, the model has {self.max_len}")
        return self._angles()

    def _paged_layers(self, tokens, attend):
        """The layers over packed new tokens, ``attend(layer, qkv)`` their attention: (residual, its last addend)."""
        cfg = self.cfg
        x, delta = self.embed[tokens], None
        for li, l in enumerate(self.layers):
            if delta is None:
                hn = ops.add_rms_norm_quant(x, None, l["ln1"], cfg.eps, quant=False)[0]
            else:
                hn, _, _, x = ops.add_rms_norm_quant(delta, x, l["ln1"], cfg.eps, quant=False)
            att = attend(li, l["qkv"](hn))
            hn, _, _, x = ops.add_rms_norm_quant(l["o"](att.view(-1, cfg.heads * cfg.head_dim)), x, l["ln2"], cfg.eps, quant=False)
            delta = l["down"](l["gate_up"].swiglu(hn))
        return x, delta

    @torch.no_grad()
    def forward_tree(self, tokens, cache: PagedKVCache, parents: Sequence[Sequence[int]]):
        """Logits ``[tokens, vocab]`` after each of the sequences' drafted tokens, packed in ``tokens`` (int64), for the positions that
        ``cache.extend`` has just made room for.  ``parents[b]`` says of each node of sequence b which earlier node it follows,
        or -1 for what the cache held before; a node sees that, its ancestors and itself, and turns by its depth.
        ``cache.keep`` takes up the accepted ones."""
        cfg, scale = self.cfg, 1.0 / math.sqrt(self.cfg.head_dim)
        if cfg.window:
            raise RuntimeError("trees are verified without a window")
        cos, sin = self._paged_checks(tokens, cache)
        if len(parents) != len(cache.length) or sum(map(len, parents)) != tokens.numel():
            raise ValueError(f"a list of parents for each of the {len(cache.length)} sequences, a parent for each of the "
                             f"{tokens.numel()} tokens")
        words = max(1, -(-max(map(len, parents)) // 64))
        starts, turns, masks = [0], [], []
        for length, nodes in zip(cache.length, parents):
            if len(nodes) > length or any(not -1 <= p < i for i, p in enumerate(nodes)):
                raise ValueError(f"a node follows an earlier one or -1, {list(nodes)} of {length} positions")
            depth, seen = [], []
            for i, p in enumerate(nodes):
                depth.append(depth[p] + 1 if p >= 0 else 0)
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            starts.append(starts[-1] + len(nodes))
            turns += [length - len(nodes) + d for d in depth]
            for s in seen:
                row = [s >> 64 * w & (1 << 64) - 1 for w in range(words)]
                masks.append([w - (1 << 64) if w >> 63 else w for w in row])
        device = tokens.device
        masks = torch.tensor(masks, dtype=torch.int64).to(device)
        starts, turns = (torch.tensor(t, dtype=torch.int32).to(device) for t in (starts, turns))

        def attend(li, qkv):
            k, v = cache.k[li], cache.v[li]
            q = ops.paged_rope_append(qkv, cos, sin, k, v, cache.table, cache.lens, starts, turns=turns)
            return ops.paged_tree_attention(q, k, v, cache.table, cache.lens, starts, masks, scale)

        x, delta = self._paged_layers(tokens, attend)
        return self.lm_head(ops.add_rms_norm_quant(delta, x, self.norm, cfg.eps, quant=False)[0])

    @torch.no_grad()
    def generate_paged(self, prompts: Sequence[torch.Tensor], new_tokens: int, cache: Optional[PagedKVCache] = None,
                       temperature=None, top_k=None, top_p=None, min_p=None, generator: Optional[torch.Generator] = None):
        """``new_tokens`` tokens after each of ``prompts`` (int64 tensors of different lengths): the prompts in one packed
        pass, then a token of every sequence per step.  ``temperature``, ``top_k``, ``top_p``, ``min_p``: one value per prompt
        or ``None`` (``ops.sample_tokens``); ``temperature`` ``None`` takes the largest logit.  Returns ``[prompts,
        new_tokens]``; a sequence whose logits leave nothing to take (all NaN or -inf) has -1 from there on."""
        device = self.embed.device
        lengths = [int(p.numel()) for p in prompts]
        if not lengths or min(lengths) < 1 or new_tokens < 1:
            raise ValueError("prompts must hold a token at least, and new_tokens must be positive")
        if cache is None:
            page = 64
            cache = self.paged_cache(len(prompts), sum(-(-(n + new_tokens) // page) * page for n in lengths), page)
        if temperature is None:
            temperature = torch.zeros(len(prompts), device=device)

        def sample(logits):
            u = torch.rand(len(prompts), device=device, generator=generator)
            return ops.sample_tokens(logits, u, temperature, top_k, top_p, min_p)[0]

        starts = cache.extend(lengths)
        tokens = sample(self.forward_paged(torch.cat([p.reshape(-1) for p in prompts]).to(device), cache, starts))
        out = [tokens]
        for _ in range(new_tokens - 1):
            if self.cfg.window:
                cache.trim(self.cfg.window, self.cfg.sinks)
            cache.extend([1] * len(prompts))
            # a sequence that has ended goes on with the vocabulary's first token, and stays ended
            tokens = sample(self.forward_paged(out[-1].clamp(min=0), cache))
            out.append(torch.where(out[-1] < 0, -1, tokens))
        return torch.stack(out, 1)

    @torch.no_grad()
    def generate_drafted(self, prompts: Sequence[torch.Tensor], new_tokens: int,
                         draft: Optional[Callable[[List[int]], Tuple[List[int], List[int]]]] = None,
                         cache: Optional[PagedKVCache] = None):
        """``generate_paged`` that takes the largest logit, with several tokens a pass where drafts come true: ``draft`` gets a
        sequence's tokens and returns ``(tokens, parents)`` of a tree of tokens that may follow (a parent: an earlier one
        of them, or -1), ``lookup_draft()`` if ``None``.  A pass verifies every sequence's tree, takes the path along which each
        token is the one that the model takes, and a token more.  Returns ``[prompts, new_tokens]``, -1 from where a sequence has
        nothing to take."""
        device, draft = self.embed.device, draft or lookup_draft()
        history = [p.reshape(-1).tolist() for p in prompts]
        lengths = [len(h) for h in history]
        if not lengths or min(lengths) < 1 or new_tokens < 1:
            raise ValueError("prompts must hold a token at least, and new_tokens must be positive")
        if self.cfg.window:
            raise RuntimeError("trees are verified without a window")
        if cache is None:
            page, spare = 64, 64
            cache = self.paged_cache(len(prompts), sum(-(-(n + new_tokens + spare) // page) * page for n in lengths), page)

        def best(logits):
            zero = torch.zeros(len(logits), device=device)
            return ops.sample_tokens(logits, zero, zero)[0].tolist()

        starts = cache.extend(lengths)
        packed = torch.cat([p.reshape(-1) for p in prompts]).to(device)
        for h, t in zip(history, best(self.forward_paged(packed, cache, starts))):
            h.append(t)
        while True:
            tokens, parents = [], []
            room = cache.free_positions() // cache.page // len(history) * cache.page  # of a sequence's pages still to be taken
            for h, n, length in zip(history, lengths, cache.length):
                left = n + new_tokens - len(h)  # to be generated yet
                if left < 1 or h[-1] < 0:
                    tokens.append([])
                    parents.append([])
                    continue
                more, follow = draft(list(h)) if left > 1 else ([], [])
                if len(more) != len(follow) or any(not -1 <= p < i for i, p in enumerate(follow)) or \
                        any(not 0 <= t < self.cfg.vocab for t in more):
                    raise ValueError("a draft has a token of the vocabulary and an earlier parent or -1 for each node")
                most = max(0, min(cache.max_len, self.max_len, -(-length // cache.page) * cache.page + room) - length - 1)
                tokens.append([h[-1], *more[:most]])
                parents.append([-1, *(p + 1 for p in follow[:most])])
            news = [len(t) for t in tokens]
            if not any(news):
                break
            cache.extend(news)
            took = best(self.forward_tree(torch.tensor([t for of in tokens for t in of], device=device), cache, parents))
            kept, first = [], 0
            for h, of, follow in zip(history, tokens, parents):
                path, node = [], 0 if of else -1
                while node >= 0:
                    path.append(node)
                    t = took[first + node]
                    h.append(t)
                    node = next((i for i, p in enumerate(follow) if p == node and of[i] == t and i > node), -1)
                kept.append(path)
                first += len(of)
            cache.keep(news, kept)
        out = torch.full((len(history), new_tokens), -1, dtype=torch.int64)
        for row, h, n in zip(out, history, lengths):
            new = h[n:n + new_tokens]
            row[:len(new)] = torch.tensor(new)
        return out.to(device)

    @torch.no_grad()
    def beam_search_paged(self, prompts: Sequence[torch.Tensor], new_tokens: int, beams: int, end: Optional[int] = None,
                          cache: Optional[PagedKVCache] = None):
        """The ``beams`` best continuations of each prompt by ``new_tokens`` tokens that a search with as many beams finds, from the
        best down: ``(tokens [prompts, beams, new_tokens], scores fp32 [prompts, beams])``, a score being the sum of the tokens' log
        probabilities.  A beam that takes the token ``end`` is over: ``end`` fills the rest and its score stays.  A request's
        beams share the pages of what they have in common.  ``cache``, if given, has ``beams`` sequences for each prompt.
        Where fewer continuations are left, scores are -inf and tokens -1."""
        device, n = self.embed.device, len(prompts)
        lengths = [int(p.numel()) for p in prompts]
        if not lengths or min(lengths) < 1 or new_tokens < 1 or not 1 <= beams <= 64:
            raise ValueError("prompts must hold a token at least, new_tokens be positive, and beams 1 to 64")
        if end is not None and not 0 <= end < self.cfg.vocab:
            raise ValueError(f"end must be a token of the {self.cfg.vocab}, got {end}")
        if cache is None:
            page = 64
            cache = self.paged_cache(n * beams, sum(-(-l // page) + beams * (-(-new_tokens // page) + 1) for l in lengths) * page, page)
        elif len(cache.length) != n * beams:
            raise ValueError(f"the cache must have {n * beams} sequences, {beams} for each prompt, got {len(cache.length)}")
        base = torch.arange(0, n * beams, beams, device=device).unsqueeze(1)
        scores = torch.full((n, beams), -math.inf, device=device)
        scores[:, 0] = 0
        starts = cache.extend([l if b == 0 else 0 for l in lengths for b in range(beams)])
        logits = self.forward_paged(torch.cat([p.reshape(-1) for p in prompts]).to(device), cache, starts)
        ended = None if end is None else torch.zeros(n, beams, dtype=torch.bool, device=device)
        history = torch.zeros(n, beams, 0, dtype=torch.int64, device=device)
        for step in range(new_tokens):
            if step:
                if self.cfg.window:
                    cache.trim(self.cfg.window, self.cfg.sinks)
                cache.extend([1] * (n * beams))
                # a beam that has ended, or never was, goes on with any token and stays as it is
                logits = self.forward_paged(history[:, :, -1].reshape(-1).clamp(min=0), cache)
            scores, parents, tokens = ops.beam_select(logits, scores, beams, ended, end or 0)
            alive = parents.clamp(min=0)
            history = torch.cat((history.gather(1, alive.unsqueeze(2).expand(-1, -1, step)), tokens.unsqueeze(2)), 2)
            history = torch.where((parents < 0).unsqueeze(2), -1, history)
            if step + 1 < new_tokens:
                cache.reorder((base + alive).reshape(-1).tolist())
            if end is not None:
                ended = ended.gather(1, alive) | (tokens == end)
        return history, scores
