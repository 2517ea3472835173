"""The operators of a paged key-value cache and of sampling against plain 64-bit forms on the CPU (``paged_reference``)."""
import math
import sys

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _ops():
    from mindpipe_amd import ops
    return ops


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(lens, kvh, dim, page, dtype, seed, layout="dense", fill=None, spare=2, extra=0):
    """Pools in which the sequences' pages lie in any order, what no sequence holds filled with ``fill``."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + spare, max(max(need), 1) + extra
    shape = (pages, kvh, page, dim)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    held = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = order.pop()
            held[table[b, i], :min(page, n - i * page)] = True
    if fill is not None:
        empty = ~held.to(DEV)[:, None, :, None].expand(shape)
        k[empty] = fill
        v[empty] = fill
    if layout == "positions":  # [pages, page, kvh, dim] in memory
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif layout == "both":     # keys and values of a page together
        both = torch.stack((k, v), 1).contiguous()
        k, v = both[:, 0], both[:, 1]
    return k, v, table.to(DEV), _ints(lens)


LENS = {"ones": [1, 1, 1], "tile": [31, 32, 33, 64, 65], "empty": [0, 5, 0], "page": [8, 16, 17, 127, 128, 129],
        "long": [1000, 3, 517], "one": [700]}


# ---------------------------------------------------------------- one new token per sequence
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 1), (64, 1, 7), (128, 2, 4), (128, 3, 1), (128, 1, 16), (256, 1, 5), (128, 1, 21),
                                         (256, 1, 16)])
@pytest.mark.parametrize("lens,page,layout", [("ones", 8, "dense"), ("tile", 8, "positions"), ("empty", 16, "dense"),
                                              ("page", 32, "both"), ("long", 16, "dense"), ("one", 64, "dense")])
def test_decode(dtype, dim, kvh, grp, lens, page, layout):
    _say("paged decode", dtype, dim, kvh, grp, lens, page, layout)
    k, v, table, ln = _cache(LENS[lens], kvh, dim, page, dtype, 1, layout, fill=float("nan"))
    q = (2 * torch.randn(len(LENS[lens]), kvh * grp, dim, generator=torch.Generator().manual_seed(2))).to(dtype).to(DEV)
    got = _ops().paged_decode_attention(q, k, v, table, ln, dim ** -0.5)
    want, tol = ref.paged_attention(q, k, v, table, ln, None, dim ** -0.5)
    ref.check(got, want, tol)
    assert torch.equal(got, _ops().paged_decode_attention(q, k, v, table, ln, dim ** -0.5))


def test_decode_batch_of_many():
    """More sequences than a wave has lanes, most of them empty or short."""
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 40, (150,), generator=g)]
    lens[3], lens[140] = 900, 2000
    k, v, table, ln = _cache(lens, 1, 64, 16, BF16, 6)
    q = torch.randn(150, 2, 64, generator=g).to(BF16).to(DEV)
    got = _ops().paged_decode_attention(q, k, v, table, ln, 0.125)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, None, 0.125))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_bad_pages_and_lengths(dtype):
    """Page numbers outside the pool are empty pages; lengths past the table's room or below zero are held to it."""
    k, v, table, ln = _cache([200, 90, 64, 40], 2, 128, 16, dtype, 3)
    table[0, 2], table[0, 5], table[1, :], table[2, 0] = -1, k.shape[0], 1 << 30, -(1 << 31)
    ln[2], ln[3] = 100000, -7
    table[2, 1:] = table[0, 0]
    q = torch.randn(4, 8, 128, device=DEV).to(dtype)
    got = _ops().paged_decode_attention(q, k, v, table, ln, 0.1)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, None, 0.1))
    assert not got[1].any() and not got[3].any()


def test_decode_extreme_scores():
    """Scores that rise along the sequence (the maximum moves in every tile), large ones, and a scale of zero."""
    k, v, table, ln = _cache([300], 1, 128, 16, F16, 4)
    for p in range(300):
        k[int(table[0, p // 16]), 0, p % 16] *= p / 40.0
    q = torch.randn(1, 4, 128, device=DEV, dtype=F16) * 4
    for scale in (0.3, -0.3, 0.0):
        got = _ops().paged_decode_attention(q, k, v, table, ln, scale)
        ref.check(got, *ref.paged_attention(q, k, v, table, ln, None, scale), what=str(scale))


def test_decode_strided_queries_and_far_pages():
    """Pools of more than 2^31 values: offsets pass 32 bits.  Only the pages used are written."""
    pages = (1 << 31) // (8 * 128 * 128) + 40
    k = torch.empty(pages, 8, 128, 128, device=DEV, dtype=BF16)
    v = torch.empty_like(k)
    table = _ints([[pages - 1, 3, pages - 20, pages // 2 + 7]])
    for p in table[0].tolist():
        k[p], v[p] = torch.randn(8, 128, 128, device=DEV), torch.randn(8, 128, 128, device=DEV)
    qkv = torch.randn(1, 16 + 16, 128, device=DEV).to(BF16)
    q = qkv[:, 4:20]
    got = _ops().paged_decode_attention(q, k, v, table, _ints([450]), 0.09)
    few = table[0].long()
    want, tol = ref.paged_attention(q, k[few], v[few], _ints([[0, 1, 2, 3]]), _ints([450]), None, 0.09)
    ref.check(got, want, tol)
    # and an append there
    cos, sin = torch.rand(600, 64, device=DEV), torch.rand(600, 64, device=DEV)
    new = torch.randn(2, 32 * 128, device=DEV).to(BF16)
    args = (k[few], v[few], _ints([[0, 1, 2, 3]]), _ints([257]), _ints([0, 2]), True)
    wq, wk, wv = ref.append(new, cos, sin, *args)
    _ops().paged_rope_append(new, cos, sin, k, v, table, _ints([257]), _ints([0, 2]), True)
    assert (k[few].cpu().double() - wk).abs().max() <= 2.0 ** -8 * wk.abs().max()
    assert torch.equal(v[few].cpu().double(), wv)


# ---------------------------------------------------------------- prompts
STARTS = {"one": [0, 1], "short": [0, 5, 5, 6, 23], "tile": [0, 64, 129], "mixed": [0, 1, 1, 140, 141, 207]}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 1), (64, 1, 7), (128, 2, 4), (128, 3, 1), (256, 1, 5), (128, 1, 21)])
@pytest.mark.parametrize("starts", list(STARTS))
def test_prompt(dtype, dim, kvh, grp, starts):
    _say("prompt", dtype, dim, kvh, grp, starts)
    at = STARTS[starts]
    rows = at[-1] + 3  # three rows behind the last sequence
    qkv = (1.5 * torch.randn(rows, kvh * (grp + 2), dim, generator=torch.Generator().manual_seed(7))).to(dtype).to(DEV)
    q, k, v = qkv[:, :kvh * grp], qkv[:, kvh * grp:-kvh], qkv[:, -kvh:]
    got = _ops().prompt_attention(q, k, v, _ints(at), dim ** -0.5)
    want, tol = ref.prompt_attention(q, k, v, torch.tensor(at), dim ** -0.5)
    ref.check(got, want, tol)
    assert torch.equal(got, _ops().prompt_attention(q, k, v, _ints(at), dim ** -0.5))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp,page", [(64, 1, 7, 8), (128, 2, 4, 16), (128, 2, 1, 64), (256, 1, 5, 32)])
@pytest.mark.parametrize("news,ctxs", [([3, 1, 0, 40], [100, 0, 9, 31]), ([130], [260]), ([17, 64], [0, 15]), ([5], [1000])])
def test_paged_prompt(dtype, dim, kvh, grp, page, news, ctxs):
    _say("paged prompt", dtype, dim, kvh, grp, page, news, ctxs)
    lens = [n + c for n, c in zip(news, ctxs)]
    k, v, table, ln = _cache(lens, kvh, dim, page, dtype, 8, "positions" if page == 16 else "dense", fill=float("nan"), extra=1)
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    q = (1.5 * torch.randn(at[-1] + 2, kvh * grp, dim, generator=torch.Generator().manual_seed(9))).to(dtype).to(DEV)
    got = _ops().paged_prompt_attention(q, k, v, table, ln, _ints(at), dim ** -0.5)
    want, tol = ref.paged_attention(q, k, v, table, ln, torch.tensor(at), dim ** -0.5)
    ref.check(got, want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_later_tokens_do_not_reach_back(dtype, dim):
    """NaN and infinities in a token's key and value reach the rows that see it and no others, where the tile is shared."""
    rows, at = 90, 41
    qkv = torch.randn(rows, 6, dim, device=DEV).to(dtype)
    q, k, v = qkv[:, :4], qkv[:, 4:5], qkv[:, 5:]
    starts = _ints([0, 70, rows])
    clean = _ops().prompt_attention(q, k, v, starts, dim ** -0.5)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in (k, v):
            keep = t[at].clone()
            t[at] = bad
            got = _ops().prompt_attention(q, k, v, starts, dim ** -0.5)
            t[at] = keep
            assert torch.isfinite(got[:at]).all() and torch.isfinite(got[70:]).all()
            off = (got[:at].float() - clean[:at].float()).abs().max()
            # the shared tile is added position by position: another order of the same fp32 sums, a step of the output
            assert off <= 4 * ref.HALF_STEP[dtype] * clean.abs().max().float()
            if bad != bad:
                assert torch.isnan(got[at:70]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_rows_over_long_contexts(dtype, dim):
    """Positions split over workgroups and joined: rows that see all of a split, a part of it, or nothing, missing pages, and a
    NaN that only the last rows see."""
    lens, news = [2500, 700, 30, 0], [20, 1, 30, 0]
    k, v, table, ln = _cache(lens, 2, dim, 32, dtype, 41)
    table[0, 3], table[1, 2] = -1, 1 << 20
    starts = torch.tensor([0, 20, 21, 51, 51], dtype=torch.int32)
    q = (1.5 * torch.randn(54, 6, dim, generator=torch.Generator().manual_seed(42))).to(dtype).to(DEV)
    args = (q, k, v, table, ln, starts.to(DEV), dim ** -0.5)
    got = _ops().paged_prompt_attention(*args)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, starts, dim ** -0.5))
    assert torch.equal(got, _ops().paged_prompt_attention(*args))
    page, row = int(table[0, 2490 // 32]), 2490 % 32
    v[page, 1, row] = float("nan")
    k[page, 0, row] = float("nan")
    got = _ops().paged_prompt_attention(*args)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, starts, dim ** -0.5))
    assert torch.isfinite(got[:10]).all() and torch.isnan(got[10:20]).all()


def test_paged_prompt_bad_pages_and_short_lengths():
    """Missing pages, lengths smaller than the number of new tokens, and lengths past the table's room."""
    k, v, table, ln = _cache([90, 40, 64], 2, 128, 16, F16, 11)
    table[0, 1], table[0, 3] = -5, 1 << 29
    ln[1], ln[2] = 7, 5000
    table[2, 4:] = table[0, 0]
    q = torch.randn(60, 4, 128, device=DEV, dtype=F16)
    starts = torch.tensor([0, 30, 50, 60], dtype=torch.int32)
    got = _ops().paged_prompt_attention(q, k, v, table, ln, starts.to(DEV), 0.1)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, starts, 0.1))
    assert not got[30:43].any()


def test_starts_of_any_kind_stay_inside():
    """Starts that descend or pass the rows: what they make of the rows is open, but nothing else is touched."""
    q = torch.randn(20, 2, 64, device=DEV, dtype=F16)
    k = torch.randn(20, 1, 64, device=DEV, dtype=F16)
    for at in ([5, 2, 30], [-4, 10, 7], [0, 1000, 20], [25, 30, 40]):
        out = _ops().prompt_attention(q, k, k, _ints(at), 0.1)
        assert out.shape == q.shape
    torch.cuda.synchronize()


# ---------------------------------------------------------------- rotation and append
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,nh,rotary", [(128, 2, 8, 128), (64, 1, 3, 64), (256, 2, 2, 64), (128, 40, 40, 128), (80, 1, 2, 32)])
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("news,ctxs", [([1, 1, 1], [0, 15, 130]), ([7, 0, 33, 1], [3, 4, 0, 64]), (None, [1, 16, 17, 100])])
def test_append(dtype, dim, kvh, nh, rotary, pairs, news, ctxs):
    _say("append", dtype, dim, kvh, nh, rotary, pairs, news)
    lens = ctxs if news is None else [n + c for n, c in zip(news, ctxs)]
    k, v, table, ln = _cache(lens, kvh, dim, 16, dtype, 12, "both" if dim == 64 else "dense")
    starts = None
    rows = len(lens)
    if news is not None:
        at = [0]
        for n in news:
            at.append(at[-1] + n)
        starts, rows = _ints(at), at[-1] + 2  # two rows behind the last sequence
    g = torch.Generator().manual_seed(13)
    wide = torch.randn(rows, (nh + 2 * kvh) * dim + 16, generator=g).to(dtype).to(DEV)
    qkv = wide[:, 8:-8]
    angle = torch.rand(max(lens) + 1, rotary // 2, generator=g) * 6.3
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    wq, wk, wv = ref.append(qkv, cos, sin, k, v, table, lens, starts, pairs)
    got = _ops().paged_rope_append(qkv, cos, sin, k, v, table, ln, starts, pairs)
    # two products and a sum in fp32, a rounding to the type: half a step and 2^-22 of the pair's magnitude
    for have, want in ((got, wq), (k, wk)):
        off = (have.cpu().double() - want).abs()
        size = qkv.abs().max().item() * 1.5
        assert (off <= ref.HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * size + 2.0 ** -24).all()
    assert torch.equal(v.cpu().double(), wv)
    if news is not None:
        assert not got[-2:].any()


def test_append_leaves_the_rest_alone():
    """Bad pages, positions without an angle, past the table or before the start: nothing is written, queries are zero
    where there is no angle."""
    k, v, table, ln = _cache([40, 40, 40, 40], 1, 64, 8, F16, 14)
    table[0, 1], table[1, 1] = -1, k.shape[0]
    ln = _ints([10, 10, 30, 41])       # the third has no angle, the fourth no room
    before = k.clone(), v.clone()
    cos, sin = torch.ones(25, 32, device=DEV), torch.zeros(25, 32, device=DEV)
    big = torch.ones(60, 32, device=DEV), torch.zeros(60, 32, device=DEV)
    qkv = torch.randn(4, 4 * 64, device=DEV, dtype=F16)
    q = _ops().paged_rope_append(qkv, cos, sin, k, v, table, ln)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    assert torch.equal(q[:2], qkv.view(4, 4, 64)[:2, :2]) and not q[2:].any()
    q = _ops().paged_rope_append(qkv, *big, k, v, table, _ints([0, -5, 10, 41]))
    assert not q[:2].any() and torch.equal(q[3], qkv.view(4, 4, 64)[3, :2])
    page = int(table[2, 1])
    assert torch.equal(k[page, 0, 1], qkv.view(4, 4, 64)[2, 2])
    k[page, 0, 1], v[page, 0, 1] = before[0][page, 0, 1], before[1][page, 0, 1]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


# ---------------------------------------------------------------- sampling
def _check_sample(logits, u, *filters):
    got, logp = _ops().sample_tokens(logits, u, *filters)
    want, wlogp = ref.sample(logits, u, *filters)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero().flatten().tolist()[:8]
    fine = torch.isfinite(wlogp)
    assert torch.equal(torch.isfinite(logp.cpu()), fine)
    # weights are whole numbers of 2^-44 (a token's own may be small), the logarithm is rounded to fp32
    tol = 2.0 ** -23 * wlogp.abs() + 2.0 ** -44 * torch.exp(-wlogp) * 64 + 1e-9
    assert ((logp.cpu().double() - wlogp).abs()[fine] <= tol[fine]).all()


def _filters(rows, g, which):
    f = [torch.rand(rows, generator=g) * 1.4 + 0.1, torch.randint(1, 60, (rows,), generator=g, dtype=torch.int32),
         torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.3]
    for t, off in zip(f, (0, 0, 1, 0)):
        t[torch.rand(rows, generator=g) < 0.15] = off
    return [t.to(DEV) if c in which else None for c, t in zip("tkpm", f)]


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 511, 512, 513, 4097, 32000])
@pytest.mark.parametrize("which", ["", "t", "tk", "tp", "tm", "kp", "tkpm"])
def test_sample(dtype, vocab, which):
    _say("sample", dtype, vocab, which)
    g = torch.Generator().manual_seed(vocab)
    rows = 9
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(DEV)
    _check_sample(logits, torch.rand(rows, generator=g).to(DEV), *_filters(rows, g, which))


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
def test_sample_ties_and_odd_values(dtype):
    """Equal values at every border, -0 beside 0, masked, infinite and NaN logits, rows that allow one token or none."""
    vocab = 3000
    g = torch.Generator().manual_seed(21)
    rows = [torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=g).float(),
            torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0),
            torch.full((vocab,), -math.inf), torch.full((vocab,), math.nan),
            torch.where(torch.rand(vocab, generator=g) < 0.99, -math.inf, 1.5),
            torch.randint(-2, 3, (vocab,), generator=g).float() * 1000, torch.randn(vocab, generator=g)]
    rows[7][[5, 900]] = math.inf
    one = torch.full((vocab,), -math.inf)
    one[1234] = -5.0
    holes = torch.randn(vocab, generator=g)
    holes[::3] = math.nan
    low = torch.full((vocab,), float(torch.finfo(dtype).min))
    low[77] = 0.0
    x = torch.stack([*rows, one, holes, low]).to(dtype).to(DEV)
    n = len(x)
    for u in (0.0, 0.3, 0.5, 1 - 2.0 ** -24):
        us = torch.full((n,), u, device=DEV)
        for f in ((None,) * 4, (1.0, 10, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (1.3, 700, 0.9, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 1, 0.0, 0.5),
                  (0.0, 5, 0.5, 0.1), (1.0, 0, 0.0, 0.0), (1e-3, 100, 0.99, 1e-4), (50.0, 2999, 0.999, 0.99), (1.0, 5000, 1.0, 2.0)):
            f = [None if a is None else torch.full((n,), a, device=DEV, dtype=torch.int32 if i == 1 else torch.float32)
                 for i, a in enumerate(f)]
            _check_sample(x, us, *f)


def test_sample_outside_u_and_strided_rows():
    wide = torch.randn(6, 1100, device=DEV, dtype=BF16)
    x = wide[:, 3:1004]
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, math.nan, 0.25], device=DEV)
    got, _ = _ops().sample_tokens(x, u)
    want, _ = ref.sample(x, torch.tensor([0.0, 1.0, 1.0, 0.0, 0.0, 0.25]))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
def test_sample_large_vocabulary(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(24, 128257, generator=g) * 2).to(dtype)
    x[:6] *= 8
    _check_sample(x.to(DEV), torch.rand(24, generator=g).to(DEV), *_filters(24, g, "tkpm"))


# ---------------------------------------------------------------- streams, graphs, registration
def test_steps_on_another_stream_and_in_graphs():
    """A step (append, attention, token) captured twice, over caches of its own: replays between eager work on grown
    lengths and new inputs give the eager step's bits."""
    ops = _ops()
    b, nh, kvh, dim, vocab = 3, 8, 2, 128, 1000
    cos, sin = torch.rand(300, 64, device=DEV), torch.rand(300, 64, device=DEV)

    def make(seed):
        k, v, table, ln = _cache([250, 120, 9], kvh, dim, 16, BF16, seed)
        s = {"k": k, "v": v, "table": table, "ln": ln, "qkv": torch.randn(b, (nh + 2 * kvh) * dim, device=DEV).to(BF16),
             "head": torch.randn(nh * dim, vocab, device=DEV) * 0.1, "u": torch.rand(b, device=DEV),
             "t": torch.full((b,), 0.8, device=DEV), "kk": torch.full((b,), 50, device=DEV, dtype=torch.int32)}
        return s

    def step(s):
        q = ops.paged_rope_append(s["qkv"], cos, sin, s["k"], s["v"], s["table"], s["ln"])
        o = ops.paged_decode_attention(q, s["k"], s["v"], s["table"], s["ln"], dim ** -0.5)
        p = ops.paged_prompt_attention(q, s["k"], s["v"], s["table"], s["ln"], torch.arange(b + 1, device=DEV, dtype=torch.int32),
                                       dim ** -0.5)
        return o, p, *ops.sample_tokens(o.float().view(b, -1) @ s["head"], s["u"], s["t"], s["kk"])

    states, graphs = [make(1), make(2)], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for s in states:
        s["ln"].copy_(_ints([200, 100, 3]))
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    for i in range(4):
        for s, (graph, out) in zip(states, graphs):
            s["ln"] += 1
            s["qkv"].normal_()
            s["u"].uniform_()
            graph.replay()
            got = [t.clone() for t in out]
            k = s["k"].clone()
            want = step(s)
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(got, want)) and torch.equal(k, s["k"])
            want64, tol = ref.paged_attention(ops.paged_rope_append(s["qkv"], cos, sin, s["k"], s["v"], s["table"], s["ln"]),
                                              s["k"], s["v"], s["table"], s["ln"], None, dim ** -0.5)
            ref.check(got[0], want64, tol)
            ref.check(got[1], want64, tol)


def test_registered_operators():
    """opcheck of the registrations, the mutation of the pools among them, and a traced call."""
    ops = _ops()
    k, v, table, ln = _cache([20, 5], 1, 64, 8, F16, 31)
    cos, sin = torch.rand(30, 32, device=DEV), torch.rand(30, 32, device=DEV)
    qkv, q = torch.randn(2, 4 * 64, device=DEV, dtype=F16), torch.randn(2, 2, 64, device=DEV, dtype=F16)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.mindpipe_amd_serve.paged_rope_append.default, (qkv, cos, sin, k, v, table, ln), test_utils=tests)
    torch.library.opcheck(torch.ops.mindpipe_amd_serve.paged_decode_attention.default, (q, k, v, table, ln, 0.1), test_utils=tests)
    torch.library.opcheck(torch.ops.mindpipe_amd_serve.paged_prompt_attention.default,
                          (q, k, v, table, ln, _ints([0, 1, 2]), 0.1), test_utils=tests)
    torch.library.opcheck(torch.ops.mindpipe_amd_serve.prompt_attention.default, (q, q[:, :1], q[:, 1:], _ints([0, 2]), 0.1),
                          test_utils=tests)
    torch.library.opcheck(torch.ops.mindpipe_amd_serve.sample_tokens.default, (qkv, torch.rand(2, device=DEV)), test_utils=tests)

    def f(qkv, k, v):
        q = ops.paged_rope_append(qkv, cos, sin, k, v, table, ln)
        return ops.paged_decode_attention(q, k, v, table, ln, 0.1)

    k2, v2 = k.clone(), v.clone()
    want = f(qkv, k, v)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(qkv, k2, v2)
    assert torch.equal(got, want) and torch.equal(k, k2) and torch.equal(v, v2)


def test_gradients_are_refused():
    ops = _ops()
    q = torch.randn(4, 2, 64, device=DEV, dtype=F16, requires_grad=True)
    out = ops.prompt_attention(q, q[:, :1].detach(), q[:, 1:].detach(), _ints([0, 4]), 0.1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        out.sum().backward()


# ---------------------------------------------------------------- calls at the edges
@pytest.mark.parametrize("paged", [False, True])
def test_rows_before_the_first_sequence(paged):
    """Rows before the first sequence are no sequence's, as those behind the last: zeros, over memory that held other values."""
    rows, nh, kvh, dim = 300, 4, 2, 64
    starts = torch.tensor([140, 150, 260], dtype=torch.int32)
    q = torch.randn(rows, nh, dim, device=DEV, dtype=F16)
    for _ in range(2):
        torch.full((rows, nh, dim), math.nan, device=DEV, dtype=F16)  # what the allocator hands out next
        if paged:
            k, v, table, ln = _cache([30, 200], kvh, dim, 16, F16, 41)
            got = _ops().paged_prompt_attention(q, k, v, table, ln, starts.to(DEV), 0.1)
            want, tol = ref.paged_attention(q[140:260], k, v, table, ln, starts - 140, 0.1)
        else:
            k, v = torch.randn(2, rows, kvh, dim, device=DEV, dtype=F16).unbind()
            got = _ops().prompt_attention(q, k, v, starts.to(DEV), 0.1)
            want, tol = ref.prompt_attention(q[140:260], k[140:260], v[140:260], starts - 140, 0.1)
        ref.check(got[140:260], want, tol)
        assert not got[:140].any() and not got[260:].any()


def test_sample_temperatures_of_every_size():
    """Temperatures and logits whose quotients, or differences, pass the range of fp32."""
    g = torch.Generator().manual_seed(51)
    vocab = 2000
    ties, small = torch.zeros(vocab), torch.randn(vocab, generator=g)
    big = (torch.rand(vocab, generator=g) * 2 - 1) * 3e38
    two = torch.where(torch.rand(vocab, generator=g) < 0.5, 3e38, -3e38)
    x = torch.stack([ties, small, big, two]).to(DEV)
    for t in (1e-44, 1e-38, 1e-30, 1e30, 5e37, 2e38, math.inf):
        for k, p in ((0, 1.0), (1, 1.0), (7, 1.0), (1500, 1.0), (0, 0.6), (1500, 0.99)):
            f = [torch.full((4,), a, device=DEV, dtype=torch.int32 if i == 1 else torch.float32) for i, a in enumerate((t, k, p))]
            _say("temperature", t, k, p)
            _check_sample(x, torch.tensor([0.99, 0.7, 0.6, 0.8], device=DEV), *f)


def test_workspaces_that_are_too_small_are_refused():
    import ctypes
    from mindpipe_amd import _lib
    lib = _lib.load()
    k, v, table, ln = _cache([400, 30], 2, 64, 16, F16, 61)
    q = torch.randn(2, 4, 64, device=DEV, dtype=F16)
    out, ws = torch.empty_like(q), torch.empty(1 << 24, device=DEV, dtype=torch.uint8)
    cache = _lib.PAGES.pack(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], 16, table.data_ptr(),
                            table.shape[1])
    starts, at = _ints([0, 1, 2]), torch.cuda.current_stream().cuda_stream
    need = lib.mp_paged_decode_workspace_bytes(2, 4, 2, 64)
    also = lib.mp_prompt_workspace_bytes(2, 4, 2, 64, 2, table.shape[1] * 16 * 40)
    assert need > 0 and also > 0
    decode = lambda scale, n: lib.mp_paged_decode_attention(  # noqa: E731
        q.data_ptr(), 256, 64, 2, 4, 2, 64, cache, ln.data_ptr(), scale, out.data_ptr(), 0, ws.data_ptr(), n, at)
    assert decode(0.1, need - 1) == 6 and decode(0.1, need) == 0
    want, tol = ref.paged_attention(q, k, v, table, ln, None, 0.1)
    torch.cuda.synchronize()
    ref.check(out, want, tol)
    for scale in (math.nan, math.inf, 3e38):
        assert decode(scale, need) == 5
    wide = table.repeat(1, 40)
    cache = _lib.PAGES.pack(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], 16, wide.data_ptr(),
                            wide.shape[1])
    prompt = lambda scale, n: lib.mp_paged_prompt_attention(  # noqa: E731
        q.data_ptr(), 256, 64, 2, 4, 2, 64, cache, ln.data_ptr(), starts.data_ptr(), 2, scale, out.data_ptr(), 0, ws.data_ptr(),
        n, at)
    assert prompt(0.1, also - 1) == 6 and prompt(0.1, also) == 0 and prompt(3e38, also) == 5
    torch.cuda.synchronize()
    ref.check(out, want, tol)


def test_calls_on_two_streams_at_once():
    """Two streams with their own calls under way together: each gets what it gets alone."""
    ops = _ops()
    calls = []
    for seed, lens in ((71, [3000, 10, 900]), (72, [50, 4000, 1])):
        k, v, table, ln = _cache(lens, 2, 128, 16, BF16, seed)
        q = torch.randn(3, 8, 128, device=DEV).to(BF16)
        calls.append((q, k, v, table, ln))
    starts = _ints([0, 1, 2, 3])
    run = lambda c: (ops.paged_decode_attention(*c, 0.1), ops.paged_prompt_attention(*c, starts, 0.1))  # noqa: E731
    alone = [run(c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(calls[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, alone[i]))


def test_append_tells_autograd_of_the_pools():
    """A backward that saved a pool before an append notices; tensors of inference mode, which keep no count, are taken."""
    ops = _ops()
    k, v, table, ln = _cache([20, 5], 1, 64, 8, F16, 81)
    cos, sin = torch.rand(30, 32, device=DEV), torch.rand(30, 32, device=DEV)
    qkv = torch.randn(2, 4 * 64, device=DEV, dtype=F16)
    w = torch.ones_like(k, requires_grad=True)
    y = (w * k).sum()
    ops.paged_rope_append(qkv, cos, sin, k, v, table, ln)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    want = k.clone()
    with torch.inference_mode():
        k2, v2 = k.clone(), v.clone()
        q = ops.paged_rope_append(qkv, cos, sin, k2, v2, table, ln)
        assert torch.equal(k2, want) and q.shape == (2, 2, 64)


def test_sequences_that_share_pages():
    """Two sequences and one of them twice over the same first pages, as behind a common prefix; decode and chunks."""
    k, v, table, ln = _cache([200, 70, 40], 2, 128, 16, F16, 91)
    table[1, :4] = table[0, :4]
    table[2] = table[0]
    starts = _ints([0, 20, 21, 45])
    q = torch.randn(45, 6, 128, device=DEV, dtype=F16)
    got = _ops().paged_prompt_attention(q, k, v, table, ln, starts, 0.09)
    ref.check(got, *ref.paged_attention(q, k, v, table, ln, starts, 0.09))
    got = _ops().paged_decode_attention(q[:3], k, v, table, ln, 0.09)
    ref.check(got, *ref.paged_attention(q[:3], k, v, table, ln, None, 0.09))


def test_chunks_over_far_pages_and_repeated_keys():
    """Chunks over pools whose offsets pass 32 bits; prompts whose keys and values are one row, or one head, repeated."""
    pages = (1 << 31) // (8 * 128 * 128) + 40
    k = torch.empty(pages, 8, 128, 128, device=DEV, dtype=BF16)
    v = torch.empty_like(k)
    table = _ints([[pages - 1, 3, pages - 20, pages // 2 + 7]])
    few = table[0].long()
    k[few], v[few] = (torch.randn(4, 8, 128, 128, device=DEV).to(BF16) for _ in range(2))
    q = torch.randn(30, 16, 128, device=DEV).to(BF16)
    got = _ops().paged_prompt_attention(q, k, v, table, _ints([450]), _ints([0, 30]), 0.09)
    ref.check(got, *ref.paged_attention(q, k[few], v[few], _ints([[0, 1, 2, 3]]), _ints([450]), _ints([0, 30]), 0.09))
    del k, v
    starts = torch.tensor([0, 70, 100], dtype=torch.int32)
    q, one, head = torch.randn(100, 4, 64, device=DEV, dtype=F16), torch.randn(1, 2, 64, device=DEV, dtype=F16), \
        torch.randn(100, 1, 64, device=DEV, dtype=F16)
    for kv in (one.expand(100, 2, 64), head.expand(100, 2, 64)):
        got = _ops().prompt_attention(q, kv, kv, starts.to(DEV), 0.1)
        ref.check(got, *ref.prompt_attention(q, kv, kv, starts, 0.1))
