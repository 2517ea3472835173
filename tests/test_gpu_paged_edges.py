"""The serving operators where several of their rules meet: the bits of decode attention's weights, chunks that pass the end of
their table, packed prompts whose positions are split, rows of logits past what registers hold.  Against plain 64-bit forms on the CPU (``paged_reference``)."""
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


# ---------------------------------------------------------------- the weights of one new token
def _pages_of(lens, kvh, dim, page, dtype, g, signs=False):
    width = max(-(-n // page) for n in lens)
    shape = (len(lens) * width, kvh, page, dim)
    k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g)
    v = torch.where(v < 0, -1.0, 1.0).to(dtype) if signs else v.to(dtype)
    return k.to(DEV), v.to(DEV), torch.randperm(shape[0], generator=g).view(len(lens), width).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 7), (128, 2, 4), (256, 1, 5)])
@pytest.mark.parametrize("lens", [[2, 3, 7, 31], [40, 129, 500, 1], [3000]])
def test_decode_keeps_the_weights_bits(dtype, dim, kvh, grp, lens):
    """Values of 1 and -1, whose sums cancel: a weight rounded once to the type would be off by half a step, and the output by
    much of that.  What the rounding leaves is added, rounded itself: half a step of half a step of the sum of magnitudes."""
    _say("decode weights", dtype, dim, kvh, grp, lens)
    g = torch.Generator().manual_seed(dim + len(lens))
    k, v, table = _pages_of(lens, kvh, dim, 16, dtype, g, signs=True)
    q = torch.randn(len(lens), kvh * grp, dim, generator=g).to(dtype).to(DEV)
    got = _ops().paged_decode_attention(q, k, v, table, _ints(lens), dim ** -0.5)
    half = ref.HALF_STEP[dtype]
    for b, n in enumerate(lens):
        rows_k, rows_v = (t[table[b].long()].cpu().transpose(1, 2).reshape(-1, kvh, dim)[:n].double() for t in (k, v))
        for h in range(kvh * grp):
            want, (out, size, rel, low) = ref.attention_row(q[b, h].cpu().double(), rows_k[:, h // grp], rows_v[:, h // grp], dim ** -0.5)
            tol = half * out + (half * half * (1 + half) + 1.01 * rel) * size + low + (2.0 ** -24 if dtype == F16 else 0.0)
            ref.check(got[b, h], want, tol, what=f"sequence {b} head {h}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 7), (128, 2, 4), (256, 1, 5)])
def test_decode_over_infinite_values(dtype, dim, kvh, grp):
    """An infinity in a value that is attended goes to its own column, with its sign, and two of different signs give NaN; the
    others keep their sums.  The first position of a sequence, whose weight may be a power of two, among them."""
    lens = [1, 5, 200, 2000]
    g = torch.Generator().manual_seed(dim)
    k, v, table = _pages_of(lens, kvh, dim, 16, dtype, g)
    for b, at in ((0, 0), (1, 0), (1, 4), (2, 33), (2, 199), (3, 0), (3, 1024), (3, 1999)):
        v[int(table[b, at // 16]), :, at % 16, 2 + at % 5] = math.inf if at % 2 else -math.inf
    for b, at in ((2, 7), (2, 150), (3, 5), (3, 1600)):
        v[int(table[b, at // 16]), :, at % 16, 9] = math.inf if at % 2 else -math.inf
    q = torch.randn(len(lens), kvh * grp, dim, generator=g).to(dtype).to(DEV)
    got = _ops().paged_decode_attention(q, k, v, table, _ints(lens), dim ** -0.5)
    ref.check(got, *ref.paged_attention(q, k, v, table, _ints(lens), None, dim ** -0.5))


# ---------------------------------------------------------------- chunks that pass the end of their table
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,grp,width", [(64, 7, 5), (128, 1, 5), (256, 4, 5), (128, 2, 60), (256, 1, 60)])
@pytest.mark.parametrize("bad", [False, True])
def test_chunks_past_the_end_of_their_table(dtype, dim, grp, width, bad):
    """A row sees the positions up to the one that the append gives it, as far as the table goes: also where the sequence's
    length passes the table's room and the last rows of the chunk have no place.  Wide tables split their positions.  ``bad``: an
    infinity in a value that only some of the rows see, whose rows are done again."""
    kvh, page = 2, 16
    room = width * page
    news = [4, 40, 9, 3, 5, 2]
    lens = [room + 2, room + 39, room, room - 1, room + 5000, 2 ** 31 - 1]
    _say("chunks past the table", dtype, dim, grp, width, bad)
    g = torch.Generator().manual_seed(dim + width)
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    pages = len(lens) * width
    k, v = (torch.randn(pages, kvh, page, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    table = torch.randperm(pages, generator=g).view(len(lens), width).to(torch.int32)
    nh = kvh * grp
    qkv = torch.randn(at[-1], (nh + 2 * kvh) * dim, generator=g).to(dtype).to(DEV)
    angle = torch.rand(room + 50, dim // 2, generator=g) * 6.3
    q = _ops().paged_rope_append(qkv, angle.cos().to(DEV), angle.sin().to(DEV), k, v, table.to(DEV), _ints(lens), _ints(at))
    q = torch.randn(q.shape, generator=g).to(dtype).to(DEV)  # (positions without an angle have zero queries)
    # which position each row has is the append's to say: the new keys are where it put them
    x, cos, sin = qkv.cpu().view(at[-1], -1, dim), angle.cos(), angle.sin()
    kc, vc = k.cpu(), v.cpu()
    for b, n in enumerate(news):
        for j in range(n):
            pos = lens[b] - n + j
            if pos >= room:
                continue
            page_of, row = int(table[b, pos // page]), pos % page
            assert torch.equal(vc[page_of, :, row], x[at[b] + j, nh + kvh:])
            want = ref.rotate(x[at[b] + j:at[b] + j + 1, nh:nh + kvh].double(), cos[pos:pos + 1], sin[pos:pos + 1], True)[0]
            assert ((kc[page_of, :, row].double() - want).abs() <= ref.HALF_STEP[dtype] * want.abs() + 2.0 ** -20).all()
    if bad:  # the table's last position of the first two sequences: the first row of the first chunk does not see it
        for b in (0, 1):
            v[int(table[b, -1]), 0, page - 1] = math.inf
        vc = v.cpu()
    got = _ops().paged_prompt_attention(q, k, v, table.to(DEV), _ints(lens), _ints(at), dim ** -0.5)
    qc = q.cpu().double()
    for b, n in enumerate(news):
        rows_k, rows_v = (t[table[b].long()].transpose(1, 2).reshape(room, kvh, dim).double() for t in (kc, vc))
        for j in range(n):
            sees = min(lens[b] - n + j + 1, room)
            for h in range(nh):
                want, bound = ref.attention_row(qc[at[b] + j, h], rows_k[:sees, h // grp], rows_v[:sees, h // grp], dim ** -0.5)
                if torch.isfinite(want).all():
                    ref.check(got[at[b] + j, h], want, ref.allowed(bound, dtype), what=f"sequence {b} row {j} head {h}")
                else:
                    assert not torch.isfinite(got[at[b] + j, h]).any()


# ---------------------------------------------------------------- packed prompts whose positions are split
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 1, 2), (64, 2, 1), (128, 1, 1), (128, 2, 1), (256, 1, 2), (256, 2, 1)])
@pytest.mark.parametrize("starts", [[0, 520], [0, 1, 300, 300, 1013], [7, 600, 640, 641]])
def test_packed_prompts_split_over_positions(dtype, dim, kvh, grp, starts):
    """Few heads over prompts of hundreds of tokens: workgroups take a part of the positions each and are joined.  Rows that
    see all of a part, some of it or nothing; rows of no sequence; an infinity, and a NaN, that only later rows see."""
    from mindpipe_amd import _lib
    rows, nh, scale = starts[-1] + 5, kvh * grp, dim ** -0.5
    _say("packed prompts, split", dtype, dim, kvh, grp, starts)
    assert _lib.load().mp_prompt_workspace_bytes(rows, nh, kvh, dim, len(starts) - 1, rows) > 0
    g = torch.Generator().manual_seed(rows + dim)
    qkv = (1.5 * torch.randn(rows, nh + 2 * kvh, dim, generator=g)).to(dtype).to(DEV)
    q, k, v = qkv[:, :nh], qkv[:, nh:nh + kvh], qkv[:, nh + kvh:]
    clean, tol = ref.prompt_attention(q, k, v, torch.tensor(starts), scale)
    got = _ops().prompt_attention(q, k, v, _ints(starts), scale)
    ref.check(got, clean, tol)
    assert torch.equal(got, _ops().prompt_attention(q, k, v, _ints(starts), scale))
    # one token of the longest sequence, past its first split, inside a tile
    first = max(range(len(starts) - 1), key=lambda b: starts[b + 1] - starts[b])
    at, end = starts[first] + 413, starts[first + 1]
    for value in (math.inf, math.nan):
        v[at, 0, 3], keep = value, v[at, 0, 3].clone()
        got = _ops().prompt_attention(q, k, v, _ints(starts), scale)
        v[at, 0, 3] = keep
        want = clean.clone()
        want[at:end, :grp, 3] = math.nan
        seen = torch.isfinite(want)
        ref.check(torch.where(seen, got.cpu().double(), 0.0), torch.where(seen, want, 0.0), tol, what=str(value))
        assert not torch.isfinite(got.cpu()[~seen]).any()


# ---------------------------------------------------------------- rows of logits past what registers hold
def _check_sample(logits, u, *filters):
    got, logp = _ops().sample_tokens(logits, u, *filters)
    want, wlogp = ref.sample(logits, u, *filters)
    assert torch.equal(got.cpu(), want), [(i, int(got[i]), int(want[i])) for i in (got.cpu() != want).nonzero().flatten().tolist()]
    fine = torch.isfinite(wlogp)
    assert torch.equal(torch.isfinite(logp.cpu()), fine)
    # a sum of `vocab` weights is off by half a unit of 2^-44 of the largest each, and the sum is at least that weight; a
    # token's own weight by half a unit, of its share exp(logp) of the sum (at least one weight of 1); rounded to fp32
    tol = 2.0 ** -23 * wlogp.abs() + 2.0 ** -44 * (logits.shape[1] + logits.shape[1] * torch.exp(-wlogp)) + 2.0 ** -48
    assert ((logp.cpu().double() - wlogp).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("vocab", [131072, 131073, 151936, 1 << 19])
@pytest.mark.parametrize("which", ["", "t", "tk", "tp", "tm", "tkp", "tkpm"])
def test_sample_rows_that_are_read_again(dtype, vocab, which):
    _say("sample", dtype, vocab, which)
    g = torch.Generator().manual_seed(vocab)
    rows = 4
    x = (torch.randn(rows, vocab + 8, generator=g) * 2).to(dtype)
    x[:2] *= 4
    f = [torch.rand(rows, generator=g) + 0.2, torch.randint(1, 3000, (rows,), generator=g, dtype=torch.int32),
         0.3 + 0.69 * torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.1]
    f = [t.to(DEV) if c in which else None for c, t in zip("tkpm", f)]
    x = x.to(DEV)
    u = torch.rand(rows, generator=g).to(DEV)
    _check_sample(x[:, :vocab], u, *f)            # rows in steps of eight values
    _check_sample(x[:, 3:3 + vocab], u, *f)       # rows that begin between them
    _check_sample(x[:, :vocab].contiguous(), u, *f)


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("vocab", [131072, 131073, 1 << 19])
def test_sample_flat_rows(dtype, vocab):
    """Every weight the largest: the sum is vocab 2^44, at 2^19 values 2^63.  Ties at every border go to the lowest indexes."""
    us = [0.0, 0.25, 0.5, 1 - 2.0 ** -23, 1 - 2.0 ** -24]
    n = len(us)
    x = torch.full((n, vocab), -2.5, device=DEV, dtype=dtype)
    x[:, 0] = -math.inf
    one = lambda a, dt=torch.float32: torch.full((n,), a, device=DEV, dtype=dt)  # noqa: E731
    u = torch.tensor(us, device=DEV)
    for f in ((None,) * 4, (one(0.7), one(vocab - 5, torch.int32), None, None), (None, None, one(0.5), None),
              (one(1.5), one(70000, torch.int32), one(0.75), one(1.0)), (one(0.0), None, None, None)):
        _check_sample(x, u, *f)
    x[:, 0] = -2.5
    _check_sample(x, u)
