"""Beam selection and the moves of a paged cache's contents against plain forms on the CPU (``masked_reference``)."""
import math
import sys

import pytest
import torch

import masked_reference as mref
import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


def _say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _ops():
    from mindpipe_amd import ops
    return ops


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- beams
def _logits(rows, vocab, dtype, seed, spread=1.7):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    stand = torch.randint(0, vocab, (rows, 12), generator=g)
    return x.scatter_add_(1, stand, 6.0 + 2.0 * torch.randn(rows, 12, generator=g)).to(dtype).to(DEV)


def _select(logits, scores, count, ended=None, pad=0):
    """The kernel's answer, checked.  Beams and tokens are those of the totals in 64 bits; a score is a total rounded to fp32 once,
    half a step of it, and the total's own error (2^-34 of the sum of exponentials) is far below that."""
    got = _ops().beam_select(logits, scores, count, ended, pad)
    best, parent, token = mref.beams(logits, scores.cpu(), count, None if ended is None else ended.cpu(), pad)
    assert torch.equal(got[1].cpu(), parent) and torch.equal(got[2].cpu(), token)
    ref.check(got[0], best, torch.where(torch.isfinite(best), 2.0 ** -24 * best.abs() + 2.0 ** -34, 0.0))
    again = _ops().beam_select(logits, scores, count, ended, pad)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("batch,beams,vocab,count", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 4, 1000, 8), (3, 3, 4097, 6), (1, 4, 32000, 8),
                                                     (5, 2, 50257, 4), (1, 64, 2049, 64), (2, 16, 16384, 32), (1, 2, 1 << 19, 64)])
def test_select(dtype, batch, beams, vocab, count):
    _say("beam select", dtype, batch, beams, vocab, count)
    x = _logits(batch * beams, vocab, dtype, vocab)
    g = torch.Generator().manual_seed(3)
    scores = (-9.0 - 2.0 * torch.rand(batch, beams, generator=g)).to(DEV)
    _select(x, scores, count)
    ended = (torch.rand(batch, beams, generator=g) < 0.4).to(DEV)
    _select(x, scores, count, ended, vocab - 1)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_select_many_rows(dtype):
    """So many rows that a part is as large as it gets."""
    x = _logits(300, 33000, dtype, 5)
    _select(x, (-torch.rand(75, 4, generator=torch.Generator().manual_seed(1))).to(DEV), 8)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_rows_and_strides(dtype):
    """Rows that do not start at 16 bytes, and rows of a wider tensor."""
    wide = _logits(12, 3001, dtype, 6)
    for x in (wide[:, 1:], wide[:, :2999], wide[:, 8:2008], wide[::2, 3:1000]):
        _select(x, torch.zeros(x.shape[0] // 2, 2, device=DEV) - torch.arange(2, device=DEV), 4)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_equal_and_ordered_values(dtype):
    """Equal values everywhere, few distinct ones, ascending and descending ones: more candidates than the lists hold."""
    v = 9000
    rows = torch.stack((torch.zeros(v), torch.full((v,), -3.0), torch.arange(v) % 7 * 0.5, torch.arange(v) / 1024.0,
                        -torch.arange(v) / 1024.0, (torch.arange(v) > 8000).float(), torch.arange(v) // 600 * 1.0,
                        torch.where(torch.arange(v) == 4000, 2.0, -0.0))).to(dtype).to(DEV)
    for i in range(8):  # alone, and beside each other
        _select(rows[i:i + 1], torch.zeros(1, 1, device=DEV), 64)
        _select(rows[i:i + 1], torch.zeros(1, 1, device=DEV), 3)
    _select(rows, torch.tensor([[0.0, -0.7, -1.3, 0.1], [-0.2, 3.0, -2.0, 1.0]], device=DEV), 64)
    _select(rows[[0, 0, 5, 5]], torch.zeros(2, 2, device=DEV), 40)  # equal beams: the lowest first


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("beams,count", [(5, 60), (40, 64), (64, 2)])
def test_select_equal_beams(dtype, beams, count):
    """Equal totals in many lists, from a few hundred of them to more than LDS holds: those of the lowest beams, then tokens."""
    x = torch.zeros(beams, 9000, dtype=dtype, device=DEV)
    x[:, 17:8999:2] = -1.0
    got = _select(x, torch.zeros(1, beams, device=DEV), count)
    assert (got[1] == 0).all() and got[2][0].tolist() == [*range(17), *range(18, 9000, 2)][:count]
    _select(x, -0.5 * (torch.arange(beams, device=DEV) % 2)[None].float(), count)
    ended = torch.arange(beams, device=DEV)[None] < beams - 1
    _select(x, torch.zeros(1, beams, device=DEV), count, ended, 5)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_what_is_masked(dtype):
    """-inf, NaN and infinities among the logits and scores, rows of nothing else, fewer candidates than are asked for."""
    x = _logits(6, 5000, dtype, 8)
    x[0, 7:] = -INF
    x[1, :] = -INF
    x[2, ::3] = float("nan")
    x[3, :] = float("nan")
    x[4, 100], x[4, 4000] = INF, INF
    x[5, 1:] = torch.finfo(dtype).min
    scores = torch.tensor([[-1.0, -2.0, -1.5, -0.5, -3.0, -2.5]], device=DEV)
    _select(x, scores, 16)
    _select(x[:2], scores[:, :2], 64)
    got = _select(x[1:2], scores[:, :1], 4)
    assert (got[0] == -INF).all() and (got[1] == -1).all() and (got[2] == -1).all()
    for bad in (-INF, float("nan")):
        scores[0, 0] = bad
        _select(x, scores.nan_to_num(nan=-INF, neginf=-INF), 16)
        got = _ops().beam_select(x, scores, 16)
        assert not (got[1] == 0).any()
    first = torch.full((2, 3), -INF, device=DEV)
    first[:, 0] = 0  # requests that begin
    got = _select(_logits(6, 5000, dtype, 9), first, 6)
    assert (got[1] == 0).all()


def test_select_far_values():
    """Logits and scores over the types' whole ranges."""
    x = torch.randn(4, 3000, device=DEV) * 1e30
    _select(x, torch.zeros(2, 2, device=DEV), 8)
    x = (torch.randn(4, 3000, device=DEV) * 20000).half()
    _select(x, torch.tensor([[0.0, -1e4], [3e4, -7.0]], device=DEV), 8)
    x = torch.randn(4, 3000, device=DEV) * 1e-3
    _select(x, torch.tensor([[0.0, -1e-4], [-2e-4, 0.0]], device=DEV), 30)


def test_select_all_ended_and_none():
    x = _logits(4, 300, BF16, 3)
    scores = torch.tensor([[-3.0, -1.0], [-INF, -2.0]], device=DEV)
    got = _select(x, scores, 3, torch.ones(2, 2, dtype=torch.bool, device=DEV), 299)
    assert got[1].tolist() == [[1, 0, -1], [1, -1, -1]] and got[2].tolist() == [[299, 299, -1], [299, -1, -1]]
    assert _ops().beam_select(x[:0], scores[:0], 3)[0].shape == (0, 3)


def test_select_captured():
    """Two graphs replayed in turn with new logits, and calls on another stream."""
    x, scores = _logits(8, 32000, F16, 2), (-torch.rand(2, 4)).to(DEV)
    call = lambda: _ops().beam_select(x, scores, 8)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for _ in range(5):
        x.normal_(0, 3)
        want = call()
        for g in graphs:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.synchronize()
        for o in (*outs, other):
            assert all(torch.equal(a, b) for a, b in zip(o, want))


# ---------------------------------------------------------------- pages
def _pools(layers, pages, kvh, page, dim, dtype, layout="dense", seed=1):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, pages, kvh, page, dim)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    if layout == "positions":
        k, v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (k, v))
    elif layout == "both":
        both = torch.stack((k, v), 2).contiguous()
        k, v = both[:, :, 0], both[:, :, 1]
    elif layout == "pages":  # all layers of a page together
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    return k, v


POOLS = [(1, 1, 8, 64, "dense"), (3, 2, 16, 128, "positions"), (2, 5, 32, 80, "both"), (4, 1, 64, 256, "pages"), (2, 3, 8, 1000, "dense")]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layers,kvh,page,dim,layout", POOLS)
def test_copy_pages(dtype, layers, kvh, page, dim, layout):
    _say("copy pages", dtype, layers, kvh, page, dim, layout)
    k, v = _pools(layers, 12, kvh, page, dim, dtype, layout)
    # one source for two, a bad number on either side, a page onto itself, nothing and more than a page of positions
    src, dst = [3, 3, -1, 5, 4, 12, 8, 9], [0, 1, 2, 1 << 30, 4, 6, 7, 10]
    for filled in (None, [page, 1, 5, 5, 5, 5, 0, page + 9], [0, page - 1, 0, 0, 0, 0, -4, 3]):
        want = [mref.copied(t, src, dst, filled) for t in (k, v)]
        _ops().paged_copy_pages(k, v, _ints(src), _ints(dst), None if filled is None else _ints(filled))
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    one = k[0].clone(), v[0].clone()  # one layer
    _ops().paged_copy_pages(*one, _ints([11]), _ints([2]))
    assert torch.equal(one[0][2], k[0, 11]) and torch.equal(one[1][2], v[0, 11])
    _ops().paged_copy_pages(k, v, _ints([]), _ints([]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layers,kvh,page,dim,layout", POOLS)
def test_keep_positions(dtype, layers, kvh, page, dim, layout):
    _say("keep positions", dtype, layers, kvh, page, dim, layout)
    k, v = _pools(layers, 14, kvh, page, dim, dtype, layout)
    table = _ints([[5, 2, 13, 0], [1, 7, -1, 3], [4, 14, 6, 8], [9, 10, 11, 12], [0, 0, 0, 0]])
    many = list(range(0, 3 * page, 2))
    keep = [[0, 1, 3, 4, 9], [1], [0, 2, 3, page + 1, 2 * page], many, []]
    first = [page - 3, 2 * page - 2, page - 1, 1, 0]  # over missing pages, and the last entries past the table
    keep[1] += [4, 2 * page + 1, 10 * page, 1 << 30]
    starts = [0]
    for e in keep:
        starts.append(starts[-1] + len(e))
    flat = [i for e in keep for i in e]
    want = [mref.kept(t, table.cpu(), first, flat, starts) for t in (k, v)]
    _ops().paged_keep_positions(k, v, table, _ints(first), _ints(flat), _ints(starts))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    one = k[0].clone(), v[0].clone()
    want = [mref.kept(t[None], table.cpu()[:1], [2], [3, 5], [0, 2])[0] for t in one]
    _ops().paged_keep_positions(*one, table[:1], _ints([2]), _ints([3, 5]), _ints([0, 2]))
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])


def test_moves_of_far_pages():
    """Pools of more than 2^31 values."""
    pages = (1 << 31) // (2 * 64 * 128) // 2 + 10
    k = torch.empty(2, pages, 2, 64, 128, device=DEV, dtype=BF16)
    v = torch.empty_like(k)
    for t in (k, v):
        t[:, [pages - 1, pages - 2, 3]] = torch.randn(2, 3, 2, 64, 128, device=DEV).to(BF16)
    want = k[:, pages - 1].clone(), v[:, pages - 1].clone()
    _ops().paged_copy_pages(k, v, _ints([pages - 1]), _ints([7]))
    assert torch.equal(k[:, 7], want[0]) and torch.equal(v[:, 7], want[1])
    row = k[1, pages - 2, :, 5].clone()
    _ops().paged_keep_positions(k, v, _ints([[3, pages - 2]]), _ints([60]), _ints([1, 9]), _ints([0, 2]))
    assert torch.equal(k[1, 3, :, 61], row)


def test_moves_captured_and_registered():
    k, v = _pools(2, 9, 2, 16, 64, F16)
    src, dst, filled = _ints([1, -1]), _ints([2, -1]), _ints([16, 0])
    table, first, keep, starts = _ints([[2, 3]]), _ints([0]), _ints([4, 17]), _ints([0, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _ops().paged_copy_pages(k, v, src, dst, filled)
        _ops().paged_keep_positions(k, v, table, first, keep, starts)
    for i in range(4):
        k.normal_()
        src[1], dst[1], filled[1] = 5 + i % 2, 7, 3 + i
        want = [mref.kept(mref.copied(t, src.tolist(), dst.tolist(), filled.tolist()), table.cpu(), [0], [4, 17], [0, 2]) for t in (k, v)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    version = k._version
    _ops().paged_copy_pages(k, v, src, dst)
    assert k._version > version
    tests = ("test_schema", "test_faketensor")
    ns = torch.ops.mindpipe_amd_serve
    torch.library.opcheck(ns.paged_copy_pages.default, (k, v, src, dst, filled), test_utils=tests)
    torch.library.opcheck(ns.paged_keep_positions.default, (k, v, table, first, keep, starts), test_utils=tests)
    x = _logits(4, 100, F16, 1)
    torch.library.opcheck(ns.beam_select.default, (x, torch.zeros(2, 2, device=DEV), 3), test_utils=tests)


def test_append_at_given_turns():
    """Rows that turn by other positions than their own: places as ever, angles by ``turns``, which may have none."""
    k, v = (t[0] for t in _pools(1, 6, 2, 8, 64, BF16))
    table, lens, starts = _ints([[0, 3, 2], [4, 1, 5]]), _ints([12, 9]), _ints([0, 5, 8])
    cos, sin = torch.rand(30, 32, device=DEV), torch.rand(30, 32, device=DEV)
    qkv = torch.randn(9, 8 * 64, device=DEV).to(BF16)
    turns = [7, 8, 8, 9, 9, 6, 30, -1, 3]
    for pairs in (True, False):
        kk, vv = k.clone(), v.clone()
        q = _ops().paged_rope_append(qkv, cos, sin, kk, vv, table, lens, starts, pairs, _ints(turns))
        want, wk, wv = torch.zeros(9, 4, 64, dtype=torch.float64), k.cpu().double(), v.cpu().double()
        x = qkv.cpu().double().view(9, 8, 64)
        for t, (b, pos) in enumerate([(0, 7), (0, 8), (0, 9), (0, 10), (0, 11), (1, 6), (1, 7), (1, 8)]):
            if 0 <= turns[t] < 30:
                y = ref.rotate(x[t:t + 1, :6], cos[turns[t]][None].cpu(), sin[turns[t]][None].cpu(), pairs)[0]
                want[t] = y[:4]
                wk[int(table[b, pos // 8]), :, pos % 8], wv[int(table[b, pos // 8]), :, pos % 8] = y[4:], x[t, 6:]
        # rotated in fp32 (three roundings of 2^-24 of the magnitudes, below 6) and rounded once
        for got, w in ((q, want), (kk, wk)):
            ref.check(got, w, 2.0 ** -8 * w.abs() + 2.0 ** -20)
        assert torch.equal(vv.cpu().double(), wv)
        same = _ops().paged_rope_append(qkv[:5], cos, sin, k.clone(), v.clone(), table[:1], lens[:1], starts[:2], pairs,
                                        _ints([7, 8, 9, 10, 11]))
        assert torch.equal(same, _ops().paged_rope_append(qkv[:5], cos, sin, k.clone(), v.clone(), table[:1], lens[:1], starts[:2], pairs))
    assert math.isfinite(float(q.float().abs().max()))
