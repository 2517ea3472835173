"""Attention of drafted trees and of windows over a paged cache against plain 64-bit forms on the CPU (``masked_reference``)."""
import random
import sys

import pytest
import torch

import masked_reference as mref
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


def _starts(news):
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    return at


def _cache(lens, kvh, dim, page, dtype, seed, layout="dense", fill=float("nan"), spare=2, extra=0):
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


def _queries(rows, heads, dim, dtype, seed=9):
    return (1.5 * torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def _trees(news, seed):
    rng = random.Random(seed)
    return [mref.ancestors([rng.randrange(-1, i) for i in range(n)]) for n in news]


HEADS = [(64, 2, 1), (64, 1, 7), (128, 2, 4), (128, 3, 1), (256, 1, 5), (128, 1, 21), (256, 2, 2)]


# ---------------------------------------------------------------- trees
def _tree(k, v, table, ln, news, heads, dtype, sets, words, scale=None, front=0, behind=2, q=None):
    at = [front + a for a in _starts(news)]
    dim = k.shape[3]
    scale = dim ** -0.5 if scale is None else scale
    rows = at[-1] + behind
    q = _queries(rows, heads, dim, dtype) if q is None else q
    m = torch.full((rows, words), -1, dtype=torch.int64)  # rows of no sequence may say anything
    m[front:at[-1]] = mref.masks(sets, words)
    m = m.to(DEV)
    got = _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), m, scale)
    want, tol = mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_tree(
        [[[i for i in s if i < 64 * words] for s in seq] for seq in sets]), scale)
    ref.check(got, want, tol)
    assert torch.equal(got, _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), m, scale)) or got.isnan().any()
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", HEADS)
@pytest.mark.parametrize("news,ctxs,page", [([1], [0], 8), ([5, 0, 1, 26], [100, 9, 0, 31], 16), ([64, 3], [63, 700], 64),
                                            ([65, 17], [64, 1], 32), ([130], [50], 8)])
def test_tree(dtype, dim, kvh, grp, news, ctxs, page):
    _say("tree", dtype, dim, kvh, grp, news, ctxs, page)
    lens = [n + c for n, c in zip(news, ctxs)]
    k, v, table, ln = _cache(lens, kvh, dim, page, dtype, 8, "positions" if page == 16 else "dense", extra=1)
    _tree(k, v, table, ln, news, kvh * grp, dtype, _trees(news, 3), -(-max(news) // 64), front=1)


@pytest.mark.parametrize("words", [1, 2, 5])
def test_tree_any_sets(words):
    """Sets that are no trees, empty ones, later nodes, and bits past the sequence's nodes and past the words."""
    news, ctxs = [70, 9, 4], [33, 0, 0]
    k, v, table, ln = _cache([n + c for n, c in zip(news, ctxs)], 2, 64, 8, BF16, 5)
    rng = random.Random(1)
    sets = [[[i for i in range(64 * words) if rng.random() < 0.3] for _ in range(n)] for n in news]
    sets[1][3], sets[1][4], sets[2][0] = [], [300], []
    got = _tree(k, v, table, ln, news, 4, BF16, sets, words)
    assert not got[70 + 3].any() and not got[79].any()  # nothing seen


def test_tree_without_context_or_place():
    """Sequences shorter than their new tokens, lengths below zero and past the table, pages that are not there."""
    for page in (8, 32):
        news, lens = [6, 6, 4, 30], [4, -3, 40, 100]
        k, v, table, ln = _cache([40, 40, 40, 100], 1, 128, page, F16, 6, fill=None)
        ln = _ints(lens)
        table = table[:, :-(-64 // page)].contiguous()  # the last sequence is longer than its table
        table[2, 0], table[3, 1] = -1, 1 << 20
        got = _tree(k, v, table, ln, news, 3, F16, _trees(news, 4), 1)
        assert not got[6:12].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_tree_siblings_do_not_reach_each_other(dtype, dim, bad):
    """NaN and infinities in a node's key or value reach its descendants and no others."""
    news, ctxs = [20, 11], [70, 300]
    sets = _trees(news, 7)
    for where in (0, 1):
        k, v, table, ln = _cache([90, 311], 2, dim, 16, dtype, 11)
        p = 70 + 6
        (k, v)[where][int(table[0, p // 16]), 0, p % 16] = bad
        q = _queries(33, 4, dim, dtype)
        m = torch.zeros(33, 1, dtype=torch.int64)
        m[:31] = mref.masks(sets, 1)
        got = _ops().paged_tree_attention(q, k, v, table, ln, _ints([0, 20, 31]), m.to(DEV), 0.1)
        want, tol = mref.masked_attention(q, k, v, table, ln, torch.tensor([0, 20, 31]), mref.in_tree(sets), 0.1)
        for j in range(20):
            if 6 not in sets[0][j]:
                assert torch.isfinite(got[j]).all()
            elif bad != bad:
                assert torch.isnan(got[j, :2]).any()
        sees = torch.tensor([6 in sets[0][j] for j in range(20)] + [False] * 13)
        ref.check(got[~sees.to(DEV)], want[~sees], tol[~sees])
        if where and bad == bad:  # an infinity in V: the others' values are as without it
            ref.check(got[:, 2:], want[:, 2:], tol[:, 2:])


def test_tree_scales():
    news = [9]
    k, v, table, ln = _cache([309], 1, 128, 16, F16, 4)
    for p in range(300):
        k[int(table[0, p // 16]), 0, p % 16] *= p / 40.0
    for scale in (0.3, -0.3, 0.0):
        _tree(k, v, table, ln, news, 4, F16, _trees(news, 2), 1, scale)


def test_tree_many_sequences():
    """More sequences than a wave has lanes, most of them without new tokens."""
    g = random.Random(5)
    news = [g.choice((0, 0, 1, 3)) for _ in range(150)]
    ctxs = [g.randrange(0, 40) for _ in news]
    ctxs[3], news[3], ctxs[140], news[140] = 900, 12, 2000, 2
    k, v, table, ln = _cache([a + b for a, b in zip(news, ctxs)], 1, 64, 16, BF16, 6)
    _tree(k, v, table, ln, news, 2, BF16, _trees(news, 6), 1)


@pytest.mark.parametrize("count", [61, 62, 63, 64, 130, 1021, 1022, 1023, 2100])
def test_any_number_of_sequences(count):
    """Sequences of many lengths, one of them so long that it is cut, in trees of few rows and of many, and with windows."""
    g = random.Random(count)
    news = [g.choice((0, 0, 1, 2)) for _ in range(count)]
    ctxs = [g.randrange(0, 20) for _ in news]
    at = (count - 1, count // 2, 0)
    for b, n, c in zip(at, (40, 3, 0), (5000, 0, 900)):
        news[b], ctxs[b] = n, c
    k, v, table, ln = _cache([a + b for a, b in zip(news, ctxs)], 1, 64, 16, F16, 7)
    _tree(k, v, table, ln, news, 2, F16, _trees(news, 8), 1)
    _tree(k, v, table, ln, news, 70, F16, _trees(news, 8), 1)  # more rows to a sequence
    q = _queries(sum(news) + 1, 2, 64, F16)
    starts = _ints(_starts(news))
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, starts, 0.125, 30, 4)
    want, tol = mref.masked_attention(q, k, v, table, ln, starts, mref.in_window(30, 4), 0.125)
    ref.check(got, want, tol)


def test_tree_runs_that_cut_items():
    """Long and short sequences with several row tiles each: runs begin and end inside of items."""
    news, ctxs = [40, 64, 2, 33], [4000, 100, 1500, 0]
    k, v, table, ln = _cache([a + b for a, b in zip(news, ctxs)], 1, 128, 64, BF16, 7)
    _tree(k, v, table, ln, news, 8, BF16, _trees(news, 8), 1)


def test_tree_long_and_alone():
    """One sequence whose tiles make many more parts than there are items: one less than 17 equal shares of them, with the one that
    the rows behind it have."""
    shares = torch.cuda.get_device_properties(0).multi_processor_count  # two workgroups to a CU, two key-value heads
    n = 64 * (17 * shares - 2)
    k, v, table, ln = _cache([n], 2, 64, 64, BF16, 12)
    v[table[0, -100:].long()] += 40  # of a part that is not there much is missing
    _tree(k, v, table, ln, [3], 16, BF16, _trees([3], 6), 1)


def test_far_pages_and_strided_queries():
    """Pools of more than 2^31 values: offsets pass 32 bits.  Only the pages used are written."""
    pages = (1 << 31) // (8 * 128 * 128) + 40
    k = torch.empty(pages, 8, 128, 128, device=DEV, dtype=BF16)
    v = torch.empty_like(k)
    table = _ints([[pages - 1, 3, pages - 20, pages // 2 + 7]])
    for p in table[0].tolist():
        k[p], v[p] = torch.randn(8, 128, 128, device=DEV), torch.randn(8, 128, 128, device=DEV)
    few, near, news = table[0].long(), _ints([[0, 1, 2, 3]]), 6
    qkv = torch.randn(news, 32, 128, device=DEV).to(BF16)
    q, at, ln = qkv[:, 4:20], torch.tensor([0, news]), _ints([450])
    sets = _trees([news], 9)
    got = _ops().paged_tree_attention(q, k, v, table, ln, _ints([0, news]), mref.masks(sets, 1).to(DEV), 0.09)
    ref.check(got, *mref.masked_attention(q, k[few], v[few], near, ln, at, mref.in_tree(sets), 0.09))
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints([0, news]), 0.09, 100, 3)
    ref.check(got, *mref.masked_attention(q, k[few], v[few], near, ln, at, mref.in_window(100, 3), 0.09))
    got = _ops().paged_decode_window_attention(q[:1], k, v, table, ln, 0.09, 100, 3)
    ref.check(got, *mref.masked_attention(q[:1], k[few], v[few], near, ln, None, mref.in_window(100, 3), 0.09))


# ---------------------------------------------------------------- windows
WINDOWS = [(1, 0), (7, 1), (64, 4), (100, 64), (100, 100), (1 << 30, 0), (33, 1 << 30)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_decode_window(dtype, dim, kvh, grp, window, sinks):
    _say("decode window", dtype, dim, kvh, grp, window, sinks)
    lens = [1, 0, 8, 33, 97, 128, 129, 700]
    k, v, table, ln = _cache(lens, kvh, dim, 16, dtype, 1, ("dense", "positions", "both")[grp % 3], extra=1)
    q = _queries(len(lens), kvh * grp, dim, dtype)
    got = _ops().paged_decode_window_attention(q, k, v, table, ln, dim ** -0.5, window, sinks)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, None, mref.in_window(window, sinks), dim ** -0.5))
    assert torch.equal(got, _ops().paged_decode_window_attention(q, k, v, table, ln, dim ** -0.5, window, sinks))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("news,ctxs", [([3, 1, 0, 40], [100, 0, 9, 31]), ([130], [260]), ([17, 64, 2], [0, 15, 900])])
def test_prompt_window(dtype, dim, kvh, grp, window, sinks, news, ctxs):
    _say("prompt window", dtype, dim, kvh, grp, window, sinks, news, ctxs)
    lens = [n + c for n, c in zip(news, ctxs)]
    page = 8 if grp == 1 else 32
    k, v, table, ln = _cache(lens, kvh, dim, page, dtype, 8, ("dense", "positions", "both")[grp % 3], extra=1)
    at = [1 + a for a in _starts(news)]
    q = _queries(at[-1] + 2, kvh * grp, dim, dtype)
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(window, sinks), dim ** -0.5))
    assert torch.equal(got, _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_window_past_the_table(dtype):
    """Lengths past the table's room keep their windows where they are: a row whose window lies past it sees the sinks alone."""
    k, v, table, ln = _cache([64, 64, 64, 64], 2, 128, 16, dtype, 3)
    ln = _ints([70, 90, 100000, -7])
    q = _queries(4, 8, 128, dtype)
    for window, sinks in ((20, 0), (20, 3), (7, 70), (30, 0)):
        sees = mref.in_window(window, sinks)
        got = _ops().paged_decode_window_attention(q, k, v, table, ln, 0.1, window, sinks)
        ref.check(got, *mref.masked_attention(q, k, v, table, ln, None, sees, 0.1))
        at = [0, 5, 30, 40, 45]
        p = _queries(45, 8, 128, dtype)
        got = _ops().paged_prompt_window_attention(p, k, v, table, ln, _ints(at), 0.1, window, sinks)
        ref.check(got, *mref.masked_attention(p, k, v, table, ln, torch.tensor(at), sees, 0.1))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_behind_the_window_may_be_gone(dim):
    """What lies between the sinks and the windows is not looked at: its pages may be missing, or hold NaN and infinities."""
    dtype, page, window, sinks = BF16, 8, 50, 5
    lens, news = [400, 200], [9, 70]
    k, v, table, ln = _cache(lens, 2, dim, page, dtype, 12)
    q, at = _queries(79, 6, dim, dtype), [0, 9, 79]
    d = _queries(2, 6, dim, dtype, 10)

    def both():
        return (_ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), 0.1, window, sinks),
                _ops().paged_decode_window_attention(d, k, v, table, ln, 0.1, window, sinks))

    want = both()
    for b, (length, n) in enumerate(zip(lens, news)):
        low = length - n - window + 1
        for p in range(sinks, low):  # unseen by all rows
            k[int(table[b, p // page]), :, p % page] = float("nan")
            v[int(table[b, p // page]), :, p % page] = float("inf") if p % 2 else float("nan")
    seen = mref.in_window(window, sinks)
    for gone in (False, True):
        if gone:
            for b, (length, n) in enumerate(zip(lens, news)):
                for e in range(1, (length - n - window + 1) // page):
                    table[b, e] = -1 if e % 2 else 1 << 30
        got = both()
        # a tile that holds such values is added position by position: another order of the same fp32 sums
        ref.check(got[0], *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), seen, 0.1))
        ref.check(got[1], *mref.masked_attention(d, k, v, table, ln, None, seen, 0.1))
        for g, w in zip(got, want):
            assert (g.float() - w.float()).abs().max() <= 4 * ref.HALF_STEP[dtype] * w.float().abs().max()


def test_later_tokens_do_not_reach_back():
    """NaN in a token's key and value reach the rows whose windows hold it and no others."""
    k, v, table, ln = _cache([120], 1, 128, 16, F16, 13)
    q = _queries(80, 2, 128, F16)
    for t in (k, v):
        t[int(table[0, 60 // 16]), 0, 60 % 16] = float("nan")
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints([0, 80]), 0.1, 30, 2)
    bad = torch.isnan(got).any(-1).any(-1).tolist()  # row j is position 40 + j
    assert bad == [60 <= 40 + j < 90 for j in range(80)]


# ---------------------------------------------------------------- how they are called
def _calls(dtype=F16, dim=128):
    news, lens = [5, 30, 1], [200, 90, 1500]
    k, v, table, ln = _cache(lens, 2, dim, 16, dtype, 21)
    q, d, starts = _queries(36, 8, dim, dtype), _queries(3, 8, dim, dtype, 22), _ints([0, 5, 35, 36])
    m = mref.masks(_trees(news, 1), 1).to(DEV)
    return (lambda: _ops().paged_tree_attention(q, k, v, table, ln, starts, m, 0.1),
            lambda: _ops().paged_prompt_window_attention(q, k, v, table, ln, starts, 0.1, 100, 4),
            lambda: _ops().paged_decode_window_attention(d, k, v, table, ln, 0.1, 100, 4)), (q, d, m)


def test_captured_and_replayed():
    """Two graphs of the same calls, replayed in turn with new inputs and eager calls between, give the eager bits."""
    calls, (q, d, m) = _calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([c() for c in calls])
    for i in range(6):
        q.normal_()
        d.normal_()
        want = [c() for c in calls]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want)), i


def test_on_another_stream():
    calls, (q, d, m) = _calls(BF16)
    want = [c() for c in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [c() for c in calls]
    here = [c() for c in calls]  # beside those
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(here, want))


def test_offsets_that_do_not_ascend_stay_inside():
    """What such a call returns is open; it reads and writes nothing outside of its tensors."""
    k, v, table, ln = _cache([64, 64, 64], 1, 64, 16, F16, 3)
    q, m = _queries(40, 2, 64, F16), torch.ones(40, 1, dtype=torch.int64, device=DEV)
    for at in ([0, 30, 10, 40], [40, 0, 0, 40], [-5, 100, 3, 1 << 30], [50, 50, 50, 50]):
        assert _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), m, 0.1).shape == q.shape
        assert _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), 0.1, 9, 1).shape == q.shape
    torch.cuda.synchronize()


def test_nothing_to_do():
    k, v, table, ln = _cache([64], 1, 64, 16, F16, 3)
    q, none = _queries(3, 2, 64, F16), torch.zeros(0, 1, dtype=torch.int64, device=DEV)
    m = torch.ones(3, 1, dtype=torch.int64, device=DEV)
    assert _ops().paged_tree_attention(q[:0], k, v, table, ln, _ints([0, 0]), none, 0.1).shape == (0, 2, 64)
    assert not _ops().paged_tree_attention(q, k, v, table[:0], ln[:0], _ints([0]), m, 0.1).any()
    assert not _ops().paged_tree_attention(q, k, v, table, ln, _ints([0, 0]), m, 0.1).any()
    assert not _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints([3, 3]), 0.1, 5, 0).any()
    assert _ops().paged_decode_window_attention(q[:0], k, v, table[:0], ln[:0], 0.1, 5, 0).shape == (0, 2, 64)


def test_registered():
    tests = ("test_schema", "test_faketensor")
    k, v, table, ln = _cache([60], 1, 64, 16, F16, 3)
    q, m = _queries(3, 2, 64, F16), torch.ones(3, 1, dtype=torch.int64, device=DEV)
    ns = torch.ops.mindpipe_amd_serve
    torch.library.opcheck(ns.paged_tree_attention.default, (q, k, v, table, ln, _ints([0, 3]), m, 0.1), test_utils=tests)
    torch.library.opcheck(ns.paged_prompt_window_attention.default, (q, k, v, table, ln, _ints([0, 3]), 0.1, 9, 1), test_utils=tests)
    torch.library.opcheck(ns.paged_decode_window_attention.default, (q[:1], k, v, table, ln, 0.1, 9, 1), test_utils=tests)
