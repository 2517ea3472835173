"""The wide form of the masked attention kernels (128 rows to a workgroup) against plain 64-bit forms on the CPU: trees and windows of
every head size and type, values that only some rows see, items that are cut, missing pages.  A table that is much wider than its
sequences sends small calls to that form; each test makes sure that it did."""
import ctypes
import random

import pytest
import torch

import masked_reference as mref
import paged_reference as ref
from test_gpu_masked import DEV, _cache, _ints, _ops, _queries, _say, _starts, _tree, _trees
from test_gpu_masked_forms import NARROW, WIDE, _form

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SIZES = [(64, 2, 1), (64, 1, 7), (64, 2, 16), (128, 2, 4), (128, 3, 1), (128, 1, 21), (256, 1, 5), (256, 2, 2), (256, 1, 16)]


def _room(kvh, page):
    """Columns that make any call a wide one: work is counted by what the table has room for."""
    return -(-(1 << 21) // (kvh * page))


def _is_wide(q, k, table, batch, window=0, sinks=0):
    assert _form(q.shape[0], q.shape[1], k.shape[1], k.shape[3], batch, table.shape[1] * k.shape[2], window, sinks) == WIDE


def _same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


# ---------------------------------------------------------------- trees
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", SIZES)
@pytest.mark.parametrize("news,ctxs,page", [([1], [0], 8), ([5, 0, 1, 26], [100, 9, 0, 31], 16), ([64, 3], [63, 700], 64), ([65, 17], [64, 1], 32)])
def test_wide_tree(dtype, dim, kvh, grp, news, ctxs, page):
    _say("wide tree", dtype, dim, kvh, grp, news, ctxs, page)
    lens = [n + c for n, c in zip(news, ctxs)]
    k, v, table, ln = _cache(lens, kvh, dim, page, dtype, 8, ("dense", "positions", "both")[grp % 3], extra=_room(kvh, page))
    q = _queries(sum(news) + 3, kvh * grp, dim, dtype)
    _is_wide(q, k, table, len(lens))
    got = _tree(k, v, table, ln, news, kvh * grp, dtype, _trees(news, 3), -(-max(news) // 64), front=1, q=q)
    assert not got[0].any() and not got[-2:].any()  # rows of no sequence


@pytest.mark.parametrize("words", [1, 2, 5])
def test_wide_tree_any_sets(words):
    """Sets that are no trees, empty ones, later nodes, and bits past the sequence's nodes and past the words."""
    news, ctxs = [70, 9, 4], [33, 0, 0]
    k, v, table, ln = _cache([n + c for n, c in zip(news, ctxs)], 2, 128, 8, BF16, 5, extra=_room(2, 8))
    rng = random.Random(1)
    sets = [[[i for i in range(64 * words) if rng.random() < 0.3] for _ in range(n)] for n in news]
    sets[1][3], sets[1][4], sets[2][0] = [], [300], []
    q = _queries(85, 4, 128, BF16)
    _is_wide(q, k, table, 3)
    got = _tree(k, v, table, ln, news, 4, BF16, sets, words, q=q)
    assert not got[70 + 3].any() and not got[79].any()  # nothing seen


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_wide_lengths_and_pages_that_are_not_there(dim):
    """Sequences shorter than their new tokens, lengths below zero and past the table, pages outside the pool."""
    news, lens = [6, 6, 4, 30], [4, -3, 40, 100]
    k, v, table, ln = _cache([40, 40, 40, 100], 1, dim, 8, F16, 6, fill=None, extra=_room(1, 8))
    ln = _ints(lens)
    table[2, 0], table[3, 1], table[3, 7] = -1, 1 << 20, k.shape[0]
    q = _queries(48, 3, dim, F16)
    _is_wide(q, k, table, 4)
    got = _tree(k, v, table, ln, news, 3, F16, _trees(news, 4), 1, q=q)
    assert not got[6:12].any()
    at = torch.tensor(_starts(news))
    for window, sinks in ((1 << 30, 0), (50, 1 << 30)):
        _is_wide(q, k, table, 4, window, sinks)
        got = _ops().paged_prompt_window_attention(q, k, v, table, ln, at.int().to(DEV), 0.1, window, sinks)
        ref.check(got, *mref.masked_attention(q, k, v, table, ln, at, mref.in_window(window, sinks), 0.1))


def test_wide_past_the_table():
    """A sequence longer than its table, with enough rows for the wide form."""
    k, v, table, ln = _cache([128, 64], 16, 128, 16, BF16, 3)
    ln = _ints([150, 60])
    news = [120, 40]
    q, at = _queries(160, 128, 128, BF16), torch.tensor(_starts(news))
    for window, sinks in ((1 << 30, 0), (20, 3), (40, 0)):
        _is_wide(q, k, table, 2, window, sinks)
        got = _ops().paged_prompt_window_attention(q, k, v, table, ln, at.int().to(DEV), 0.05, window, sinks)
        ref.check(got, *mref.masked_attention(q, k, v, table, ln, at, mref.in_window(window, sinks), 0.05))


@pytest.mark.parametrize("dtype,dim,whole", [*((t, d, False) for t in (F16, BF16) for d in (64, 128, 256)), (BF16, 64, True),
                                             (F16, 128, True), (BF16, 256, True)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_wide_siblings_do_not_reach_each_other(dtype, dim, whole, bad):
    """NaN and infinities in a node's key or value reach its descendants and no others, in items that are cut and in whole ones."""
    # whole: 16 sequences of four tiles for 16 workgroups of a head at most, so that none is longer than what they stay whole with
    kvh, grp, news, ctxs = (32, 1, [3] * 16, [250] * 16) if whole else (2, 2, [20, 11], [70, 300])
    heads = kvh * grp
    sets, at = _trees(news, 7), _starts(news)
    bad_node = 1 if whole else 6
    first = [b for b in range(len(news)) if any(bad_node in s for s in sets[b])][0]
    for where in (0, 1):
        k, v, table, ln = _cache([n + c for n, c in zip(news, ctxs)], kvh, dim, 16, dtype, 11, extra=_room(kvh, 16))
        p = ctxs[first] + bad_node
        (k, v)[where][int(table[first, p // 16]), 0, p % 16] = bad
        q = _queries(at[-1] + 2, heads, dim, dtype)
        _is_wide(q, k, table, len(news))
        m = torch.zeros(at[-1] + 2, 1, dtype=torch.int64)
        m[:at[-1]] = mref.masks(sets, 1)
        got = _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), m.to(DEV), 0.1)
        want, tol = mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_tree(sets), 0.1)
        sees = torch.zeros(at[-1] + 2, dtype=torch.bool)
        for j in range(news[first]):
            sees[at[first] + j] = bad_node in sets[first][j]
        assert torch.isfinite(got[~sees.to(DEV)]).all()
        if bad != bad:
            assert torch.isnan(got[sees.to(DEV)][:, :grp]).any(-1).all()
        ref.check(got[~sees.to(DEV)], want[~sees], tol[~sees])
        if where and bad == bad:  # an infinity in V: an infinity to those who see it, and other heads' values as without it
            ref.check(got, want, tol)
        assert _same_bits(got, _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), m.to(DEV), 0.1))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_wide_scales(dim):
    news = [9]
    k, v, table, ln = _cache([309], 1, dim, 16, F16, 4, extra=_room(1, 16))
    for p in range(300):
        k[int(table[0, p // 16]), 0, p % 16] *= p / 40.0
    q = _queries(11, 4, dim, F16)
    _is_wide(q, k, table, 1)
    for scale in (0.3, -0.3, 0.0):
        _tree(k, v, table, ln, news, 4, F16, _trees(news, 2), 1, scale, q=q)


@pytest.mark.parametrize("dtype,dim", [(F16, 256), (BF16, 128), (F16, 64)])
def test_wide_items_that_are_cut(dtype, dim):
    """Long and short sequences with several row tiles each, remainders among them."""
    news, ctxs = [40, 64, 2, 33], [1500, 100, 900, 0]
    k, v, table, ln = _cache([a + b for a, b in zip(news, ctxs)], 1, dim, 64, dtype, 7, extra=_room(1, 64))
    q = _queries(141, 8, dim, dtype)
    _is_wide(q, k, table, 4)
    _tree(k, v, table, ln, news, 8, dtype, _trees(news, 8), 1, q=q)


# ---------------------------------------------------------------- windows
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 7), (64, 3, 1), (128, 2, 4), (128, 1, 21), (256, 1, 5), (256, 2, 2)])
@pytest.mark.parametrize("window,sinks", [(1 << 30, 0), (33, 1 << 30)])
@pytest.mark.parametrize("news,ctxs", [([3, 1, 0, 40], [100, 0, 9, 31]), ([130], [260])])
def test_wide_window_of_all(dtype, dim, kvh, grp, window, sinks, news, ctxs):
    _say("wide window", dtype, dim, kvh, grp, window, sinks, news, ctxs)
    lens = [n + c for n, c in zip(news, ctxs)]
    page = 8 if grp == 1 else 32
    k, v, table, ln = _cache(lens, kvh, dim, page, dtype, 8, ("dense", "positions", "both")[grp % 3], extra=_room(kvh, page))
    at = [1 + a for a in _starts(news)]
    q = _queries(at[-1] + 2, kvh * grp, dim, dtype)
    _is_wide(q, k, table, len(news), window, sinks)
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(window, sinks), dim ** -0.5))
    assert _same_bits(got, _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks))


# rows enough for the wide form at any window: heads of the three sizes, groups that do and do not divide 128 rows
MANY = [(64, 16, 6), (128, 16, 8), (256, 8, 12)]


def _many(dim, kvh, grp, dtype, page, lens=(420, 150), news=(140, 33), fill=float("nan")):
    k, v, table, ln = _cache(list(lens), kvh, dim, page, dtype, 12, ("dense", "positions", "both")[page % 3], fill=fill, extra=1)
    at = _starts(list(news))
    return k, v, table, ln, at, _queries(at[-1], kvh * grp, dim, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", MANY)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (100, 64), (64, 4)])
def test_wide_window(dtype, dim, kvh, grp, window, sinks):
    _say("wide window", dtype, dim, kvh, grp, window, sinks)
    k, v, table, ln, at, q = _many(dim, kvh, grp, dtype, 8 if window == 7 else 16)
    _is_wide(q, k, table, 2, window, sinks)
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(window, sinks), dim ** -0.5))
    assert _same_bits(got, _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), dim ** -0.5, window, sinks))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", MANY)
def test_wide_pages_behind_the_window_may_be_gone(dtype, dim, kvh, grp):
    """What lies between the sinks and the windows is not looked at: it may hold NaN and infinities, and its pages may be missing."""
    lens, news, page, window, sinks = (400, 200), (90, 70), 8, 50, 5
    k, v, table, ln, at, q = _many(dim, kvh, grp, dtype, page, lens, news)
    _is_wide(q, k, table, 2, window, sinks)
    want, tol = mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(window, sinks), 0.1)
    for b, (length, n) in enumerate(zip(lens, news)):
        for p in range(sinks, length - n - window + 1):  # unseen by all rows
            k[int(table[b, p // page]), :, p % page] = float("nan")
            v[int(table[b, p // page]), :, p % page] = float("inf") if p % 2 else float("nan")
    for gone in (False, True):
        if gone:
            for b, (length, n) in enumerate(zip(lens, news)):
                for e in range(1, (length - n - window + 1) // page):
                    table[b, e] = -1 if e % 2 else 1 << 30
        ref.check(_ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), 0.1, window, sinks), want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", MANY)
def test_wide_values_inside_the_windows(dtype, dim, kvh, grp):
    """NaN in a key, an infinity in a value: they reach the rows whose windows hold them and no others."""
    k, v, table, ln, at, q = _many(dim, kvh, grp, dtype, 16, (260,), (140,))
    _is_wide(q, k, table, 1, 30, 2)
    k[int(table[0, 150 // 16]), 0, 150 % 16] = float("nan")
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), 0.1, 30, 2)
    assert torch.isnan(got[:, :grp]).any(-1).any(-1).tolist() == [150 <= 120 + j < 180 for j in range(140)]
    assert torch.isfinite(got[:, grp:]).all()
    k[int(table[0, 150 // 16]), 0, 150 % 16] = 0
    v[int(table[0, 200 // 16]), :, 200 % 16, 5] = -float("inf")
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), 0.1, 30, 2)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(30, 2), 0.1))


# ---------------------------------------------------------------- how they are called
def test_wide_far_pages_and_strided_queries():
    """Pools of more than 2^31 values: offsets pass 32 bits.  Only the pages used are written."""
    pages = (1 << 31) // (8 * 128 * 128) + 40
    k = torch.empty(pages, 8, 128, 128, device=DEV, dtype=BF16)
    v = torch.empty_like(k)
    table = torch.zeros(1, _room(8, 128), device=DEV, dtype=torch.int32)
    table[0, :4] = _ints([pages - 1, 3, pages - 20, pages // 2 + 7])
    few = table[0, :4].long()
    for p in few.tolist():
        k[p], v[p] = torch.randn(8, 128, 128, device=DEV), torch.randn(8, 128, 128, device=DEV)
    near, news = _ints([[0, 1, 2, 3]]), 6
    qkv = torch.randn(news, 32, 128, device=DEV).to(BF16)
    q, at, ln = qkv[:, 4:20], torch.tensor([0, news]), _ints([450])
    _is_wide(q, k, table, 1)
    sets = _trees([news], 9)
    got = _ops().paged_tree_attention(q, k, v, table, ln, _ints([0, news]), mref.masks(sets, 1).to(DEV), 0.09)
    ref.check(got, *mref.masked_attention(q, k[few], v[few], near, ln, at, mref.in_tree(sets), 0.09))
    _is_wide(q, k, table, 1, 1 << 30)
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints([0, news]), 0.09, 1 << 30, 3)
    ref.check(got, *mref.masked_attention(q, k[few], v[few], near, ln, at, mref.in_window(1 << 30, 3), 0.09))


def test_wide_captured_and_replayed():
    """Two graphs of the same calls, replayed in turn with new inputs, eager calls between and another stream beside, give the eager
    bits."""
    k, v, table, ln, at, q = _many(128, 16, 8, F16, 16)
    wide = torch.cat((table, torch.zeros(2, _room(16, 16), device=DEV, dtype=torch.int32)), 1).contiguous()
    _is_wide(q, k, wide, 2)
    _is_wide(q, k, table, 2, 100, 4)
    m, starts = mref.masks(_trees([140, 33], 1), 3).to(DEV), _ints(at)
    calls = (lambda: _ops().paged_tree_attention(q, k, v, wide, ln, starts, m, 0.1),
             lambda: _ops().paged_prompt_window_attention(q, k, v, table, ln, starts, 0.1, 100, 4))
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
    for i in range(5):
        q.normal_()
        want = [c() for c in calls]
        for g in graphs:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [c() for c in calls]
        torch.cuda.synchronize()
        for o in (*outs, other):
            assert all(_same_bits(a, b) for a, b in zip(o, want)), i


def _guarded(values, dtype, fill):
    """A tensor of so many values between two runs of a known pattern, at 16 bytes, and a check that the pattern is as it was."""
    edge = 8192
    whole = torch.full((values + 2 * edge,), fill, dtype=dtype, device=DEV)
    inside = whole[edge:edge + values]
    assert inside.data_ptr() % 16 == 0
    return inside, lambda: bool((whole[:edge] == fill).all() and (whole[edge + values:] == fill).all())


@pytest.mark.parametrize("form", [NARROW, WIDE])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [3, 70])  # planned by every workgroup, and once
def test_nothing_is_written_outside(form, dim, batch):
    """Any offsets, ascending or not, ends among them: outputs, workspace and what lies before and behind them."""
    from mindpipe_amd import _lib
    lib, page, rows, nh, kvh = _lib.load(), 16, 40, 4, 2
    k, v, table, ln = _cache([64, 130, 64] + [1] * (batch - 3), kvh, dim, page, F16, 3, extra=_room(kvh, page) if form == WIDE else 0)
    q, m = _queries(rows, nh, dim, F16), torch.ones(rows, 1, dtype=torch.int64, device=DEV)
    capacity = table.shape[1] * page
    cache = _lib.PAGES.pack(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], page, table.data_ptr(), table.shape[1])
    for window, sinks in ((0, 0), (1 << 30 if form == WIDE else 9, 1)):
        assert _form(rows, nh, kvh, dim, batch, capacity, window, sinks) == form
        with torch.cuda.device(DEV):
            size = lib.mp_masked_workspace_bytes(rows, nh, kvh, dim, batch, capacity, window, sinks)
        for head in ([0, 30, 10, 40], [40, 0, 0, 40], [-5, 100, 3, 1 << 30], [50, 50, 50, 50], [0, 13, 13, 40], [5, 6, 7, 20]):
            starts = _ints(head + [head[-1]] * (batch - 3))
            out, out_whole = _guarded(rows * nh * dim, F16, 7.0)
            ws, ws_whole = _guarded(size, torch.uint8, 0xA5)
            ws[:] = 0xFF  # nothing that was there counts
            with torch.cuda.device(DEV):
                a = (q.data_ptr(), nh * dim, dim, rows, nh, kvh, dim, cache, ln.data_ptr(), starts.data_ptr(), batch)
                z = (ctypes.c_float(0.1), out.data_ptr(), 0, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
                if window:
                    rc = lib.mp_paged_prompt_window_attention(*a, window, sinks, *z)
                else:
                    rc = lib.mp_paged_tree_attention(*a, m.data_ptr(), 1, *z)
            torch.cuda.synchronize()
            assert rc == 0 and out_whole() and ws_whole(), (head, window)
            if head == [0, 13, 13, 40]:  # these do ascend: all is written
                sees = mref.in_window(window, sinks) if window else mref.in_tree([[[0]] * 13, [], [[0]] * 27] + [[]] * (batch - 3))
                want, tol = mref.masked_attention(q, k, v, table, ln, torch.tensor(starts.tolist()), sees, 0.1)
                ref.check(out.view(rows, nh, dim), want, tol)
