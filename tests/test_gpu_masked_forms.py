"""Which form of the masked attention kernels a call takes (``mp_masked_item_rows``), and each form against plain 64-bit forms."""
import pytest
import torch

import masked_reference as mref
import paged_reference as ref
from test_gpu_masked import _ints, _ops, _starts, _trees

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
NARROW, WIDE = 16, 128


def _form(rows, nh, kvh, dim, batch, capacity, window=0, sinks=0):
    from mindpipe_amd import _lib
    with torch.cuda.device(DEV):
        torch.cuda.current_stream()
        return _lib.load().mp_masked_item_rows(rows, nh, kvh, dim, batch, capacity, window, sinks)


def test_new_tokens_of_one_sequence_among_many():
    """Sequences without new tokens do not make a call one of few rows: its rows may all be one sequence's, behind all that the
    table has room for."""
    for rows, nh, kvh in ((512, 32, 8), (512, 32, 32), (128, 64, 8), (2048, 64, 64)):
        assert _form(rows, nh, kvh, 128, 64, 9000) == WIDE
        assert _form(rows, nh, kvh, 128, 1, 9000) == WIDE
        assert _form(rows, nh, kvh, 128, 64, 1 << 20, 4096, 4) == WIDE
    assert _form(512, 8, 8, 256, 64, 3000) == WIDE and _form(2048, 32, 8, 64, 256, 20000) == WIDE


def test_few_rows_and_little_work():
    assert _form(1, 32, 32, 128, 1, 2048) == NARROW and _form(26, 32, 32, 128, 1, 1600) == NARROW
    assert _form(64, 64, 8, 128, 64, 2000) == NARROW and _form(128, 8, 8, 256, 32, 3000) == NARROW
    assert _form(16, 32, 8, 128, 1, 4096) == NARROW and _form(200, 4, 1, 64, 3, 300) == NARROW


def test_no_such_call():
    for bad in ((0, 4, 2, 64, 1, 64), (9, 5, 2, 64, 1, 64), (9, 4, 2, 64, 0, 64), (9, 4, 2, 64, 1, 0), (9, 4, 2, 64, 1, 64, -1)):
        assert _form(*bad) == 0


# ---------------------------------------------------------------- the narrow form's weights
def _pages_of(lens, kvh, dim, page, dtype, g, signs=False):
    width = max(-(-n // page) for n in lens)
    shape = (len(lens) * width, kvh, page, dim)
    k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g)
    v = torch.where(v < 0, -1.0, 1.0).to(dtype) if signs else v.to(dtype)
    return k.to(DEV), v.to(DEV), torch.randperm(shape[0], generator=g).view(len(lens), width).to(torch.int32).to(DEV)


def _rows(pages, table, b, n):
    return pages[table[b].long()].cpu().transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])[:n].double()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 7), (128, 2, 4), (256, 1, 5)])
@pytest.mark.parametrize("news,lens", [([1, 2, 3, 1], [2, 3, 7, 31]), ([3, 1, 5, 1], [40, 129, 500, 1]), ([4], [3000])])
def test_narrow_keeps_the_weights_bits(dtype, dim, kvh, grp, news, lens):
    """Values of 1 and -1, whose sums cancel: a weight rounded once to the type would be off by half a step, and the output by
    much of that.  What the rounding leaves is added, rounded itself: half a step of half a step of the sum of magnitudes, as for
    the single tokens that a draft's nodes stand in for."""
    g = torch.Generator().manual_seed(dim + len(lens))
    k, v, table = _pages_of(lens, kvh, dim, 16, dtype, g, signs=True)
    at, scale, ln = _starts(news), dim ** -0.5, _ints(lens)
    q = torch.randn(at[-1], kvh * grp, dim, generator=g).to(dtype).to(DEV)
    sets, window, sinks = _trees(news, 5), 300, 3
    capacity = 16 * table.shape[1]
    assert _form(at[-1], kvh * grp, kvh, dim, len(lens), capacity) == NARROW
    assert _form(at[-1], kvh * grp, kvh, dim, len(lens), capacity, window, sinks) == NARROW
    for got, sees in ((_ops().paged_tree_attention(q, k, v, table, ln, _ints(at), mref.masks(sets, 1).to(DEV), scale), mref.in_tree(sets)),
                      (_ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), scale, window, sinks),
                       mref.in_window(window, sinks))):
        for b, (n, length) in enumerate(zip(news, lens)):
            of_k, of_v = _rows(k, table, b, length), _rows(v, table, b, length)
            for j in range(n):
                of = sees(b, j, n, length)
                for h in range(kvh * grp):
                    want, bound = ref.attention_row(q[at[b] + j, h].cpu().double(), of_k[of, h // grp], of_v[of, h // grp], scale)
                    ref.check(got[at[b] + j, h], want, _allowed_twice(bound, dtype), what=f"sequence {b} row {j} head {h}")


def _allowed_twice(bound, dtype):
    """``ref.allowed`` where the rounding's rest is added: its own rounding in place of half a step of the magnitudes."""
    if isinstance(bound, torch.Tensor):
        return bound
    out, size, rel, low = bound
    half = ref.HALF_STEP[dtype]
    return half * out + (half * half * (1 + half) + 1.01 * rel) * size + low + (2.0 ** -24 if dtype == F16 else 0.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kvh,grp", [(64, 2, 7), (128, 2, 4), (256, 1, 5)])
def test_narrow_over_infinite_values(dtype, dim, kvh, grp):
    """An infinity in a value that all rows see goes to its own column, with its sign, and two of different signs give NaN; the
    others keep their sums.  One in a node goes to its descendants."""
    news, lens = [1, 3, 4, 6], [1, 8, 200, 2000]
    g = torch.Generator().manual_seed(dim)
    k, v, table = _pages_of(lens, kvh, dim, 16, dtype, g)
    for b, at in ((0, 0), (1, 0), (1, 6), (2, 33), (2, 198), (3, 0), (3, 1024), (3, 1997)):
        v[int(table[b, at // 16]), :, at % 16, 2 + at % 5] = float("inf") if at % 2 else -float("inf")
    for b, at in ((2, 7), (2, 150), (3, 5), (3, 1600)):
        v[int(table[b, at // 16]), :, at % 16, 9] = float("inf") if at % 2 else -float("inf")
    at, scale, ln = _starts(news), dim ** -0.5, _ints(lens)
    q = torch.randn(at[-1], kvh * grp, dim, generator=g).to(dtype).to(DEV)
    sets = _trees(news, 5)
    assert _form(at[-1], kvh * grp, kvh, dim, len(lens), 16 * table.shape[1]) == NARROW
    got = _ops().paged_tree_attention(q, k, v, table, ln, _ints(at), mref.masks(sets, 1).to(DEV), scale)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_tree(sets), scale))
    got = _ops().paged_prompt_window_attention(q, k, v, table, ln, _ints(at), scale, 1500, 2)
    ref.check(got, *mref.masked_attention(q, k, v, table, ln, torch.tensor(at), mref.in_window(1500, 2), scale))


# ---------------------------------------------------------------- what a launch does not hold
@pytest.mark.parametrize("batch,kvh", [(65536, 65536), (1 << 20, 4096), (1 << 18, 64)])
def test_more_workgroups_than_a_launch_holds(batch, kvh):
    """Sequences times key-value heads past what a grid has: refused, not cut to its low bits."""
    k = torch.zeros(1, kvh, 8, 64, device=DEV, dtype=F16)
    table, ln = torch.zeros(batch, 1, device=DEV, dtype=torch.int32), torch.ones(batch, device=DEV, dtype=torch.int32)
    starts = torch.ones(batch + 1, device=DEV, dtype=torch.int32)
    starts[0] = 0
    q, m = torch.zeros(1, kvh, 64, device=DEV, dtype=F16), torch.ones(1, 1, device=DEV, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="shape"):
        _ops().paged_tree_attention(q, k, k, table, ln, starts, m, 0.1)
    with pytest.raises(RuntimeError, match="shape"):
        _ops().paged_prompt_window_attention(q, k, k, table, ln, starts, 0.1, 4, 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_narrow_repeats_its_bits(dtype, dim):
    """NaN in a key, an infinity and NaN in values: the same bits again, those of the NaN included."""
    news, lens = [5, 1, 30], [700, 90, 400]
    g = torch.Generator().manual_seed(dim)
    k, v, table = _pages_of(lens, 2, dim, 16, dtype, g)
    k[int(table[0, 43]), 0, 10], v[int(table[2, 24]), 1, 3], v[int(table[0, 1]), 0, 2, 5] = float("nan"), float("nan"), float("inf")
    at, ln = _ints(_starts(news)), _ints(lens)
    q = torch.randn(36, 6, dim, generator=g).to(dtype).to(DEV)
    m = mref.masks(_trees(news, 2), 1).to(DEV)
    assert _form(36, 6, 2, dim, 3, 16 * table.shape[1]) == NARROW
    for call in (lambda: _ops().paged_tree_attention(q, k, v, table, ln, at, m, 0.1),
                 lambda: _ops().paged_prompt_window_attention(q, k, v, table, ln, at, 0.1, 300, 40)):
        got = call()
        assert got.isnan().any() and torch.isfinite(got).any()
        for _ in range(5):
            assert torch.equal(got.view(torch.int16), call().view(torch.int16))
