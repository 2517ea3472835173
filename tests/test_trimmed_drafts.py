"""Drafts of a paged cache whose pages were trimmed: none is taken up so short that a later token would look at a page that is gone."""
import pytest

from test_paged_cache import _Model, _plain_moves  # noqa: F401


def _look(m, window, sinks=0):
    """What the next token of each sequence looks at is there."""
    c = m.cache
    for b, n in enumerate(c.length):
        for p in range(n):
            if p < sinks or p > n - window:
                assert int(c.table[b, p // 8]) >= 0, (b, p)


@pytest.mark.parametrize("window,sinks", [(8, 0), (8, 3), (11, 0), (20, 8)])
def test_a_draft_is_not_cut_below_what_was_trimmed(window, sinks):
    m = _Model(2, 8 * 20)
    m.extend([40, 5])
    m.extend([9, 3])
    assert m.cache.trim(window, sinks) > 0
    before = (list(m.cache.length), m.cache.table.tolist(), list(m.cache._free))
    refused = 0
    for n in range(10):
        least = 40 + n  # what would be left
        gone = any(p < least and sinks <= p and p > least - window and int(m.cache.table[0, p // 8]) < 0 for p in range(least))
        if gone:
            refused += 1
            with pytest.raises(RuntimeError, match="trimmed"):
                m.cache.keep([9, 0], [list(range(n)), []])
            assert before == (list(m.cache.length), m.cache.table.tolist(), list(m.cache._free))
    assert refused
    m.cache.keep([9, 3], [list(range(9)), [0]])
    assert m.cache.length == [49, 6]
    _look(m, window, sinks)


def test_drafts_behind_trimmed_pages_are_taken_up():
    """Trimmed before the draft, as a server does it: any path is taken up, and forks and released sequences keep to it."""
    m = _Model(2, 8 * 30)
    m.extend([60, 0])
    for kept in ([0], [], [0, 3, 5], [0, 1, 2, 3, 4, 5, 6, 7, 8]):
        m.cache.trim(10, 2)
        m.extend([9, 0])
        m.cache.keep([9, 0], [kept, []])
        _look(m, 10, 2)
    m.extend([9, 0])
    m.cache.trim(10, 2)
    m.cache.fork(0, 1)
    m.extend([1, 1])
    m.cache.keep([1, 1], [[], [0]])
    _look(m, 10, 2)
    n = m.cache.length[1]
    m.cache.release(0)
    m.extend([5, 9])
    m.cache.keep([5, 9], [[], [2]])
    assert m.cache.length == [0, n + 1]
    m.extend([30, 0])
    m.cache.keep([20, 0], [[0], []])  # a new sequence in the place of one that was trimmed
    assert m.cache.length[0] == 11
    with pytest.raises(RuntimeError, match="trimmed"):
        m.cache.keep([0, 9], [[], []])
