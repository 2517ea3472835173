"""Sequences that share no page cost ``extend`` no look at each one's begun page, and the count of shared holds that says so is right
after any forks, copies, drafts and releases."""
import random

from test_paged_cache import _Model, _plain_moves  # noqa: F401


class _Counted(list):
    reads = 0

    def __getitem__(self, i):
        _Counted.reads += 1
        return list.__getitem__(self, i)


def _shared(cache):
    return sum(max(0, n - 1) for n in cache._uses)


def test_no_looks_where_nothing_is_shared():
    m = _Model(6, 8 * 60)
    m.extend([13, 5, 0, 22, 8, 1])
    m.cache._uses = _Counted(m.cache._uses)
    for _ in range(10):
        m.extend([1] * 6)
    assert _Counted.reads == 0
    m.cache.release(2)
    m.cache.fork(0, 2)
    m.said[2] = list(m.said[0])
    _Counted.reads = 0
    m.extend([1] * 6)
    assert _Counted.reads > 0
    m.check()


def test_the_count_of_shared_holds():
    rng, m = random.Random(3), _Model(5, 8 * 60)
    for _ in range(120):
        what = rng.randrange(4)
        if what == 0:
            order = [rng.randrange(5) for _ in range(5)]
            m.cache.reorder(order)
            m.said = [list(m.said[o]) for o in order]
        elif what == 1:
            b = rng.randrange(5)
            m.cache.release(b)
            m.said[b] = []
        else:
            news = [rng.choice((0, 1, 1, 5)) if len(s) < 60 else 0 for s in m.said]
            m.extend(news)
            if what == 3:
                kept = [[i for i in range(n) if rng.random() < 0.5] for n in news]
                m.cache.keep(news, kept)
                m.said = [s[:len(s) - n] + [s[len(s) - n + i] for i in k] for s, n, k in zip(m.said, news, kept)]
        m.check()
        assert m.cache._shared == _shared(m.cache)
