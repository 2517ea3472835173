"""The bookkeeping of a paged cache on the host: forks, copies of begun pages, drafts taken up, trimmed pages.  The moves of keys and
values are the plain forms here."""
import random

import pytest
import torch

import masked_reference as mref
from mindpipe_amd import decoder
from mindpipe_amd.decoder import DecoderConfig, PagedKVCache, lookup_draft

CFG = DecoderConfig(layers=2, hidden=32, heads=2, kv_heads=1, ffn=64, vocab=50)


@pytest.fixture(autouse=True)
def _plain_moves(monkeypatch):
    def copy(k, v, src, dst, filled=None):
        for t in (k, v):
            t.copy_(mref.copied(t, src.tolist(), dst.tolist(), None if filled is None else filled.tolist()))

    def keep(k, v, table, first, keep, starts):
        for t in (k, v):
            t.copy_(mref.kept(t, table, first.tolist(), keep.tolist(), starts.tolist()))

    monkeypatch.setattr(decoder.ops, "paged_copy_pages", copy)
    monkeypatch.setattr(decoder.ops, "paged_keep_positions", keep)


class _Model:
    """What each sequence should hold, as lists of numbers that are written to the pages after each ``extend``."""

    def __init__(self, sequences, positions, max_len=None):
        self.cache = PagedKVCache(CFG, sequences, positions, 8, max_len, device="cpu")
        self.said = [[] for _ in range(sequences)]
        self.next = 1

    def extend(self, news):
        before = list(self.cache.length)
        self.cache.extend(news)
        for b, n in enumerate(news):
            for p in range(before[b], before[b] + n):
                page = int(self.cache.table[b, p // 8])
                for t in (self.cache.k, self.cache.v):
                    t[:, page, :, p % 8] = self.next % 2000
                self.said[b].append(self.next % 2000)
                self.next += 1

    def check(self, gone=lambda b, p: False):
        c = self.cache
        assert c.lens.tolist() == c.length == [len(s) for s in self.said]
        uses = [0] * c.k.shape[1]
        for b, said in enumerate(self.said):
            assert len(c._held[b]) == -(-len(said) // 8)
            for i, page in enumerate(c._held[b]):
                assert int(c.table[b, i]) == page
                if page >= 0:
                    uses[page] += 1
            for p, x in enumerate(said):
                page = int(c.table[b, p // 8])
                if page < 0:
                    assert gone(b, p)
                    continue
                assert (c.k[:, page, :, p % 8] == x).all() and (c.v[:, page, :, p % 8] == x).all(), (b, p)
        assert uses == c._uses and sorted(c._free) == [p for p, n in enumerate(uses) if not n]


def test_forks_share_pages_until_they_write():
    m = _Model(4, 8 * 12)
    m.extend([20, 0, 0, 3])
    m.cache.fork(0, 1)
    m.cache.fork(0, 2)
    m.said[1], m.said[2] = list(m.said[0]), list(m.said[0])
    m.check()
    assert m.cache.free_positions() == 8 * (12 - 4)  # nothing was copied
    m.extend([1, 1, 0, 1])  # two of three go on: both copy, the third keeps the page
    m.check()
    assert m.cache.free_positions() == 8 * (12 - 4 - 2)
    m.extend([0, 0, 4, 0])  # alone on its page: no copy
    m.check()
    assert m.cache.free_positions() == 8 * (12 - 4 - 2)
    with pytest.raises(ValueError):
        m.cache.fork(0, 3)
    for b in (0, 1, 2, 3):
        m.cache.release(b)
        m.said[b] = []
        m.check()
    assert m.cache.free_positions() == 8 * 12


def test_full_pages_are_not_copied():
    m = _Model(2, 8 * 4)
    m.extend([16, 0])
    m.cache.fork(0, 1)
    m.said[1] = list(m.said[0])
    m.extend([1, 1])
    m.check()
    assert m.cache.free_positions() == 0


def test_copies_that_do_not_fit_change_nothing():
    m = _Model(3, 8 * 3)
    m.extend([12, 0, 0])
    m.cache.fork(0, 1)
    m.cache.fork(0, 2)
    m.said[1], m.said[2] = list(m.said[0]), list(m.said[0])
    for news in ([1, 1, 1], [1, 1, 0]):  # two of three holders write, or two beside one that keeps it: two copies
        with pytest.raises(RuntimeError, match="2 pages"):
            m.cache.extend(news)
        m.check()
    m.extend([1, 0, 0])
    m.check()


def test_reorder_any_way():
    rng = random.Random(1)
    m = _Model(5, 8 * 40)
    for _ in range(60):
        order = [rng.randrange(5) for _ in range(5)]
        m.cache.reorder(order)
        m.said = [list(m.said[o]) for o in order]
        m.check()
        m.extend([rng.choice((0, 1, 1, 3)) if len(s) < 50 else 0 for s in m.said])
        m.check()
        if rng.random() < 0.2:
            b = rng.randrange(5)
            m.cache.release(b)
            m.said[b] = []
            m.check()
    for bad in ([0, 1, 2, 3], [0, 1, 2, 3, 5], [0, 1, 2, 3, -1]):
        with pytest.raises(ValueError):
            m.cache.reorder(bad)


def test_keep_takes_up_a_path():
    m = _Model(3, 8 * 12)
    m.extend([14, 3, 7])
    m.extend([9, 4, 0])
    m.cache.keep([9, 4, 0], [[0, 2, 5, 8], [], []])
    m.said[0][14:] = [m.said[0][14 + i] for i in (0, 2, 5, 8)]
    m.said[1][3:] = []
    m.check()
    assert m.cache.free_positions() == 8 * (12 - 3 - 1 - 1)
    m.extend([1, 1, 1])
    m.cache.keep([1, 1, 1], [[0], [0], [0]])  # nothing moves
    m.check()
    for drafted, kept in (([1, 1], [[], []]), ([1, 1, 1], [[1], [], []]), ([2, 0, 0], [[1, 0], [], []]), ([2, 0, 0], [[1, 1], [], []]),
                          ([99, 0, 0], [[], [], []]), ([-1, 0, 0], [[], [], []])):
        with pytest.raises(ValueError):
            m.cache.keep(drafted, kept)
    m.extend([3, 0, 0])
    m.cache.release(1)
    m.cache.fork(0, 1)
    with pytest.raises(RuntimeError, match="forked"):
        m.cache.keep([3, 0, 0], [[2], [], []])


def test_trim_frees_what_no_later_token_sees():
    m = _Model(2, 8 * 20)
    m.extend([50, 9])
    assert m.cache.trim(16, 3) == 3  # of pages 0 .. 6: 1, 2 and 3 lie before position 35, 0 holds the sinks
    gone = lambda b, p: b == 0 and 8 <= p < 32  # noqa: E731
    m.check(gone)
    assert m.cache.trim(16, 3) == 0
    assert m.cache.table[0, :7].tolist()[1:4] == [-1, -1, -1]
    m.cache.reorder([0, 0])
    m.said[1] = list(m.said[0])
    either = lambda b, p: 8 <= p < 32  # noqa: E731
    m.check(either)
    m.extend([7, 8])
    m.check(either)
    assert m.cache.trim(1) > 0
    m.cache.release(0)
    m.cache.release(1)
    assert m.cache.free_positions() == 8 * 20
    for bad in ((0, 0), (5, -1)):
        with pytest.raises(ValueError):
            m.cache.trim(*bad)


def test_lookup_draft():
    draft = lookup_draft(2, 6, 2)
    # "1 2" stood before "3 4 5" and, later, before "3 9 7": one tree, the later first
    assert draft([1, 2, 3, 4, 5, 0, 1, 2, 3, 9, 7, 1, 2]) == ([3, 9, 7, 4, 5], [-1, 0, 1, 0, 3])
    assert draft([1, 2, 3]) == ([], []) and draft([1, 2]) == ([], []) and draft([5]) == ([], [])
    tokens, parents = lookup_draft(1, 3, 3)([4, 4, 4, 4])
    assert len(tokens) == len(parents) <= 3 and all(p < i for i, p in enumerate(parents))
