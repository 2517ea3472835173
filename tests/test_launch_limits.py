"""Calls of more workgroups than a launch holds are refused before any launch: the C entry points' own checks, on host buffers that no
check reaches through."""
import ctypes

import pytest

from mindpipe_amd import _lib

SHAPE = 1
MOST = (1 << 24) - 1  # workgroups of 256 threads: a grid has below 2^32 threads


@pytest.fixture
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    for n in ("mp_paged_copy_pages", "mp_paged_keep_positions", "mp_beam_select"):
        getattr(lib, n).restype, getattr(lib, n).argtypes = _lib.SIGNATURES[n]
    return lib


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 15) // 16 * 16


def _cache(p, size, dim):
    return _lib.PAGES.pack(p, p, size * dim, size * dim, dim, size * dim, size * dim, dim, 6, size, p, 4)


def test_page_moves(lib, p):
    for dim, each in ((64, 1), (1024, 16)):  # 32 positions of a head: 256 pieces of 16 bytes, and 16 times as many
        c = _cache(p, 32, dim)
        assert lib.mp_paged_copy_pages(c, 1, 4096, 4096, 1, dim, p, p, None, MOST // each + 1, None) == SHAPE
        assert lib.mp_paged_copy_pages(c, 2, 4096, 4096, 1, dim, p, p, None, 1 << 30, None) == SHAPE
    c = _cache(p, 16, 1024)
    assert lib.mp_paged_keep_positions(c, 1, 4096, 4096, 1, 1024, MOST + 1, p, p, 3, p, None) == SHAPE  # 256 columns a sequence
    assert lib.mp_paged_keep_positions(c, 8, 4096, 4096, 1, 1024, MOST // 8 + 1, p, p, 3, p, None) == SHAPE


def test_beams(lib, p):
    for batch, beams, vocab in ((131071, 64, 32769), (131071, 64, 1 << 19), (8388607, 1, 40000)):
        assert lib.mp_beam_select(p, 1 << 19, batch, beams, vocab, 0, p, None, 0, 4, p, p, p, p, 1 << 60, None) == SHAPE
