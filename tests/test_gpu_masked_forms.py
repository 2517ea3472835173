"""Which form of the masked attention kernels a call takes (``mp_masked_item_rows``), and each form against plain 64-bit forms."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
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
