"""What the operators of trees, windows, beams and page moves refuse, before any launch: the operators' own checks on tensors that
only say they are on the GPU, and the C entry points' on host buffers that no check reaches through."""
import contextlib
import ctypes

import pytest
import torch

import masked_reference as mref
from mindpipe_amd import _lib, ops


class _Said(torch.Tensor):
    is_cuda = True


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Said)


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def _f(*shape):
    return _t(*shape, dtype=torch.float32)


class _NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture(autouse=True)
def _no_launch(monkeypatch):
    monkeypatch.setattr(ops._lib, "load", _NoLaunch)


CACHE = dict(k_pages=_t(6, 2, 16, 64), v_pages=_t(6, 2, 16, 64), table=_i(3, 4), lens=_i(3))
TREE = dict(q=_t(9, 4, 64), starts=_i(4), masks=_t(9, 1, dtype=torch.int64), scale=0.1, **CACHE)
DECODE = dict(q=_t(3, 4, 64), scale=0.1, window=8, sinks=1, **CACHE)
CHUNK = dict(q=_t(9, 4, 64), starts=_i(4), scale=0.1, window=8, sinks=1, **CACHE)
POOLS = dict(k_pages=_t(2, 6, 2, 16, 64), v_pages=_t(2, 6, 2, 16, 64))
COPY = dict(**POOLS, src=_i(5), dst=_i(5), filled=_i(5))
KEEP = dict(**POOLS, table=_i(3, 4), first=_i(3), keep=_i(7), starts=_i(4))
BEAM = dict(logits=_t(6, 50), scores=_f(2, 3), count=6, ended=_t(2, 3, dtype=torch.bool), pad=1)
TURNS = dict(qkv=_t(3, 8 * 64), cos=_f(20, 32), sin=_f(20, 32), turns=_i(3), **CACHE)
BASE = {"paged_tree_attention": TREE, "paged_decode_window_attention": DECODE, "paged_prompt_window_attention": CHUNK,
        "paged_copy_pages": COPY, "paged_keep_positions": KEEP, "beam_select": BEAM, "paged_rope_append": TURNS}
BAD_CACHE = [dict(k_pages=_t(6, 2, 16, 64, dtype=torch.bfloat16)), dict(v_pages=_t(6, 2, 8, 64)), dict(table=_t(3, 4)),
             dict(lens=_t(3, dtype=torch.int64)), dict(table=_i(2, 4)), dict(table=_i(3, 0)),
             dict(k_pages=_t(6, 2, 12, 64), v_pages=_t(6, 2, 12, 64)), dict(k_pages=_t(0, 2, 16, 64), v_pages=_t(0, 2, 16, 64)),
             dict(k_pages=_t(6, 2, 64, 16).transpose(2, 3)), dict(k_pages=_t(6, 2, 16, 68)[..., :64]), dict(table=_i(4, 3).t()),
             dict(table=_i(1).expand(3, 1 << 27))]
WINDOWS = [dict(window=0), dict(window=-1), dict(window=(1 << 30) + 1), dict(sinks=-1), dict(sinks=(1 << 30) + 1)]
BAD_POOLS = [dict(k_pages=_t(2, 6, 2, 16, 64, dtype=torch.bfloat16)), dict(v_pages=_t(2, 6, 2, 8, 64)), dict(k_pages=_t(6, 2, 16, 64)),
             dict(k_pages=_t(2, 6, 2, 12, 64), v_pages=_t(2, 6, 2, 12, 64)), dict(k_pages=_t(2, 6, 2, 4, 64), v_pages=_t(2, 6, 2, 4, 64)),
             dict(k_pages=_t(2, 6, 2, 16, 60), v_pages=_t(2, 6, 2, 16, 60)), dict(k_pages=_t(2, 0, 2, 16, 64), v_pages=_t(2, 0, 2, 16, 64)),
             dict(k_pages=_t(2, 6, 2, 16, 1032), v_pages=_t(2, 6, 2, 16, 1032)), dict(k_pages=_t(0, 6, 2, 16, 64), v_pages=_t(0, 6, 2, 16, 64)),
             dict(k_pages=_f(2, 6, 2, 16, 64), v_pages=_f(2, 6, 2, 16, 64)), dict(v_pages=_t(2, 6, 2, 64, 16).transpose(3, 4)),
             dict(k_pages=_t(6, 2, 16, 64).expand(2, 6, 2, 16, 64)), dict(v_pages=_t(2, 6, 1, 16, 64).expand(2, 6, 2, 16, 64)),
             dict(k_pages=_t(16, 64), v_pages=_t(16, 64))]
BAD = {
    "paged_tree_attention": BAD_CACHE + [
        dict(starts=_i(3)), dict(starts=_t(4)), dict(q=_t(9, 3, 64)), dict(q=_t(9, 4, 128)), dict(q=_f(9, 4, 64)), dict(q=_t(9, 256)),
        dict(masks=_i(9, 1)), dict(masks=_t(8, 1, dtype=torch.int64)), dict(masks=_t(9, 0, dtype=torch.int64)),
        dict(masks=_t(9, 1025, dtype=torch.int64)), dict(masks=_t(9, dtype=torch.int64)), dict(masks=_t(2, 9, dtype=torch.int64).t())],
    "paged_decode_window_attention": BAD_CACHE + WINDOWS + [dict(q=_t(2, 4, 64)), dict(q=_t(3, 3, 64)), dict(q=_t(3, 4, 96))],
    "paged_prompt_window_attention": BAD_CACHE + WINDOWS + [dict(starts=_i(3)), dict(starts=_t(4)), dict(q=_t(9, 3, 64)), dict(q=_t(9, 4, 128))],
    "paged_copy_pages": BAD_POOLS + [dict(src=_i(4)), dict(dst=_t(5, dtype=torch.int64)), dict(src=_i(5, 1)), dict(filled=_i(6)),
                                     dict(filled=_f(5)), dict(src=_i(10)[::2])],
    "paged_keep_positions": BAD_POOLS + [dict(table=_t(3, 4)), dict(table=_i(3, 0)), dict(table=_i(2, 4)), dict(first=_i(2)),
                                         dict(first=_f(3)), dict(keep=_i(7, 1)), dict(keep=_t(7, dtype=torch.int64)), dict(starts=_i(3)),
                                         dict(starts=_t(4)), dict(table=_i(1).expand(3, 1 << 27))],
    "beam_select": [dict(logits=_t(6, 50, dtype=torch.float64)), dict(logits=_t(300)), dict(logits=_t(50, 6).t()), dict(logits=_t(6, 0)),
                    dict(logits=_t(5, 50)), dict(logits=_t(1, 50).expand(6, 50)), dict(logits=_t(1, 1).expand(6, (1 << 19) + 1)),
                    dict(scores=_t(2, 3)), dict(scores=_f(6)), dict(scores=_f(3, 2).t()), dict(count=0), dict(count=65),
                    dict(logits=_t(130, 50), scores=_f(2, 65), ended=None), dict(logits=_t(0, 50), scores=_f(2, 0), ended=None), dict(pad=50), dict(pad=-1),
                    dict(ended=_t(2, 3)), dict(ended=_t(3, 2, dtype=torch.bool)), dict(ended=_t(6, dtype=torch.bool))],
    "paged_rope_append": [dict(turns=_i(2)), dict(turns=_t(3, dtype=torch.int64)), dict(turns=_i(3, 1)), dict(turns=_i(6)[::2])],
}


@pytest.mark.parametrize("name,bad", [(n, b) for n, l in BAD.items() for b in l])
def test_operators_refuse(name, bad):
    with pytest.raises(RuntimeError):
        getattr(ops, name)._init_fn(**{**BASE[name], **bad})


@pytest.mark.parametrize("name", list(BASE))
def test_operators_refuse_the_cpu_and_other_things(name):
    first = next(iter(BASE[name]))
    plain = torch.Tensor(BASE[name][first].detach().as_subclass(torch.Tensor))
    with pytest.raises(RuntimeError, match="GPU"):
        getattr(ops, name)._init_fn(**{**BASE[name], first: plain})
    with pytest.raises(TypeError):
        getattr(ops, name)._init_fn(**{**BASE[name], first: None})


@pytest.mark.parametrize("name", list(BASE))
def test_the_base_calls_get_as_far_as_the_launch(name, monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda t: contextlib.nullcontext())
    with pytest.raises(AssertionError, match="was reached"):
        getattr(ops, name)._init_fn(**BASE[name])


def test_c_entry_points_refuse():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    for n in ("mp_paged_tree_attention", "mp_paged_prompt_window_attention", "mp_paged_decode_window_attention", "mp_paged_copy_pages",
              "mp_paged_keep_positions", "mp_beam_select", "mp_beam_select_workspace_bytes", "mp_masked_workspace_bytes",
              "mp_paged_rope_append_at"):
        getattr(lib, n).restype, getattr(lib, n).argtypes = _lib.SIGNATURES[n]
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    SHAPE, DTYPE, ALIGN, ARG, WORKSPACE = 1, 2, 3, 5, 6

    def cache(**over):
        f = dict(k=p, v=p, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024, v_row=64, pages=6, page_size=16, table=p,
                 width=4)
        return _lib.PAGES.pack(*(v or 0 for v in {**f, **over}.values()))

    def tree(c, q=p, rows=9, nh=4, kvh=2, d=64, b=3, masks=p, words=1, scale=0.1, dt=0, ws=p):
        return lib.mp_paged_tree_attention(q, 256, 64, rows, nh, kvh, d, c, p, p, b, masks, words, scale, p, dt, ws, 1 << 40, None)

    def chunk(c, window=5, sinks=0, **o):
        a = dict(q=p, row=256, rows=9, nh=4, kvh=2, d=64, b=3, dt=0, ws=p, starts=p)
        a.update(o)
        return lib.mp_paged_prompt_window_attention(a["q"], a["row"], 64, a["rows"], a["nh"], a["kvh"], a["d"], c, p, a["starts"], a["b"],
                                                    window, sinks, 0.1, p, a["dt"], a["ws"], 1 << 40, None)

    def decode(c, window=5, sinks=0, b=3, nh=4, dt=0):
        return lib.mp_paged_decode_window_attention(p, 256, 64, b, nh, 2, 64, c, p, window, sinks, 0.1, p, dt, p, 1 << 40, None)

    for call in (tree, chunk, decode):
        assert call(None) == ARG and call(cache(k=None)) == ARG and call(cache(table=None)) == ARG
        assert call(cache(), dt=2) == DTYPE and call(cache(), nh=5) == SHAPE and call(cache(), b=-1) == SHAPE
        assert call(cache(v=p + 8)) == ALIGN
        for bad in (dict(page_size=24), dict(page_size=4), dict(pages=0), dict(width=0), dict(width=1 << 27), dict(k_row=60), dict(v_head=-64)):
            assert call(cache(**bad)) == SHAPE
    assert tree(cache(), masks=None) == ARG and tree(cache(), words=0) == SHAPE and tree(cache(), words=1025) == SHAPE
    assert tree(cache(), q=None) == ARG and tree(cache(), q=p + 2) == ALIGN and tree(cache(), ws=None) == ARG and tree(cache(), d=96) == SHAPE
    assert tree(cache(), scale=float("nan")) == ARG and tree(cache(), scale=3e38) == ARG and tree(cache(), rows=1 << 40) == SHAPE
    for call in (chunk, decode):
        for bad in (dict(window=0), dict(window=1 << 31), dict(sinks=-1), dict(sinks=1 << 31)):
            assert call(cache(), **bad) == SHAPE
    assert chunk(cache(), starts=None) == ARG and chunk(cache(), b=0) == SHAPE and chunk(cache(), row=252) == SHAPE
    assert lib.mp_masked_workspace_bytes(0, 4, 2, 64, 3, 64, 0, 0) == 0
    assert lib.mp_masked_workspace_bytes(9, 5, 2, 64, 3, 64, 0, 0) == 0 and lib.mp_masked_workspace_bytes(9, 4, 2, 64, 3, 0, 0, 0) == 0

    def copy(c, layers=2, kvh=2, d=64, src=p, n=3):
        return lib.mp_paged_copy_pages(c, layers, 12288, 12288, kvh, d, src, p, None, n, None)

    def keep(c, layers=2, kvh=2, d=64, first=p, total=3, b=2, starts=p):
        return lib.mp_paged_keep_positions(c, layers, 12288, 12288, kvh, d, b, first, p, total, starts, None)

    for call in (copy, keep):
        assert call(None) == ARG and call(cache(v=None)) == ARG and call(cache(k=p + 8)) == ALIGN
        for bad in (dict(layers=0), dict(layers=1 << 20), dict(kvh=0), dict(d=60), dict(d=1032)):
            assert call(cache(), **bad) == SHAPE
        for bad in (dict(page_size=24), dict(pages=0), dict(k_row=60), dict(v_page=-8)):
            assert call(cache(**bad)) == SHAPE
    assert copy(cache(), src=None) == ARG and copy(cache(), n=-1) == SHAPE and copy(cache(), n=0) == 0
    assert keep(cache(table=None)) == ARG and keep(cache(width=0)) == SHAPE and keep(cache(), starts=None) == ARG
    assert keep(cache(), total=-1) == SHAPE and keep(cache(), b=-1) == SHAPE and keep(cache(), total=0) == 0

    def beam(x=p, stride=50, batch=2, beams=3, vocab=50, dt=0, pad=0, count=6, ws=p, wsb=1 << 40):
        return lib.mp_beam_select(x, stride, batch, beams, vocab, dt, p, None, pad, count, p, p, p, ws, wsb, None)

    assert beam(x=None) == ARG and beam(ws=None) == ARG and beam(dt=3) == DTYPE and beam(x=p + 1) == ALIGN and beam(ws=p + 8) == ALIGN
    for bad in (dict(stride=49), dict(batch=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=(1 << 19) + 1, stride=1 << 20),
                dict(pad=50), dict(pad=-1), dict(count=0), dict(count=65), dict(batch=1 << 40)):
        assert beam(**bad) == SHAPE
    assert beam(wsb=0) == WORKSPACE and beam(batch=0) == 0 and lib.mp_beam_select_workspace_bytes(1, 65, 50, 6) == 0


def test_the_reference_forms():
    """The plain forms that the GPU tests compare with, on small cases worked by hand or by torch."""
    x = torch.tensor([[0.0, 1.0, 1.0], [2.0, float("-inf"), 0.0]])
    scores = torch.tensor([[0.0, -0.5]])
    best, beam, token = mref.beams(x, scores, 4)
    total = (torch.log_softmax(x.double(), 1) + scores.double().view(2, 1)).flatten()
    order = torch.sort(total, descending=True, stable=True)[1][:4]
    assert beam[0].tolist() == (order // 3).tolist() and token[0].tolist() == (order % 3).tolist()
    assert torch.allclose(best[0], total[order], atol=1e-15)
    assert mref.beams(x, scores, 3, torch.tensor([[True, False]]), 2)[2][0].tolist() == [2, 0, 2]
    assert mref.ancestors([-1, 0, 0, 2]) == [[0], [0, 1], [0, 2], [0, 2, 3]]
    assert mref.masks([[[0, 63], [64]]], 2).tolist() == [[1 - (1 << 63), 0], [0, 1]]
    assert mref.in_window(3, 1)(0, 1, 2, 8) == [0, 5, 6, 7] and mref.in_tree([[[1]]])(0, 0, 2, 4) == [0, 1, 3]
    pages = torch.arange(8.0).view(1, 2, 1, 4, 1)
    assert mref.copied(pages, [0], [1], [2]).flatten().tolist() == [0, 1, 2, 3, 0, 1, 6, 7]
    assert mref.kept(pages, torch.tensor([[1, 0]]), [1], [1, 4], [0, 2]).flatten().tolist() == [0, 1, 2, 3, 4, 6, 1, 7]
