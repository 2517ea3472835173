"""What the paged-cache and sampling operators refuse, before any launch: the operators' own checks on tensors that only say
they are on the GPU, and the C entry points' on host buffers that no check reaches through."""
import ctypes

import pytest
import torch

import paged_reference as ref
from mindpipe_amd import _lib, ops


class _Said(torch.Tensor):
    is_cuda = True


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Said)


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


class _NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture(autouse=True)
def _no_launch(monkeypatch):
    monkeypatch.setattr(ops._lib, "load", _NoLaunch)


CACHE = dict(k_pages=_t(6, 2, 16, 64), v_pages=_t(6, 2, 16, 64), table=_i(3, 4), lens=_i(3))
APPEND = dict(qkv=_t(3, 8 * 64), cos=_t(20, 32, dtype=torch.float32), sin=_t(20, 32, dtype=torch.float32), **CACHE)
DECODE = dict(q=_t(3, 4, 64), scale=0.1, **CACHE)
CHUNK = dict(q=_t(9, 4, 64), starts=_i(4), scale=0.1, **CACHE)
PROMPT = dict(q=_t(9, 4, 64), k=_t(9, 2, 64), v=_t(9, 2, 64), starts=_i(4), scale=0.1)
SAMPLE = dict(logits=_t(3, 50), u=_t(3, dtype=torch.float32))
BASE = {"paged_rope_append": APPEND, "paged_decode_attention": DECODE, "paged_prompt_attention": CHUNK, "prompt_attention": PROMPT,
        "sample_tokens": SAMPLE}
BAD_CACHE = [dict(k_pages=_t(6, 2, 16, 64, dtype=torch.bfloat16)), dict(v_pages=_t(6, 2, 8, 64)), dict(table=_t(3, 4)),
             dict(lens=_t(3, dtype=torch.int64)), dict(table=_i(2, 4)), dict(table=_i(3, 0)),
             dict(k_pages=_t(6, 2, 12, 64), v_pages=_t(6, 2, 12, 64)), dict(k_pages=_t(6, 2, 4, 64), v_pages=_t(6, 2, 4, 64)),
             dict(k_pages=_t(0, 2, 16, 64), v_pages=_t(0, 2, 16, 64)), dict(k_pages=_t(6, 2, 64, 16).transpose(2, 3)),
             dict(k_pages=_t(6, 2, 16, 68)[..., :64]), dict(v_pages=_t(2 * 6 * 16 * 64 + 1)[1:].view(6, 2, 16, 64)),
             dict(table=_i(4, 3).t()), dict(table=_i(1).expand(3, 1 << 27))]
BAD = {
    "paged_rope_append": BAD_CACHE + [
        dict(qkv=_t(4, 8 * 64)), dict(qkv=_t(3, 4 * 64)), dict(qkv=_t(3, 8 * 64 + 8)), dict(qkv=_t(3, 8 * 64, dtype=torch.float32)),
        dict(qkv=_t(3, 8 * 64 + 4)[:, :8 * 64]), dict(cos=_t(20, 32)), dict(sin=_t(19, 32, dtype=torch.float32)),
        dict(cos=_t(20, 40, dtype=torch.float32), sin=_t(20, 40, dtype=torch.float32)),
        dict(cos=_t(20, 4, dtype=torch.float32), sin=_t(20, 4, dtype=torch.float32)), dict(starts=_i(3)),
        dict(starts=_t(4, dtype=torch.int64)), dict(cos=_t(0, 32, dtype=torch.float32), sin=_t(0, 32, dtype=torch.float32))],
    "paged_decode_attention": BAD_CACHE + [
        dict(q=_t(2, 4, 64)), dict(q=_t(3, 3, 64)), dict(q=_t(3, 4, 128)), dict(q=_t(3, 4, 64, dtype=torch.bfloat16)),
        dict(q=_t(3, 4, 64, dtype=torch.float32)), dict(q=_t(3, 64, 4).transpose(1, 2)), dict(q=_t(3, 0, 64)),
        dict(q=_t(3, 4, 32), k_pages=_t(6, 2, 16, 32), v_pages=_t(6, 2, 16, 32)), dict(q=_t(3, 256))],
    "paged_prompt_attention": BAD_CACHE + [dict(starts=_i(3)), dict(starts=_t(4)), dict(q=_t(9, 3, 64)), dict(q=_t(9, 4, 128))],
    "prompt_attention": [dict(k=_t(8, 2, 64)), dict(v=_t(9, 1, 64)), dict(k=_t(9, 2, 64, dtype=torch.bfloat16)),
                         dict(starts=_i(0)), dict(starts=_t(4, dtype=torch.int64)), dict(q=_t(9, 3, 64)), dict(q=_t(9, 4, 128)),
                         dict(k=_t(9, 0, 64), v=_t(9, 0, 64)), dict(k=_t(9, 2, 68)[..., 2:66])],
    "sample_tokens": [dict(logits=_t(3, 50, dtype=torch.float64)), dict(logits=_t(50)), dict(logits=_t(50, 3).t()),
                      dict(logits=_t(3, 0)), dict(logits=_t(1, 1).expand(3, (1 << 19) + 1)), dict(u=_t(2, dtype=torch.float32)),
                      dict(u=_t(3, dtype=torch.float64)), dict(temperature=_t(3)), dict(top_k=_t(3, dtype=torch.int64)),
                      dict(top_p=_t(1, dtype=torch.float32)), dict(min_p=_t(3, 1, dtype=torch.float32)),
                      dict(logits=_t(1, 50).expand(3, 50)), dict(top_k=_i(6)[::2])],
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
    import contextlib
    monkeypatch.setattr(ops, "_dev", lambda t: contextlib.nullcontext())
    with pytest.raises(AssertionError, match="was reached"):
        getattr(ops, name)._init_fn(**BASE[name])


def test_c_entry_points_refuse():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    for n in ("mp_paged_rope_append", "mp_paged_decode_attention", "mp_prompt_attention", "mp_paged_prompt_attention",
              "mp_sample_tokens"):
        getattr(lib, n).argtypes = _lib.SIGNATURES[n][1]
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def cache(**over):
        f = dict(k=p, v=p, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024, v_row=64, pages=6, page_size=16, table=p,
                 width=4)
        return _lib.PAGES.pack(*(v or 0 for v in {**f, **over}.values()))

    def decode(c, q=p, b=3, nh=4, kvh=2, d=64, dt=0, ws=p, wsb=1 << 40):
        return lib.mp_paged_decode_attention(q, 256, 64, b, nh, kvh, d, c, p, 0.1, p, dt, ws, wsb, None)

    SHAPE, DTYPE, ALIGN, ARG = 1, 2, 3, 5
    assert decode(None) == ARG and decode(cache(), q=None) == ARG and decode(cache(k=None)) == ARG
    assert decode(cache(table=None)) == ARG and decode(cache(), ws=None) == ARG
    assert decode(cache(), dt=2) == DTYPE and decode(cache(), q=p + 2) == ALIGN and decode(cache(v=p + 8)) == ALIGN
    for bad in (dict(nh=5), dict(kvh=0), dict(d=96), dict(b=-1)):
        assert decode(cache(), **bad) == SHAPE
    for bad in (dict(page_size=24), dict(page_size=4), dict(pages=0), dict(width=0), dict(width=1 << 27), dict(k_row=60),
                dict(v_head=-64)):
        assert decode(cache(**bad)) == SHAPE
        assert lib.mp_paged_prompt_attention(p, 256, 64, 9, 4, 2, 64, cache(**bad), p, p, 3, 0.1, p, 0, p, 1 << 40, None) == SHAPE
        assert lib.mp_paged_rope_append(p, 512, 3, 4, 2, 64, p, p, 64, 20, 1, p, cache(**bad), p, None, 3, 0, None) == SHAPE
    for bad in ((p, 500, 3, 4, 2, 64, p, p, 64), (p, 512, 3, 4, 2, 60, p, p, 48), (p, 512, 3, 4, 2, 64, p, p, 80),
                (p, 512, 3, 4, 2, 64, p, p, 8), (p, 512, 4, 4, 2, 64, p, p, 64)):
        assert lib.mp_paged_rope_append(*bad, 20, 1, p, cache(), p, None, 3, 0, None) == SHAPE
    assert lib.mp_paged_rope_append(p, 512, 3, 4, 2, 64, p, p, 64, 0, 1, p, cache(), p, None, 3, 0, None) == SHAPE
    assert lib.mp_paged_rope_append(p, 512, 3, 4, 2, 64, p, p, 64, 20, 1, None, cache(), p, None, 3, 0, None) == ARG
    prompt = lambda *a, nh=4, kvh=2, d=64, rows=9, b=3, row=256, dt=0: lib.mp_prompt_attention(  # noqa: E731
        p, row, 64, p, 128, 64, p, 128, 64, rows, nh, kvh, d, *(a or (p,)), b, 0.1, p, dt, p, 1 << 40, None)
    assert prompt(None) == ARG and prompt(nh=3) == SHAPE and prompt(d=80) == SHAPE and prompt(b=0) == SHAPE
    assert prompt(row=-8) == SHAPE and prompt(row=252) == SHAPE and prompt(dt=2) == DTYPE and prompt(rows=1 << 40) == SHAPE
    sample = lambda x=p, stride=50, rows=3, vocab=50, dt=0, u=p: lib.mp_sample_tokens(  # noqa: E731
        x, stride, rows, vocab, dt, u, None, None, None, None, p, p, None)
    assert sample(x=None) == ARG and sample(u=None) == ARG and sample(dt=3) == DTYPE and sample(x=p + 1) == ALIGN
    assert sample(vocab=0) == SHAPE and sample(stride=49) == SHAPE and sample(vocab=(1 << 19) + 1, stride=1 << 20) == SHAPE


def test_the_reference_forms_agree_with_torch():
    """The plain forms that the GPU tests compare with, against torch's own softmax and sort."""
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(5, 2, 64, generator=g).half(), torch.randn(5, 1, 64, generator=g).half(), torch.randn(5, 1, 64, generator=g).half()
    out, _ = ref.prompt_attention(q, k, v, torch.tensor([0, 2, 5]), 0.125)
    s = (q.double().transpose(0, 1) @ k.double().squeeze(1).t()) * 0.125
    seq = torch.tensor([0, 0, 1, 1, 1])
    seen = (seq[:, None] == seq) & torch.ones(5, 5).tril().bool()
    want = (torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v.double().squeeze(1)).transpose(0, 1)
    assert torch.allclose(out, want, atol=1e-12)
    x = torch.tensor([[1.0, 3.0, 3.0, 2.0], [0.0, 0.0, 0.0, 0.0]])
    u = torch.tensor([0.0, 0.99])
    assert ref.sample(x, u, None, torch.tensor([1, 2]))[0].tolist() == [1, 1]
    assert ref.sample(x, u, None, None, torch.tensor([0.5, 0.5]))[0].tolist() == [1, 1]
    assert ref.sample(x, u, torch.zeros(2))[0].tolist() == [1, 0]
