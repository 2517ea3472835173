"""The decoder stack on a paged cache (append, prompt and decode attention, sampling, as a server runs them) against the same
stack in PyTorch ops over a contiguous cache."""
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _rel(a, b):
    return ((a - b).norm() / b.norm()).item()


def _model(heads, kv_heads, max_len=160, seed=5):
    from mindpipe_amd.decoder import DecoderConfig, W4Decoder
    cfg = DecoderConfig(layers=2, hidden=heads * 128, heads=heads, kv_heads=kv_heads, ffn=512, vocab=512)
    return W4Decoder(cfg, max_batch=1, max_len=max_len, device=DEV, seed=seed)


def _tokens(*lengths, seed=6):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(0, 512, (n,), device=DEV, generator=g) for n in lengths]


# Bounds as for the stack's other paths: fp16 hidden states through two layers, fused kernels on one side and PyTorch ops
# with other roundings on the other.
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1), (8, 2)])
@pytest.mark.parametrize("page", [8, 64])
def test_prompts_chunks_and_steps_match_torch(heads, kv_heads, page):
    _say("paged decoder", heads, kv_heads, page)
    model = _model(heads, kv_heads)
    prompts = _tokens(70, 1, 33)
    cache = model.paged_cache(3, 3 * 160, page)
    # the first 40 tokens of the first prompt and all of the last, then the rest
    starts = cache.extend([40, 0, 33])
    model.forward_paged(torch.cat([prompts[0][:40], prompts[2]]), cache, starts)
    starts = cache.extend([30, 1, 0])
    logits = model.forward_paged(torch.cat([prompts[0][40:], prompts[1]]), cache, starts)
    steps = _tokens(3, seed=7)[0]
    cache.extend([1, 1, 1])
    after = model.forward_paged(steps, cache)
    for b in range(3):
        want = model.prefill_torch(prompts[b][None], return_logits=True)
        if b < 2:
            assert _rel(logits[b].float(), want[0].float()) <= 2e-2
        n = prompts[b].numel()
        cur = torch.tensor([n], device=DEV)
        want = model.decode_step_torch(steps[b:b + 1], cur, return_logits=True)
        assert _rel(after[b].float(), want[0].float()) <= 2e-2
        # what the pages hold is what the contiguous cache holds
        pages = cache.table[b, :-(-(n + 1) // page)].long()
        for paged, flat in ((cache.k, model.k_cache), (cache.v, model.v_cache)):
            have = paged[:, pages].transpose(1, 2).flatten(2, 3)[:, :, :n + 1]
            assert _rel(have.float(), flat[:, 0, :, :n + 1].float()) <= 1e-2


def test_captured_steps():
    """A step captured once and replayed after each extend, with new tokens copied in, gives the eager step's bits."""
    model = _model(4, 2)
    prompts = _tokens(50, 9)
    caches = [model.paged_cache(2, 2 * 160, 16) for _ in range(2)]
    for c in caches:
        model.forward_paged(torch.cat(prompts), c, c.extend([50, 9]))
    tokens = _tokens(2, seed=8)[0]
    u, t = torch.rand(2, device=DEV), torch.full((2,), 0.7, device=DEV)

    def step(cache):
        from mindpipe_amd import ops
        logits = model.forward_paged(tokens, cache)
        return logits, *ops.sample_tokens(logits, u, t)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    caches[0].extend([1, 1])
    caches[1].extend([1, 1])
    with torch.cuda.stream(side):
        step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(12):
        graph.replay()
        got = [o.clone() for o in out]
        want = step(caches[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        tokens.copy_(got[1])
        u.uniform_()
        for c in caches:
            c.extend([1, 1])
        torch.cuda.synchronize()


def test_generate_greedy_and_sampled():
    model = _model(4, 2)
    prompts = _tokens(17, 64, 5)
    got = model.generate_paged(prompts, 6)
    assert got.shape == (3, 6)
    for b, p in enumerate(prompts):  # each prompt alone, and again whole after every token
        assert torch.equal(model.generate_paged([p], 6)[0], got[b])
    g = torch.Generator(device=DEV)
    settings = dict(temperature=torch.tensor([0.0, 0.9, 1.2], device=DEV), top_k=torch.tensor([0, 20, 0], device=DEV, dtype=torch.int32),
                    top_p=torch.tensor([1.0, 0.9, 0.8], device=DEV), min_p=torch.tensor([0.0, 0.0, 0.05], device=DEV))
    a = model.generate_paged(prompts, 6, generator=g.manual_seed(1), **settings)
    b = model.generate_paged(prompts, 6, generator=g.manual_seed(1), **settings)
    assert torch.equal(a, b) and torch.equal(a[0], got[0]) and int(a.min()) >= 0 and int(a.max()) < 512


def test_cache_keeps_its_pages():
    model = _model(2, 2)
    cache = model.paged_cache(3, 40, 8)
    with pytest.raises(RuntimeError, match="pages"):
        cache.extend([20, 20, 8])
    with pytest.raises(RuntimeError, match="pass"):
        cache.extend([161, 0, 0])
    with pytest.raises(ValueError):
        cache.extend([1, 1])
    assert cache.length == [0, 0, 0] and cache.free_positions() == 40
    cache.extend([9, 8, 1])
    held = set(cache.table[0, :2].tolist() + cache.table[1, :1].tolist() + cache.table[2, :1].tolist())
    assert len(held) == 4 and cache.free_positions() == 8 and cache.lens.tolist() == [9, 8, 1]
    cache.release(0)
    assert cache.free_positions() == 24 and cache.lens.tolist() == [0, 8, 1]
    starts = cache.extend([1, 1, 1])
    assert starts is None and cache.lens.tolist() == [1, 9, 2]
    assert cache.extend([0, 2, 0]).tolist() == [0, 0, 2, 2]


def test_calls_that_are_refused():
    from mindpipe_amd.decoder import PagedKVCache
    model = _model(2, 2, max_len=20)
    cache = PagedKVCache(model.cfg, 2, 100, 8)
    graph, tokens = torch.cuda.CUDAGraph(), torch.zeros(2, device=DEV, dtype=torch.int64)
    cache.extend([1, 1])
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            model.forward_paged(tokens, cache)
    for bad in (tokens[:0], tokens.view(1, 2)):
        with pytest.raises(ValueError, match="tokens"):
            model.forward_paged(bad, cache)
    with pytest.raises(RuntimeError):
        model.forward_paged(tokens[:1], cache)
    starts = cache.extend([20, 0])
    with pytest.raises(RuntimeError, match="positions"):
        model.forward_paged(torch.zeros(20, device=DEV, dtype=torch.int64), cache, starts)


def test_fewer_tokens_than_the_offsets_say():
    """What such a call returns is open; it reads no token that is not there."""
    model = _model(2, 2)
    cache = model.paged_cache(2, 100, 8)
    starts = cache.extend([30, 5])
    assert model.forward_paged(_tokens(10)[0], cache, starts).shape == (2, 512)
    torch.cuda.synchronize()
