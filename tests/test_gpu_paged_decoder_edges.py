"""The decoder stack on a paged cache where a sequence has nothing to answer with, or nothing new to answer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(heads, kv_heads, max_len=160, seed=5):
    from mindpipe_amd.decoder import DecoderConfig, W4Decoder
    cfg = DecoderConfig(layers=2, hidden=heads * 128, heads=heads, kv_heads=kv_heads, ffn=512, vocab=512)
    return W4Decoder(cfg, max_batch=1, max_len=max_len, device=DEV, seed=seed)


def _tokens(*lengths, seed=6):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(0, 512, (n,), device=DEV, generator=g) for n in lengths]


@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_a_sequence_without_a_token_stays_ended(monkeypatch, value):
    """Logits that leave nothing to take in one step only: -1 from there on, no token outside the vocabulary is looked up, and
    the other sequences answer as they do without."""
    model = _model(4, 2)
    prompts = _tokens(17, 9, 5)
    g = torch.Generator(device=DEV)
    t = torch.full((3,), 0.9, device=DEV)
    want = model.generate_paged(prompts, 7, temperature=t, generator=g.manual_seed(3))
    forward, seen = model.forward_paged, []

    def spoilt(tokens, cache, starts=None):
        logits = forward(tokens, cache, starts)
        seen.append(tokens.clone())
        if len(seen) == 3:
            logits[1] = value
        return logits

    monkeypatch.setattr(model, "forward_paged", spoilt)
    got = model.generate_paged(prompts, 7, temperature=t, generator=g.manual_seed(3))
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[1, :2], want[1, :2])
    assert (got[1, 2:] == -1).all()
    assert len(seen) == 7 and all(int(s.min()) >= 0 and int(s.max()) < 512 for s in seen)


def test_a_sequence_without_new_tokens_has_no_logits():
    """Idle sequences, first, between others, last and ended ones among them: -inf, and no token, in place of another sequence's;
    the others' logits are those of a step without them (fp16 hidden states; other counts of rows take other kernels)."""
    from mindpipe_amd import ops
    model = _model(4, 2)
    cache = model.paged_cache(5, 5 * 160, 16)
    alone = model.paged_cache(2, 2 * 160, 16)
    a, b = _tokens(40, 7)
    cache.extend([1, 30, 1, 1, 1])  # what the idle ones hold is of no matter here
    for s in (0, 1, 2, 3):
        cache.release(s)
    logits = model.forward_paged(torch.cat((a, b)), cache, cache.extend([0, 40, 0, 7, 0]))
    want = model.forward_paged(torch.cat((a, b)), alone, alone.extend([40, 7]))
    assert (logits[[1, 3]].float() - want.float()).norm() <= 2e-2 * want.float().norm()
    assert (logits[[0, 2, 4]] == -math.inf).all()
    tokens, logprobs = ops.sample_tokens(logits, torch.full((5,), 0.5, device=DEV))
    assert (tokens[[0, 2, 4]] == -1).all() and (tokens[[1, 3]] >= 0).all()
    tokens, _ = ops.sample_tokens(logits, torch.full((5,), 0.5, device=DEV), torch.zeros(5, device=DEV))
    assert (tokens[[0, 2, 4]] == -1).all() and torch.equal(tokens[[1, 3]], logits[[1, 3]].argmax(-1))
