"""Drafts that come true are taken up, several tokens a pass; drafts that do not cost no token and save no pass."""
import pytest
import torch

from test_gpu_drafts_beams_windows import VOCAB, _model, _near_best, _reference, _tokens

pytestmark = pytest.mark.gpu
NEW = 12


def _run(model, prompts, draft):
    """(tokens, lengths of the paths that each pass took of each sequence)"""
    from mindpipe_amd.decoder import PagedKVCache
    took, keep = [], PagedKVCache.keep

    def watched(self, drafted, kept):
        took.append([len(k) for k in kept])
        return keep(self, drafted, kept)

    PagedKVCache.keep = watched
    try:
        return model.generate_drafted(prompts, NEW, draft), took
    finally:
        PagedKVCache.keep = keep


def _after(prompts, said, tokens):
    for p, t in zip(prompts, said.tolist()):
        n = p.numel()
        if tokens[:n] == p.tolist():
            return t[len(tokens) - n:]
    raise AssertionError("a draft of no prompt")


def test_true_drafts_save_passes():
    """What the model says without drafts is drafted, beside wrong tokens: one token from the prompts, then four drafted ones and one
    more a pass."""
    model, prompts = _model(4, 2, seed=11), _tokens(20, 33, 6, seed=12)
    said, took = _run(model, prompts, lambda t: ([], []))
    assert took == [[1, 1, 1]] * (NEW - 1)

    def knows(tokens):
        true = _after(prompts, said, tokens)[:4]
        wrong = [(x + 1) % VOCAB for x in true]
        chain = list(range(-1, len(true) - 1))
        return wrong + true, chain + [p + len(true) if p >= 0 else -1 for p in chain]

    got, took = _run(model, prompts, knows)
    assert torch.equal(got, said)
    assert took == [[5, 5, 5], [5, 5, 5], [1, 1, 1]]

    def errs(tokens):
        wrong = [(x + 1) % VOCAB for x in _after(prompts, said, tokens)[:4]]
        return wrong, list(range(-1, len(wrong) - 1))

    got, took = _run(model, prompts, errs)
    assert torch.equal(got, said) and took == [[1, 1, 1]] * (NEW - 1)
    for p, row in zip(prompts, got):
        logits = _reference(model, torch.cat((p, row)))
        assert all(_near_best(logits[p.numel() - 1 + i], row[i]) for i in range(NEW))

