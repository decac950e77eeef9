"""Verification with every number of CTAs a sequence (1, 2, 4, 8) and bushes of many siblings, against the plain walk in 64 bits:
whole numbers, which are equal."""
from __future__ import annotations

import pytest
import torch

from test_verify_gpu import _case, _expected, _ints

pytestmark = pytest.mark.gpu


def _clusters(n_seqs, vocab):
    """CTAs a sequence: the most that their number of sequences allows, in parts of 2048 tokens or more."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    most = 8 if n_seqs <= sms // 2 else 4 if n_seqs <= 2 * sms else 2
    n = 1
    while n < most and vocab // (2 * n) >= 2048:
        n *= 2
    return n


@pytest.mark.parametrize("new,vocab,chain,drafted,dtype,clusters", [
    ([4] * 100, 9001, False, True, torch.float32, 4),
    ([5] * 290, 8192, False, True, torch.bfloat16, 4),
    ([3] * 150, 20011, True, False, torch.float16, 4),
    ([9, 1, 30], 12345, False, True, torch.float32, 4),
    ([7] * 20, 16383, False, False, torch.float32, 4),
    ([3] * 300, 9000, False, True, torch.float32, 2),
    ([8, 2], 8191, False, True, torch.float16, 2),
    ([8, 2], 4095, False, True, torch.float32, 1),
    ([8] * 70, 16385, False, True, torch.float16, 8),
])
def test_walk_and_token_are_the_plain_ones(cuda, new, vocab, chain, drafted, dtype, clusters):
    from asterq.speculative import verify_drafts

    assert _clusters(len(new), vocab) == clusters
    for seed in range(2):
        target, draft, tokens, parents, starts, accept, sample = _case(new, vocab, chain, drafted, dtype, seed)
        want = _expected(target, draft, tokens, parents, starts, accept, sample)
        status = _ints([0])
        up = None if chain else _ints([p for t in parents for p in t])
        got = verify_drafts(target, tokens, _ints(starts), up, accept, sample, draft_probs=draft, status=status)
        assert status.item() == 0
        for x, y in zip(got, want):
            assert x.tolist() == y


@pytest.mark.parametrize("children", [16, 40, 200])
@pytest.mark.parametrize("vocab,n_seqs,drafted", [(700, 4, True), (9000, 100, True), (40000, 3, True), (9000, 100, False)])
def test_roots_of_many_children(cuda, children, vocab, n_seqs, drafted):
    """Most of a root's children are rejected, so that what is left of the target is taken down again and again."""
    from asterq.speculative import verify_drafts

    if children * vocab * n_seqs > 40_000_000:
        n_seqs = max(2, 40_000_000 // (children * vocab))
    new = [children + 1] * n_seqs
    target, draft, tokens, parents, starts, accept, sample = _case(new, vocab, True, drafted, torch.float32, 5)
    parents = [[-1] + [0] * children] * n_seqs
    base = draft if drafted else target
    g = torch.Generator(device="cuda").manual_seed(6)
    roots = torch.tensor(starts[:-1], device="cuda")
    tokens = torch.multinomial(base[roots] + 1e-9, children + 1, replacement=True, generator=g).flatten().int()
    accept = 0.9 + 0.1 * accept
    want = _expected(target, draft, tokens, parents, starts, accept, sample)
    got = verify_drafts(target, tokens, _ints(starts), _ints([p for t in parents for p in t]), accept, sample, draft_probs=draft)
    for x, y in zip(got, want):
        assert x.tolist() == y
