"""Verification of drafted tokens against a plain walk in 64 bits: whole numbers, which are equal, and how often tokens come.

The frequencies' tolerance: of n draws a token of probability p comes n p times, give or take sqrt(n p (1 - p)); six of these are
passed once in 10^9 draws of a test, which its fixed seed makes once for all.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _walk(target, tokens, parents, accept, sample, draft):
    """One sequence: float64 arrays."""
    n = len(tokens)
    cur, kept, r, m, lost = 0, [0], target[0].copy(), 1.0, False
    for i in range(1, n):
        if parents[i] != cur:
            continue
        x = int(tokens[i])
        q = 1.0 if draft is None else draft[cur][x]
        if accept[i] * q * m < r[x]:
            cur, r, m, lost = i, target[i].copy(), 1.0, False
            kept.append(i)
        elif draft is None:
            m -= r[x]
            r[x] = 0.0
            lost = True
        else:
            r = np.maximum(r - m * draft[cur], 0.0)
            m = r.sum()
            if m == 0.0:
                r, m = target[cur].copy(), 1.0
    if r.sum() == 0.0 and lost:
        r = target[cur].copy()
    sums = np.cumsum(r)
    return kept, int(min(np.searchsorted(sums, sample * sums[-1], side="right"), len(r) - 1))


def _tree(n, rng):
    return [-1] + [int(rng.randint(max(0, i - 5), i)) for i in range(1, n)]


def _case(new, vocab, chain, drafted, dtype, seed, sharp=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed)
    rows = sum(new)
    logits = torch.randn(rows, vocab, device="cuda", generator=g) * sharp
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits + torch.randn(rows, vocab, device="cuda", generator=g) * 0.8, -1).to(dtype) if drafted else None
    parents = [list(range(-1, n - 1)) if chain else _tree(n, rng) for n in new]
    starts = [0] + np.cumsum(new).tolist()
    above = torch.tensor([starts[s] + max(p, 0) for s, t in enumerate(parents) for p in t], device="cuda", dtype=torch.long)
    base = draft if drafted else target
    tokens = torch.multinomial(base[above].float() + 1e-9, 1, generator=g)[:, 0].int() if rows else torch.zeros(0, dtype=torch.int32, device="cuda")
    accept = torch.rand(rows, device="cuda", generator=g)
    sample = torch.rand(len(new), device="cuda", generator=g)
    return target, draft, tokens, parents, starts, accept, sample


def _expected(target, draft, tokens, parents, starts, accept, sample):
    kept, count, nxt = [], [], []
    t, x, u, f = target.double().cpu().numpy(), tokens.cpu().numpy(), accept.double().cpu().numpy(), sample.double().cpu().numpy()
    d = None if draft is None else draft.double().cpu().numpy()
    for s, up in enumerate(parents):
        a, b = starts[s], starts[s + 1]
        if a == b:
            count.append(0)
            nxt.append(-1)
            continue
        k, token = _walk(t[a:b], x[a:b], up, u[a:b], f[s], None if d is None else d[a:b])
        kept += k + [-1] * (b - a - len(k))
        count.append(len(k))
        nxt.append(token)
    return kept, count, nxt


@pytest.mark.parametrize("new,vocab,chain,drafted,dtype", [
    ([1], 5, True, False, torch.float32),
    ([1, 2, 0, 7], 100, True, True, torch.float32),
    ([6] * 5, 1000, True, False, torch.float32),
    ([12, 1, 30, 5], 5003, False, True, torch.float32),
    ([12, 1, 30, 5], 5003, False, False, torch.float16),
    ([9, 4], 50257, False, True, torch.bfloat16),
    ([16] * 3, 128256, False, True, torch.float32),
    ([8] * 200, 2049, False, True, torch.float32),
    ([5] * 640, 300, False, False, torch.float32),
    ([1024, 700], 64, False, True, torch.float32),
    ([3] * 30, 31, False, True, torch.float32),
])
def test_walk_and_token_are_the_plain_ones(cuda, new, vocab, chain, drafted, dtype):
    from asterq.speculative import verify_drafts

    for seed in range(3):
        target, draft, tokens, parents, starts, accept, sample = _case(new, vocab, chain, drafted, dtype, seed)
        want = _expected(target, draft, tokens, parents, starts, accept, sample)
        status = _ints([0])
        up = None if chain else _ints([p for t in parents for p in t])
        got = verify_drafts(target, tokens, _ints(starts), up, accept, sample, draft_probs=draft, status=status)
        assert status.item() == 0
        for x, y in zip(got, want):
            assert x.tolist() == y


def test_rows_with_a_stride_and_unaligned(cuda):
    from asterq.speculative import verify_drafts

    target, draft, tokens, parents, starts, accept, sample = _case([6, 9], 333, False, True, torch.float32, 4)
    wide = torch.zeros(2, 15, 351, device="cuda")
    wide[0, :, 5:338], wide[1, :, 7:340] = target, draft
    up = _ints([p for t in parents for p in t])
    a = verify_drafts(target, tokens, _ints(starts), up, accept, sample, draft_probs=draft)
    b = verify_drafts(wide[0, :, 5:338], tokens, _ints(starts), up, accept, sample, draft_probs=wide[1, :, 7:340])
    c = verify_drafts(target.t().contiguous().t(), tokens, _ints(starts), up, accept, sample, draft_probs=draft)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


def test_what_is_kept_and_drawn_is_distributed_as_the_target(cuda):
    """Two drawn siblings and a next token: the first token behind the root has the target's distribution."""
    from asterq.speculative import verify_drafts

    n, vocab = 40000, 7
    g = torch.Generator(device="cuda").manual_seed(11)
    p = torch.softmax(torch.randn(vocab, device="cuda", generator=g), 0)
    q = torch.softmax(torch.randn(vocab, device="cuda", generator=g), 0)
    target, draft = p.expand(3 * n, vocab), q.expand(3 * n, vocab)
    tokens = torch.multinomial(q.expand(3 * n, vocab), 1, generator=g)[:, 0].int()
    starts, up = _ints(list(range(0, 3 * n + 1, 3))), _ints([-1, 0, 0] * n)
    accept, sample = (torch.rand(k, device="cuda", generator=g) for k in (3 * n, n))
    for probs in (draft, None):
        drafted = tokens
        if probs is None:  # drafts that were not drawn: always the same two
            drafted = _ints([0, 2, 5] * n)
        kept, count, nxt = verify_drafts(target, drafted, starts, up, accept, sample, draft_probs=probs)
        kept = kept.view(n, 3).long()
        first = torch.where(count > 1, drafted.view(n, 3).gather(1, kept[:, 1:2].clamp(min=0))[:, 0], nxt)
        freq = torch.bincount(first.long(), minlength=vocab).double()
        want = n * p.double()
        assert ((freq - want).abs() <= 6 * (want * (1 - p.double())).sqrt()).all()


def test_certain_and_impossible_tokens(cuda):
    from asterq.speculative import verify_drafts

    one = torch.zeros(4, 50, device="cuda")
    one[:, 7] = 1.0
    starts = _ints([0, 4])
    high = torch.full((4,), 1 - 2.0**-24, device="cuda")
    last = torch.full((1,), 1 - 2.0**-24, device="cuda")
    kept, count, nxt = verify_drafts(one, _ints([0, 7, 7, 7]), starts, None, high, last)
    assert kept.tolist() == [0, 1, 2, 3] and count.tolist() == [4] and nxt.tolist() == [7]
    kept, count, nxt = verify_drafts(one, _ints([0, 8, 7, 7]), starts, None, torch.zeros(4, device="cuda"), last)
    assert kept.tolist() == [0, -1, -1, -1] and count.tolist() == [1] and nxt.tolist() == [7]
    # the draft is the target itself: all is kept, and a rejection of the only token leaves the target
    kept, count, nxt = verify_drafts(one, _ints([0, 7, 7, 8]), starts, None, high, last, draft_probs=one)
    assert kept.tolist() == [0, 1, 2, -1] and nxt.tolist() == [7]
    # the same token twice among siblings: the second cannot be taken once the first is gone
    two = torch.full((3, 2), 0.5, device="cuda")
    kept, count, nxt = verify_drafts(two, _ints([0, 1, 1]), _ints([0, 3]), _ints([-1, 0, 0]),
                                     torch.tensor([0.0, 0.75, 0.0], device="cuda"), torch.zeros(1, device="cuda"))
    assert kept.tolist() == [0, -1, -1] and nxt.tolist() == [0]


def test_inputs_that_are_wrong_are_reported(cuda):
    from asterq.speculative import verify_drafts

    p = torch.full((4, 8), 1 / 8, device="cuda")
    zero, half = torch.zeros(4, device="cuda"), torch.full((1,), 0.5, device="cuda")

    def run(tokens, starts, up, target=p, sample=half):
        status = _ints([0])
        kept, count, nxt = verify_drafts(target, _ints(tokens), _ints(starts), up, zero, sample, status=status)
        return kept.tolist(), count.tolist(), nxt.tolist(), status.item()

    assert run([0, 1, 2, 3], [0, 4], None) == ([0, 1, 2, 3], [4], [4], 0)
    assert run([9, 1, 2, 3], [0, 4], None) == ([0, 1, 2, 3], [4], [4], 0)  # the root's token is not looked at
    assert run([0, 1, 8, 3], [0, 4], None) == ([0, 1, -1, -1], [2], [4], 1)
    assert run([0, -1, 2, 3], [0, 4], None) == ([0, -1, -1, -1], [1], [4], 1)
    assert run([0, 1, 2, 3], [0, 4], _ints([-1, 0, 2, 2])) == ([0, 1, -1, -1], [2], [4], 1)
    assert run([0, 1, 2, 3], [0, 4], _ints([-1, -1, 0, 2])) == ([0, 2, 3, -1], [3], [4], 0)  # another root is not reached
    assert run([0, 1, 2, 3], [0, 4], _ints([0, 0, 0, 2]))[3] == 1
    assert run([0, 1, 2, 3], [0, 5], None)[1:] == ([0], [-1], 1)
    assert run([0, 1, 2, 3], [2, 0], None)[1:] == ([0], [-1], 1)
    none = p.clone()
    none[3] = 0.0
    assert run([0, 1, 2, 3], [0, 4], None, none)[1:] == ([4], [-1], 1)
    none[3] = math.nan
    assert run([0, 1, 2, 3], [0, 4], None, none)[1:] == ([4], [-1], 1)
    for u in (1.0, 7.0, math.nan, math.inf):
        assert run([0, 1, 2, 3], [0, 4], None, sample=torch.full((1,), u, device="cuda"))[2] == [7]
    assert run([0, 1, 2, 3], [0, 4], None, sample=torch.full((1,), -1.0, device="cuda"))[2] == [0]


def test_rows_of_no_sequence_are_not_written(cuda):
    from asterq import _lib
    from asterq.speculative import _PARAMS

    p = torch.full((6, 8), 1 / 8, device="cuda")
    kept = torch.full((6,), 77, dtype=torch.int32, device="cuda")
    out = torch.full((2,), 77, dtype=torch.int32, device="cuda")
    tokens, starts, u = _ints([0, 1, 2, 3, 4, 5]), _ints([1, 4]), torch.zeros(6, device="cuda")
    _lib.check(_lib.load().asterq_verify_drafts(
        _PARAMS.pack(_lib.DTYPE_F32, 1, 8, 0, 6, 8, 0, p.data_ptr(), 0, tokens.data_ptr(), 0, starts.data_ptr(), u.data_ptr(),
                     u.data_ptr(), kept.data_ptr(), out.data_ptr(), out.data_ptr() + 4, 0), _lib.stream_handle()))
    assert kept.tolist() == [77, 0, 1, 2, 77, 77] and out.tolist() == [3, 0]


def test_refusals(cuda):
    from asterq.speculative import verify_drafts

    p, x, s = torch.full((4, 8), 1 / 8, device="cuda"), _ints([0, 1, 2, 3]), _ints([0, 4])
    u, v = torch.zeros(4, device="cuda"), torch.zeros(1, device="cuda")
    for exc, args, kw in (
            (ValueError, (p[0], x, s, None, u, v), {}), (TypeError, (p.double(), x, s, None, u, v), {}),
            (RuntimeError, (p.cpu(), x, s, None, u, v), {}), (ValueError, (p[:, :0], x, s, None, u, v), {}),
            (ValueError, (p, x.long(), s, None, u, v), {}), (ValueError, (p, x[:3], s, None, u, v), {}),
            (ValueError, (p, x, s, x[:3], u, v), {}), (ValueError, (p, x, s, None, u[:3], v), {}),
            (ValueError, (p, x, s, None, u, u), {}), (ValueError, (p, x, s, None, u.double(), v), {}),
            (TypeError, (p, x, s, None, u, v), dict(draft_probs=p.half())),
            (ValueError, (p, x, s, None, u, v), dict(draft_probs=p[:3])),
            (RuntimeError, (p.clone().requires_grad_(), x, s, None, u, v), {})):
        with pytest.raises(exc):
            verify_drafts(*args, **kw)
