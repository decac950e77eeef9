"""Prompts of the linear layers at their edges: values that are not finite must stay in their column and out of
the rows before them; inputs and outputs that the chunked form cannot address take the other one."""
from __future__ import annotations

import pytest
import torch

from asterq import linear_attention as la

pytestmark = pytest.mark.gpu


def _inputs(lengths, heads, dk, dv, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(lengths)
    q, k, v = (torch.randn((total, heads, d), device="cuda", generator=gen).bfloat16() for d in (dk, dk, dv))
    decay = -torch.rand((total, heads), device="cuda", generator=gen) * 0.2
    state = torch.randn((len(lengths), heads, dk, dv), device="cuda", generator=gen)
    offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return q, k, v, decay, state, offsets


def _run(q, k, v, decay, state, offsets, **kw):
    state = state.clone()
    slots = torch.arange(state.shape[0], dtype=torch.int32, device="cuda")
    return la.linear_attention_prefill(state, slots, None, offsets, q, k, v, decay, **kw), state


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("lengths,heads,at", [
    ([100], 2, 0), ([100], 2, 63), ([100], 2, 99), ([40, 128, 130], 3, 41), ([40, 128, 130], 3, 39),
    ([2000, 77], 2, 1000), ([2000, 77], 2, 127), ([600, 600], 60, 700)])
def test_values_that_are_not_finite_stay_in_their_column(lengths, heads, at, dk, dv, value):
    q, k, v, decay, state, offsets = _inputs(lengths, heads, dk, dv)
    want, end = _run(q, k, v, decay, state, offsets)
    head, dim = heads - 1, dv - 3
    v[at, head, dim] = value
    got, got_end = _run(q, k, v, decay, state, offsets)
    seq = next(s for s in range(len(lengths)) if offsets[s + 1] > at)
    rows = slice(at, int(offsets[seq + 1]))
    assert not got[rows, head, dim].isfinite().any()
    assert not got_end[seq, head, :, dim].isfinite().any()
    # everything else is what it was, to the bit: the rows before, other columns, heads and sequences
    got[rows, head, dim] = want[rows, head, dim]
    got_end[seq, head, :, dim] = end[seq, head, :, dim]
    assert torch.equal(got, want) and torch.equal(got_end, end)


def test_many_values_that_are_not_finite():
    q, k, v, decay, state, offsets = _inputs([700, 300], 4, 128, 128)
    want, end = _run(q, k, v, decay, state, offsets)
    gen = torch.Generator(device="cuda").manual_seed(1)
    bad = torch.rand(v.shape, device="cuda", generator=gen) < 0.002
    v[bad] = float("nan")
    got, got_end = _run(q, k, v, decay, state, offsets)
    for begin, end_row, s in ((0, 700, 0), (700, 1000, 1)):
        reached = bad[begin:end_row].int().cumsum(0) > 0
        assert torch.equal(got[begin:end_row].isnan(), reached)
        assert torch.equal(got[begin:end_row][~reached], want[begin:end_row][~reached])
        column = bad[begin:end_row].any(0)[:, None, :].expand(4, 128, 128)
        assert torch.equal(got_end[s].isnan(), column)
        assert torch.equal(got_end[s][~column], end[s][~column])


@pytest.mark.parametrize("what", ["out", "state", "repeated values", "keys in reverse"])
def test_inputs_that_the_chunked_form_cannot_address(what):
    """The same numbers through the other form: 3 2^-9 of the largest output for three bf16 roundings (an output's
    own on each side, and one between two neighbours), 1e-5 of the largest state for a few hundred fp32 sums."""
    q, k, v, decay, state, offsets = _inputs([300, 41], 2, 64, 64)
    kw = {}
    if what == "repeated values":
        v = v[:, :1].expand(-1, 2, -1)
        q, k = q.contiguous(), k.contiguous()
        want, end = _run(q, k, v.contiguous(), decay, state, offsets)
    else:
        want, end = _run(q, k, v, decay, state, offsets)
    if what == "out":
        kw["out"] = torch.empty(q.numel() + 8, dtype=q.dtype, device="cuda")[8:].view(want.shape)
    if what == "state":
        room = torch.empty(state.numel() + 4, device="cuda")[4:].view(state.shape)
        room.copy_(state)
        slots = torch.arange(2, dtype=torch.int32, device="cuda")
        got, got_end = la.linear_attention_prefill(room, slots, None, offsets, q, k, v, decay), room
    elif what == "keys in reverse":
        # heads held in another order: every head's dims are contiguous, the heads lie across the rows
        k = k.transpose(0, 1).contiguous().transpose(0, 1)
        got, got_end = _run(q, k, v, decay, state, offsets)
    else:
        got, got_end = _run(q, k, v, decay, state, offsets, **kw)
    assert (got.float() - want.float()).abs().max() <= 3 * 2.0**-9 * want.float().abs().max()
    assert (got_end - end).abs().max() <= 1e-5 * end.abs().max()
