"""Keys, queries and states of the linear layers that are not finite: they reach what the recurrence lets them reach, and
leave everything else to the bit (values are in test_linear_edges_gpu)."""
from __future__ import annotations

import pytest
import torch

from test_linear_edges_gpu import _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("lengths,heads,at", [([100], 2, 63), ([40, 128, 130], 3, 41), ([2000, 77], 2, 1000), ([600, 600], 60, 700)])
def test_keys_that_are_not_finite_reach_their_row_of_the_state(lengths, heads, at, dk, dv, value):
    q, k, v, decay, state, offsets = _inputs(lengths, heads, dk, dv)
    want, end = _run(q, k, v, decay, state, offsets)
    head, dim = heads - 1, dk - 5
    k[at, head, dim] = value
    got, got_end = _run(q, k, v, decay, state, offsets)
    seq = next(s for s in range(len(lengths)) if offsets[s + 1] > at)
    rows = slice(at, int(offsets[seq + 1]))
    assert not got[rows, head].isfinite().any() and not got_end[seq, head, dim].isfinite().any()
    got[rows, head], got_end[seq, head, dim] = want[rows, head], end[seq, head, dim]
    assert torch.equal(got, want) and torch.equal(got_end, end)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_queries_that_are_not_finite_reach_their_row(value):
    q, k, v, decay, state, offsets = _inputs([300, 129], 2, 128, 128)
    want, end = _run(q, k, v, decay, state, offsets)
    for at in (0, 127, 128, 299, 301, 428):
        q[at, 1, 7] = value
    got, got_end = _run(q, k, v, decay, state, offsets)
    for at in (0, 127, 128, 299, 301, 428):
        assert not got[at, 1].isfinite().any()
        got[at, 1] = want[at, 1]
    assert torch.equal(got, want) and torch.equal(got_end, end)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_states_that_are_not_finite_reach_their_column(value):
    q, k, v, decay, state, offsets = _inputs([1500, 129], 2, 64, 128)
    want, end = _run(q, k, v, decay, state, offsets)
    state[0, 1, 9, 33] = value
    got, got_end = _run(q, k, v, decay, state, offsets)
    assert not got[:1500, 1, 33].isfinite().any() and not got_end[0, 1, 9, 33].isfinite().any()
    got[:1500, 1, 33], got_end[0, 1, 9, 33] = want[:1500, 1, 33], end[0, 1, 9, 33]
    assert torch.equal(got, want) and torch.equal(got_end, end)
