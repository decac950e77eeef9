"""Prompts of the linear layers as the SMs share them: many chunks to a CTA, so that its buffers are used again and
again and shares begin inside sequences; calls of a single chunk's rows.  Against the recurrence in 64 bits, by the
tolerances of test_linear_attention_gpu."""
from __future__ import annotations

import math

import pytest
import torch

from test_linear_attention_gpu import _check, _inputs, _ints, _offsets

pytestmark = pytest.mark.gpu


def _run(new, h, dk, dv, decay):
    from asterq.linear_attention import linear_attention_prefill

    n = len(new)
    q, k, v, g = _inputs(sum(new), h, dk, dv, torch.bfloat16, 11, decay)
    slots, lengths = list(range(n, 0, -1)), [i % 2 for i in range(n)]
    state = torch.randn(n + 1, h, dk, dv, device="cuda")
    for slot, length in zip(slots, lengths):
        if length == 0 and new[n - slot]:
            state[slot] = math.nan  # a fresh sequence does not read its slot
    state0, offsets = state.clone(), _offsets(new)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = linear_attention_prefill(state, _ints(slots), _ints(lengths), _ints(offsets), q, k, v, g, status=status)
    assert int(status) == 0
    _check(state0, state, out, slots, lengths, offsets, q, k, v, g, dk**-0.5)


@pytest.mark.parametrize("new,h", [([2900, 1, 700, 129], 64), ([128 * 9, 128 * 9 + 1], 148)])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
def test_many_chunks_a_cta(cuda, new, h, dk, dv):
    _run(new, h, dk, dv, "token")


@pytest.mark.parametrize("new", [[128], [100], [40, 0, 60], [30, 31, 32, 33], [64, 64], [24]])
@pytest.mark.parametrize("dk,dv,h", [(128, 128, 3), (64, 64, 200), (64, 128, 2), (128, 64, 160)])
def test_rows_of_one_chunk(cuda, new, dk, dv, h):
    _run(new, h, dk, dv, "head")
