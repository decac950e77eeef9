"""Prompts of the linear layers whose last chunks end on whole steps of 16 tokens: the keys past their ends are cleared in
a tile that the next chunk's keys are loaded over, many times a CTA.  Against the recurrence in 64 bits, by the
tolerances of test_linear_attention_gpu, and to the bit over repetitions."""
from __future__ import annotations

import pytest
import torch

from test_linear_attention_gpu import _check, _inputs, _ints, _offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,h", [([64, 80, 16, 112] * 4, 96), ([192, 32, 320] * 3, 64), ([48] * 40, 48)])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
def test_tiles_with_cleared_keys_are_filled_again(cuda, new, h, dk, dv):
    from asterq.linear_attention import linear_attention_prefill

    n = len(new)
    q, k, v, g = _inputs(sum(new), h, dk, dv, torch.bfloat16, 12)
    slots, lengths, offsets = list(range(n)), [1] * n, _offsets(new)
    state0 = torch.randn(n, h, dk, dv, device="cuda")
    first = None
    for _ in range(6):
        state = state0.clone()
        out = linear_attention_prefill(state, _ints(slots), _ints(lengths), _ints(offsets), q, k, v, g)
        if first is None:
            first = out, state
        assert torch.equal(first[0], out) and torch.equal(first[1], state)
    _check(state0, first[1], first[0], slots, lengths, offsets, q, k, v, g, dk**-0.5)
