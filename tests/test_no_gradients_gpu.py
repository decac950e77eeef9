"""The paged and linear layers' calls have no backward pass: inputs that would need one are refused, both ways."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quick", [True, False])
def test_inputs_that_require_a_gradient_are_refused(cuda, monkeypatch, quick):
    from asterq import paged_kv
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step
    from asterq.paged_kv import PagedKVPools, append_kv, paged_attention

    if not quick:
        monkeypatch.setattr(paged_kv, "_quick_module", None)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    x = torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    y = x.clone().requires_grad_()
    pools = PagedKVPools.empty(4, 2, 16, 64)
    table, lengths, offsets = ints([[0], [1]]), ints([0, 0]), ints([0, 1, 2])
    state, decay = torch.zeros(2, 2, 64, 64, device="cuda"), torch.zeros(2, device="cuda")
    calls = [lambda t, d, s: append_kv(pools, table, lengths, offsets, t, x, q=x),
             lambda t, d, s: append_kv(pools, table, lengths, offsets, x, t, q=x),
             lambda t, d, s: append_kv(pools, table, lengths, offsets, x, x, q=t),
             lambda t, d, s: paged_attention(pools, table, lengths, t, n_new=1),
             lambda t, d, s: linear_attention_step(state, lengths, t, x, x, decay),
             lambda t, d, s: linear_attention_step(state, lengths, x, t, x, decay),
             lambda t, d, s: linear_attention_step(state, lengths, x, x, t, decay),
             lambda t, d, s: linear_attention_step(state, lengths, x, x, x, d),
             lambda t, d, s: linear_attention_step(s, lengths, x, x, x, decay),
             lambda t, d, s: linear_attention_prefill(state, lengths[:1], None, ints([0, 2]), t, x, x, decay)]
    for call in calls:
        args = x, decay, state
        wanting = y, decay.clone().requires_grad_(), state.clone().requires_grad_()
        call(*args)
        with pytest.raises(RuntimeError, match="gradient"):
            call(*wanting)
        with torch.no_grad():  # a model's parameters at inference
            call(*wanting)
        call(*(t.detach() for t in wanting))
