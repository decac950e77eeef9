"""The hybrid example's steps leave slots alone whose request has been released."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_released_slot_is_idle_at_once(cuda):
    path = Path(__file__).resolve().parent.parent / "examples" / "hybrid_decode.py"
    spec = importlib.util.spec_from_file_location("hybrid_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    torch.manual_seed(33)
    server = module.Server(module.Weights(cuda), cuda)

    def rows(n):
        return torch.randn(n, module.WIDTH, device=cuda).to(module.BF16)

    slots = [server.admit(rows(n))[0] for n in (30, 20)]
    server.step(rows(module.MAX_SEQS))
    server.release(slots[0])
    states = [s.clone() for s in server.states]
    x = rows(module.MAX_SEQS)
    y = server.step(x)
    for before, after in zip(states, server.states):
        assert torch.equal(before[slots[0]], after[slots[0]])
        assert not torch.equal(before[slots[1]], after[slots[1]])
    assert torch.equal(y[slots[0]], x[slots[0]])  # its row passes through, as rows of free slots do
    server.kv.raise_if_failed()
