"""Calls captured in CUDA graphs on streams that have made no call before (torch.cuda.graph captures on one of its own):
each graph is complete by itself, whatever is replayed first."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("stream", [None, "new"])
def test_graphs_of_attention_replay_in_any_order(cuda, stream):
    from asterq import paged_kv
    from asterq.paged_kv import PagedKVPools, paged_attention

    torch.manual_seed(30)
    pools = PagedKVPools(*[torch.randn(160, 2, 64, 128, device="cuda").bfloat16() for _ in range(2)])
    table, lengths = torch.randperm(160).int().cuda()[None], _ints([160 * 64 - 5])  # one sequence over all SMs
    q = [torch.randn(1, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [paged_attention(pools, table, lengths, x) for x in q]
    known = set(paged_kv._workspaces)
    kw = {} if stream is None else dict(stream=torch.cuda.Stream())
    graphs, got = [torch.cuda.CUDAGraph() for _ in q], []
    for graph, x in zip(graphs, q):
        with torch.cuda.graph(graph, **kw):
            got.append([paged_attention(pools, table, lengths, x) for _ in range(3)])
    # what a capture has left behind for later calls has not run yet: its memory holds anything
    for key in set(paged_kv._workspaces) - known:
        paged_kv._workspaces[key].buffer.fill_(0x55)
    for order in ((1, 0), (1, 1, 0, 0, 1)):
        for i in order:
            for x in got[i]:
                x.fill_(float("nan"))
            graphs[i].replay()
            torch.cuda.synchronize()
            for x in got[i]:
                assert torch.equal(x, want[i])
    # nor do calls on the stream itself find it
    if stream is not None:
        with torch.cuda.stream(kw["stream"]):
            x = paged_attention(pools, table, lengths, q[0])
        torch.cuda.synchronize()
        assert torch.equal(x, want[0])


def test_graphs_of_prompts_replay_in_any_order(cuda):
    from asterq import linear_attention
    from asterq.linear_attention import linear_attention_prefill

    torch.manual_seed(31)
    q, k, v = (torch.randn(1500, 4, 128, device="cuda").bfloat16() for _ in range(3))
    decay, state0 = torch.full((4,), -0.05, device="cuda"), torch.randn(1, 4, 128, 128, device="cuda")
    slots, offsets = _ints([0]), _ints([0, 1500])
    state = state0.clone()
    want = linear_attention_prefill(state, slots, None, offsets, q, k, v, decay)
    known = set(linear_attention._workspaces)
    graphs, got, states = [torch.cuda.CUDAGraph() for _ in range(2)], [], [state0.clone() for _ in range(2)]
    for graph, s in zip(graphs, states):
        with torch.cuda.graph(graph):
            got.append(linear_attention_prefill(s, slots, None, offsets, q, k, v, decay))
    assert set(linear_attention._workspaces) == known  # a graph's memory is not kept for calls outside of it
    for i in (1, 0, 0, 1):
        states[i].copy_(state0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(got[i], want) and torch.equal(states[i], state)
