"""The quick way into the library (asterq._calls) takes the calls of prompts and drafted tokens, and gives the bits and the
refusals of the checks in Python."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _calls():
    """name -> a call through the public entry points; what it answers and writes."""
    from asterq.paged_kv import (PagedKVPools, PagedKVStack, append_kv, keep_kv_rows, paged_prompt_attention,
                                 paged_tree_attention)
    from asterq.speculative import verify_drafts

    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    pools = PagedKVPools(randn(9, 2, 32, 64), randn(9, 2, 32, 64))
    stack = PagedKVStack([pools, PagedKVPools(randn(9, 2, 32, 64), randn(9, 2, 32, 64))])
    table, lengths, offsets, x = _ints([[3, 1, 7], [0, 8, 2]]), _ints([33, 62]), _ints([0, 3, 7]), randn(7, 12, 64)
    parents = _ints([-1, 0, 0, -1, 0, 1, 1])
    cos, sin = torch.rand(96, 32, device="cuda", generator=g), torch.rand(96, 32, device="cuda", generator=g)
    q_norm, k_norm = randn(64, dtype=torch.float32), randn(64, dtype=torch.float32)
    probs = torch.softmax(torch.randn(7, 301, device="cuda", generator=g), 1)
    drafts = torch.softmax(torch.randn(7, 301, device="cuda", generator=g), 1)
    tokens = torch.randint(0, 301, (7,), device="cuda", generator=g, dtype=torch.int32)
    u, w = torch.rand(7, device="cuda", generator=g), torch.rand(2, device="cuda", generator=g)

    def append(**kw):
        given = {"q": x[:, :8], "cos": cos, "sin": sin, "q_norm": q_norm, "k_norm": k_norm, "norm_eps": 1e-5,
                 "positions": _ints([33, 34, 34, 62, 63, 64, 64])} | kw
        return append_kv(pools, table, lengths, offsets, x[:, 8:10], x[:, 10:], **given), pools.k.clone(), pools.v.clone()

    def prompt(**kw):
        return paged_prompt_attention(pools, table, lengths, offsets, x[:, :8], **({"return_lse": True} | kw))

    def tree(**kw):
        out = torch.empty(7, 8, 64, device="cuda")
        assert paged_tree_attention(pools, table, lengths, offsets, parents, x[:, :8],
                                    **({"out": out, "window_size": 20, "sink_tokens": 3, "softmax_scale": 0.2,
                                        "logit_softcap": 5.0} | kw)) is kw.get("out", out)
        return (out,)

    def keep(**kw):
        keep_kv_rows(stack, table, lengths, offsets, _ints([0, 2, -1, 0, 1, 3, -1]), _ints([2, 3]), **kw)
        return [t.clone() for p in stack.layers for t in (p.k, p.v)]

    def verify(**kw):
        return verify_drafts(probs, tokens, offsets, parents, u, w, **({"draft_probs": drafts} | kw))

    return {"append": append, "rows of prompts": prompt, "rows of trees": tree, "keep": keep, "verify": verify}


@pytest.mark.parametrize("name", ["append", "rows of prompts", "rows of trees", "keep", "verify"])
def test_the_quick_way_takes_the_call(cuda, monkeypatch, name):
    from asterq import _lib, paged_kv

    module = _lib.quick_calls()
    assert module is not None, "asterq._calls is not built"
    answers = []

    class Watched:
        def __getattr__(self, attribute):
            def call(*args):
                answer = getattr(module, attribute)(*args)
                if attribute == name.split()[0]:
                    answers.append(answer is not NotImplemented)
                return answer
            return call

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        monkeypatch.setattr(paged_kv, "_quick_module", Watched())
        call = _calls()[name]
        status = _ints([0])
        call(status=status)  # makes the stream's workspace
        call = _calls()[name]  # the pools anew
        answers.clear()
        got = call(status=status)
        assert answers == [True]
        monkeypatch.setattr(paged_kv, "_quick_module", None)
        want = _calls()[name]()
    torch.cuda.synchronize()
    assert int(status) == 0
    for x, y in zip(got, want, strict=True):
        assert torch.equal(x, y)


@pytest.mark.parametrize("quick", [True, False])
def test_refusals_are_the_same(cuda, monkeypatch, quick):
    from asterq import _lib, paged_kv
    from asterq.speculative import verify_drafts

    calls = _calls()
    for name in calls:
        calls[name]()  # the workspaces are there
    if not quick:
        monkeypatch.setattr(paged_kv, "_quick_module", None)
    half = torch.ones(64, dtype=torch.float16, device="cuda")
    for error, name, kw in [
        (TypeError, "append", {"q_norm": half, "k_norm": None}),
        (TypeError, "append", {"q_norm": half.bfloat16()}),
        (ValueError, "append", {"k_norm": half[:32]}),
        (ValueError, "append", {"norm_eps": -1.0}),
        (ValueError, "append", {"cos": None, "sin": None}),
        (ValueError, "append", {"positions": _ints([0] * 6)}),
        (ValueError, "append", {"q": None}),
        (RuntimeError, "append", {"q_norm": torch.ones(64, device="cuda", requires_grad=True)}),
        (ValueError, "rows of prompts", {"window_size": 0}),
        (ValueError, "rows of prompts", {"window_size": -3}),
        (ValueError, "rows of trees", {"sink_tokens": -1}),
        (_lib.AsterqError, "rows of trees", {"out": torch.empty(7, 8, 64, dtype=torch.float16, device="cuda")}),
        (ValueError, "rows of trees", {"status": _ints([0, 0])}),
        (ValueError, "keep", {"status": _ints([0]).long()}),
        (TypeError, "verify", {"draft_probs": torch.ones(7, 301, dtype=torch.float16, device="cuda")}),
        (ValueError, "verify", {"draft_probs": torch.ones(6, 301, device="cuda")}),
        (RuntimeError, "verify", {"draft_probs": torch.ones(7, 301, device="cuda", requires_grad=True)}),
    ]:
        with pytest.raises(error):
            calls[name](**kw)
    with pytest.raises(RuntimeError):
        verify_drafts(torch.ones(1, 8), _ints([0]), _ints([0, 1]), None, torch.zeros(1), torch.zeros(1))


def test_a_graphs_rows_have_a_workspace_of_their_own(cuda):
    """Two graphs captured on the stream of eager calls, then run beside each other: one workspace would be shared."""
    from asterq import paged_kv
    from asterq.paged_kv import PagedKVPools, paged_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(1)
    pools = PagedKVPools(*(torch.randn(160, 1, 128, 128, device="cuda", generator=g).bfloat16() for _ in range(2)))
    table = torch.randperm(160, device="cuda", generator=g).int().view(1, 160)
    lengths, offsets = _ints([20000]), _ints([0, 8])
    qs = [torch.randn(8, 4, 128, device="cuda", generator=g).bfloat16() for _ in range(2)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = [paged_prompt_attention(pools, table, lengths, offsets, q) for q in qs]
    torch.cuda.synchronize()
    before = dict(paged_kv._rows_workspaces)
    graphs, got = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got.append(paged_prompt_attention(pools, table, lengths, offsets, q))
        graphs.append(graph)
    assert paged_kv._rows_workspaces == before
    side = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        for graph, s in zip(graphs, side):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
