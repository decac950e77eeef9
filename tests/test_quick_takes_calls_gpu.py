"""The quick way into the library (asterq._calls) takes the calls that a decode step makes, and answers as the checks in
Python do."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _calls():
    """name -> a call through the public entry points and what it has written."""
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step
    from asterq.paged_kv import PagedKVPools, append_kv, paged_attention

    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    pools = PagedKVPools(randn(9, 2, 32, 64), randn(9, 2, 32, 64))
    table, lengths, x = _ints([[3, 1, 7], [0, 8, 2]]), _ints([33, 62]), randn(2, 12, 64)
    cos, sin = torch.rand(96, 32, device="cuda", generator=g), torch.rand(96, 32, device="cuda", generator=g)
    state = torch.randn(4, 3, 64, 128, device="cuda", generator=g)
    q, k, v, d = randn(200, 3, 64), randn(200, 3, 64), randn(200, 3, 128), -torch.rand(200, 3, device="cuda", generator=g)

    def append():
        return append_kv(pools, table, lengths, _ints([0, 1, 2]), x[:, 8:10], x[:, 10:], q=x[:, :8], cos=cos, sin=sin), \
            pools.k.clone(), pools.v.clone()

    def prefill():
        s = state.clone()
        return linear_attention_prefill(s, _ints([2, 0]), _ints([0, 4]), _ints([0, 150, 200]), q, k, v, d), s

    def step():
        s = state.clone()
        return linear_attention_step(s, _ints([1, -1, 3]), q[:3], k[:3], v[:3], d[:3]), s

    return {"append": append, "attend": lambda: paged_attention(pools, table, lengths, x[:, :8], n_new=1, return_lse=True),
            "linear": prefill, "linear of one token": step}


@pytest.mark.parametrize("name", ["append", "attend", "linear", "linear of one token"])
@pytest.mark.parametrize("first", ["quick", "python"])
def test_the_quick_way_takes_the_call(cuda, monkeypatch, name, first):
    """Also on a stream whose workspace was made while calls went the other way."""
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

    call, stream = _calls()[name], torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        monkeypatch.setattr(paged_kv, "_quick_module", Watched() if first == "quick" else None)
        call()  # makes the stream's workspace
        monkeypatch.setattr(paged_kv, "_quick_module", Watched())
        call()  # finds it
        answers.clear()
        got = call()
        assert answers == [True]
        monkeypatch.setattr(paged_kv, "_quick_module", None)
        want = call()
        assert answers == [True]
    torch.cuda.synchronize()
    for x, y in zip(got, want, strict=True):
        assert torch.equal(x, y)
