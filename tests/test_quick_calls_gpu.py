"""The quick way into the library (asterq._calls) and the checks in Python make the same calls."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["quick", "python"])
def way(request, monkeypatch, cuda):
    from asterq import _lib, paged_kv

    assert _lib.quick_calls() is not None, "asterq._calls is not built"
    if not request.param:
        monkeypatch.setattr(paged_kv, "_quick_module", None)
    return request.param


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _everything():
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step
    from asterq.paged_kv import PagedKVPools, append_kv, paged_attention

    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    pools = PagedKVPools(randn(9, 2, 32, 64), randn(9, 2, 32, 64))
    table = _ints([[3, 1, 7], [0, 8, 2]])
    x = randn(5, 12, 64)
    cos, sin = torch.rand(96, 32, device="cuda", generator=g), torch.rand(96, 32, device="cuda", generator=g)
    status = _ints([0])
    got = [append_kv(pools, table, _ints([30, 60]), _ints([0, 3, 5]), x[:, 8:10], x[:, 10:], q=x[:, :8], cos=cos, sin=sin,
                     interleaved=True, status=status)]
    assert append_kv(pools, table, _ints([33, 62]), _ints([0, 1, 2]), x[:2, 8:10], x[:2, 10:]) is None
    got += [pools.k.clone(), pools.v.clone()]
    got += paged_attention(pools, table, _ints([33, 62]), got[0][:2], return_lse=True, n_new=1)
    out = torch.empty(2, 8, 64, device="cuda")
    assert paged_attention(pools, table, _ints([33, -1]), x[:2, :8], out=out, window_size=20, sink_tokens=3,
                           softmax_scale=0.2, logit_softcap=5.0, status=status) is out
    got.append(out)
    state = torch.randn(4, 3, 64, 128, device="cuda", generator=g)
    q, k, v, d = randn(200, 3, 64), randn(200, 3, 64), randn(200, 3, 128), -torch.rand(200, 3, device="cuda", generator=g)
    got.append(linear_attention_prefill(state, _ints([2, 0]), _ints([0, 4]), _ints([0, 150, 200]), q, k, v, d, status=status))
    got.append(state.clone())
    out = torch.empty(3, 3, 128, dtype=torch.bfloat16, device="cuda")
    assert linear_attention_step(state, _ints([1, -1, 3]), q[:3], k[:3], v[:3], d[0], out=out, scale=0.5) is out
    assert int(status) == 0
    return got + [out, state]


_seen = []


def test_both_ways_give_the_same_bits(way):
    _seen.append([t.cpu() for t in _everything()])
    for x, y in zip(_seen[0], _seen[-1], strict=True):
        assert torch.equal(x, y)


def test_refusals_are_the_same(way):
    from asterq import _lib
    from asterq.linear_attention import linear_attention_step
    from asterq.paged_kv import PagedKVPools, append_kv, paged_attention

    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    pools = PagedKVPools(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda"),
                         torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda"))
    table, lengths = _ints([[0], [1]]), _ints([0, 0])
    for error, call in [
        (TypeError, lambda: append_kv(pools, table, lengths, _ints([0, 1, 2]), x, x.half())),
        (ValueError, lambda: append_kv(pools, table, lengths, _ints([0, 1]), x, x)),
        (ValueError, lambda: append_kv(pools, table, lengths, _ints([0, 1, 2]), x, x, q_out=x)),
        (ValueError, lambda: paged_attention(pools, table, lengths, x[:, :1])),
        (ValueError, lambda: paged_attention(pools, table, lengths, x, window_size=0)),
        (ValueError, lambda: paged_attention(pools, table.long(), lengths, x)),
        (ValueError, lambda: paged_attention(pools, table, lengths, x, out=x[:1])),
        (_lib.AsterqError, lambda: paged_attention(pools, table, lengths, x, out=x.half())),
        (ValueError, lambda: linear_attention_step(torch.zeros(2, 2, 64, 64, device="cuda"), lengths[:1], x, x, x,
                                                   torch.zeros(2, device="cuda"))),
        (TypeError, lambda: linear_attention_step(torch.zeros(2, 2, 64, 64, device="cuda"), lengths, x, x.half(), x,
                                                  torch.zeros(2, device="cuda"))),
        (ValueError, lambda: PagedKVPools(pools.k, pools.v[:2])),
        (RuntimeError, lambda: PagedKVPools(pools.k.cpu(), pools.v.cpu())),
    ]:
        with pytest.raises(error):
            call()
