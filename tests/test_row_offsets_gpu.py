"""Row offsets that are out of order: calls stay inside their buffers and say so."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("offsets", [[0, 6, 3, 8], [0, 8, 0, 8], [0, 7, 1, 2, 8], [3, 1, 8], [0] + [8, 0] * 40 + [8]])
def test_append_leaves_out_rows_that_offsets_out_of_order_hide(cuda, offsets):
    """Every row is either where one of the sequences that hold it puts it, or left out with its query."""
    from asterq.paged_kv import PagedKVPools, append_kv

    n, rows, page = len(offsets) - 1, 8, 16
    # a guard page on each side of the sequences' own, one page each
    pools = PagedKVPools(*[torch.full((n + 2, 1, page, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)])
    table = _ints([[s + 1] for s in range(n)])
    lengths = [s % 3 for s in range(n)]
    x = torch.randn(rows, 3, 64, device="cuda").bfloat16()
    cos, sin = torch.ones(16, 32, device="cuda"), torch.zeros(16, 32, device="cuda")
    q_out, status = torch.full((rows, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda"), _ints([0])
    append_kv(pools, table, _ints(lengths), _ints(offsets), x[:, :1], x[:, 1:2], q=x[:, 2:], cos=cos, sin=sin, q_out=q_out,
              status=status)
    want = torch.full_like(pools.k, 7.0)
    hidden = 0
    for row in range(rows):
        if bool((q_out[row] == 7.0).all()):
            hidden += offsets[0] <= row < offsets[-1]
            continue
        assert torch.equal(q_out[row, 0], x[row, 2])
        places = [(s + 1, lengths[s] + row - offsets[s]) for s in range(n) if offsets[s] <= row < offsets[s + 1]]
        found = [(pg, at) for pg, at in places if torch.equal(pools.k[pg, 0, at], x[row, 0])]
        assert len(found) == 1 and torch.equal(pools.v[found[0][0], 0, found[0][1]], x[row, 1])
        want[found[0][0], 0, found[0][1]] = x[row, 0]
    assert int(status) == (hidden > 0)
    assert torch.equal(pools.k, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offsets", [[0, 300, 100, 300], [0, 300, 0, 300, 0, 300], [200, 100], [0, 1, 0, 299, 300]])
def test_prompts_say_that_offsets_are_out_of_order(cuda, dtype, offsets):
    """Both forms (bf16 in chunks, f16 token by token) report it; slots of no sequence keep their states, and calls that
    follow are right."""
    from asterq.linear_attention import linear_attention_prefill

    n, h = len(offsets) - 1, 2
    q, k, v = (torch.randn(300, h, 64, device="cuda").to(dtype) for _ in range(3))
    decay = torch.full((h,), -0.1, device="cuda")
    state = torch.randn(n + 1, h, 64, 64, device="cuda")
    last, status = state[n].clone(), _ints([0])
    linear_attention_prefill(state, _ints(list(range(n))), None, _ints(offsets), q, k, v, decay, status=status)
    assert int(status) == 1 and torch.equal(state[n], last)
    if dtype == torch.bfloat16:
        fresh = [torch.zeros(1, h, 64, 64, device="cuda") for _ in range(2)]
        out = [linear_attention_prefill(s, _ints([0]), None, _ints([0, 300]), q, k, v, decay) for s in fresh]
        assert torch.equal(*out) and torch.equal(*fresh) and bool(out[0].isfinite().all())


def test_chunks_of_sequences_that_share_rows_would_not_fit_32_bits(cuda):
    """Every other sequence holds all rows: 20833 times 7813 chunks of 16 heads would count up to 2.6e9."""
    from asterq.linear_attention import linear_attention_prefill

    rows, h = 1000000, 16
    n = 2 * (rows // 48) - 1
    offsets = torch.tensor([0, rows], dtype=torch.int32).repeat((n + 1) // 2).cuda()
    x = torch.zeros(rows, h, 64, dtype=torch.bfloat16, device="cuda")
    state = torch.ones(n, h, 64, 64, device="cuda")
    status = _ints([0])
    out = torch.zeros_like(x)
    linear_attention_prefill(state, torch.arange(n, dtype=torch.int32, device="cuda"), None, offsets, x, x, x,
                             torch.zeros(h, device="cuda"), out=out, status=status)
    assert int(status) == 1 and bool((state == 1).all()) and bool((out == 0).all())
