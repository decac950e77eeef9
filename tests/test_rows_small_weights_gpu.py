"""Infinities among visible values whose weights are small: they reach the output of prompts and trees down to 2^-32 (f16) and 2^-126
(bf16) of the largest weight.  Scores are whole numbers of log2 units, so that weights are powers of two."""
from __future__ import annotations

import math

import pytest
import torch

from test_rows_attention_gpu import _ints, _pools, _starts, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,low", [(torch.float16, -31), (torch.bfloat16, -124)])
@pytest.mark.parametrize("dim,group", [(128, 4), (64, 8), (256, 2)])
@pytest.mark.parametrize("length,places", [(1000, (0, 100, 999)), (9000, (3, 4500, 8999))])
@pytest.mark.parametrize("before", [0, -7])  # scores of the tokens in front: the maximum stays behind or moves on
@pytest.mark.parametrize("tree", [False, True])
def test_infinities_of_small_weights(cuda, dtype, low, dim, group, length, places, before, tree):
    from asterq.paged_kv import paged_prompt_attention, paged_tree_attention

    n = 20
    table, n_pages = _table([length + n], 64)
    pools = _pools(n_pages, 1, 64, dim, dtype, 1)
    pools.k.zero_()
    t = torch.arange(length + n, device="cuda")
    page = table[0].long()[t // 64]
    pools.k[page, 0, t % 64, 0] = torch.where(t < length // 2, before, 0).to(dtype)
    q = torch.zeros(n, group, dim, device="cuda", dtype=dtype)
    q[:, :, 0] = 1
    for sign, at in enumerate(places):
        pools.k[page[at], 0, at % 64, 0] = low
        pools.v[page[at], 0, at % 64, 5 + sign] = -math.inf if sign else math.inf
    args = (pools, table, _ints([length]), _starts([n]))
    kw = dict(softmax_scale=math.log(2.0), return_lse=True)
    out, lse = paged_tree_attention(*args, _ints([-1] + [0] * (n - 1)), q, **kw) if tree else paged_prompt_attention(*args, q, **kw)
    assert (out[:, :, 5] == math.inf).all() and (out[:, :, 6:8] == -math.inf).all()
    assert torch.isfinite(out[:, :, 8:]).all() and torch.isfinite(lse).all()
