"""Paged attention of sequences whose weights span many powers of two: one token, whose value is zero, takes most of a row,
and what the many others add is all that the output is.  Against the formula in 64 bits, by the tolerances of
test_paged_kv_gpu, and to 2^-9 of the output: weights down to 2^-30 of the largest carry two 16-bit parts' bits."""
from __future__ import annotations

import pytest
import torch

from test_paged_kv_gpu import _attention_ref, _pools, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,dim,group", [(1, 131072, 64, 8), (300, 4000, 64, 8), (300, 2111, 128, 16), (300, 1000, 256, 2),
                                              (300, 50, 64, 1)])
def test_many_small_weights_beside_a_large_one(cuda, dtype, rows, n, dim, group):
    from asterq.paged_kv import paged_attention

    lengths = [n] * rows
    table, n_pages = _table(lengths, 64)
    pools = _pools(n_pages, 1, 64, dim, dtype, 23)
    pools.k.zero_()
    pools.v.fill_(1.0)
    # query head h's first token outweighs each of the others by 2^10 to 2^30, in steps over all fractions of a power
    gap = torch.arange(group, device="cuda") * (20.0 / group) + 10.03
    first = table[:, 0].long()
    pools.k[first, 0, 0, 0] = 4.0
    pools.v[first, 0, 0] = 0.0
    q = torch.zeros(rows, group, dim, device="cuda")
    q[:, :, 0] = gap * 0.6931472 * dim**0.5 / 4.0
    q = q.to(dtype)
    out = torch.empty(q.shape, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got, lse = paged_attention(pools, table, lens, q, out=out, return_lse=True)
    ref, ref_lse, _ = _attention_ref(pools, table, lengths[:1], q[:1], dim**-0.5, 0.0, 0, 0)  # all rows are the same
    err = (got.double() - ref).abs()
    assert bool((err <= 2.0**-13).all()), float(err.max())
    assert bool((err <= 2.0**-9 * ref).all()), float((err / ref).max())
    assert bool(((lse.double() - ref_lse).abs() <= 2.0**-17 * (1 + ref_lse.abs())).all())
