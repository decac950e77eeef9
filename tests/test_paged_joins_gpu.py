"""Units of paged attention that all warps of a CTA join, beside units that one team joins by itself: the shared
buffers of the joins change hands between them.  Against the formula in 64 bits, by the tolerances of
test_paged_kv_gpu, and to the bit over repetitions."""
from __future__ import annotations

import pytest
import torch

from test_paged_kv_gpu import _attention_ref, _pools, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,kv,group,long,short", [
    (torch.bfloat16, 128, 4, 4, 330, 1),  # tiles of 64 tokens: units of six tiles and of one
    (torch.float16, 128, 2, 16, 385, 200),
    (torch.bfloat16, 64, 8, 1, 700, 100),  # tiles of 128
    (torch.bfloat16, 256, 2, 7, 170, 33),  # tiles of 32
])
def test_units_of_all_warps_beside_units_of_one_team(cuda, dtype, dim, kv, group, long, short):
    from asterq.paged_kv import paged_attention

    # runs of one, two and three units of each kind, many a CTA
    lengths = [long if (s // 3 + s // 7) % 2 else short for s in range(900)]
    table, n_pages = _table(lengths, 64)
    pools = _pools(n_pages, kv, 64, dim, dtype, 21)
    g = torch.Generator(device="cuda").manual_seed(22)
    q = torch.randn(len(lengths), kv * group, dim, device="cuda", generator=g).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = torch.empty(q.shape, device="cuda")
    first = paged_attention(pools, table, lens, q, out=out).clone()
    for _ in range(20):
        assert torch.equal(first, paged_attention(pools, table, lens, q, out=out))
    ref, _, vmax = _attention_ref(pools, table, lengths, q, dim**-0.5, 0.0, 0, 0)
    assert bool(((first.double() - ref).abs() <= 2.0**-13 * vmax).all())
