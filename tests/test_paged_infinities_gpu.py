"""Infinities and NaN in values that paged attention sees reach the output as the formula has them, in their dims alone.
Against 64 bits, by the tolerances of test_paged_kv_gpu where the formula is finite."""
from __future__ import annotations

import math

import pytest
import torch

from test_paged_kv_gpu import _attention_ref, _pools, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kv,group,lengths,window,softcap", [
    (128, 2, 4, [20000, 3, 700, 64], 0, 0.0),  # cut over all SMs, by one team, by all warps
    (64, 1, 16, [3000, 129, 1], 0, 0.0),
    (256, 1, 7, [5000, 40], 0, 30.0),
    (64, 4, 1, [1000, 90], 80, 0.0),
])
def test_values_that_are_not_finite(cuda, dtype, dim, kv, group, lengths, window, softcap):
    from asterq.paged_kv import paged_attention

    table, n_pages = _table(lengths, 16)
    pools = _pools(n_pages, kv, 16, dim, dtype, 24)
    clean = pools.v.clone()
    g = torch.Generator(device="cuda").manual_seed(25)
    q = torch.randn(len(lengths), kv * group, dim, device="cuda", generator=g).to(dtype)
    for r, n in enumerate(lengths):
        for i, values in enumerate([(math.inf,), (-math.inf,), (math.nan,), (math.inf, math.inf), (math.inf, -math.inf)]):
            for j, x in enumerate(values):
                t = max(0, n - 1 - 17 * j - 5 * i)  # within the window
                pools.v[table[r, t // 16].long(), :, t % 16, 7 * i + r] = x
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ref = _attention_ref(pools, table, lengths, q, dim**-0.5, softcap, window, 0)[0]
    assert bool((ref == math.inf).any()) and bool((ref == -math.inf).any()) and bool(ref.isnan().any())
    got = paged_attention(pools, table, lens, q, logit_softcap=softcap or None, window_size=window or None).double()
    assert torch.equal(got.isnan(), ref.isnan())
    whole = ref.isinf()
    assert torch.equal(got[whole], ref[whole])
    fine = ref.isfinite()
    bound = (2.0**-8 if dtype == torch.bfloat16 else 2.0**-11) * ref.abs() + 2.0**-13 * float(clean.abs().max())
    assert bool(((got - ref).abs() <= bound)[fine].all())
