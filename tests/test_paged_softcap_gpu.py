"""Softcaps of any size beside the scores, from far below them to far above, where the cap does nothing.  Against the
formula in 64 bits, by the tolerances of test_paged_kv_gpu: the cap's tanh costs a score a few 2^-22 of itself."""
from __future__ import annotations

import pytest
import torch

from test_paged_kv_gpu import _attention_ref, _pools, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [0.1, 2.0, 30.0, 300.0, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("dtype,dim,group", [(torch.bfloat16, 128, 4), (torch.float16, 64, 12), (torch.bfloat16, 256, 1)])
def test_any_softcap(cuda, dtype, dim, group, softcap):
    from asterq.paged_kv import paged_attention

    lengths = [4000, 1, 77]
    table, n_pages = _table(lengths, 64)
    pools = _pools(n_pages, 2, 64, dim, dtype, 26)
    g = torch.Generator(device="cuda").manual_seed(27)
    q = (3 * torch.randn(len(lengths), 2 * group, dim, device="cuda", generator=g)).to(dtype)
    out = torch.empty(q.shape, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got, lse = paged_attention(pools, table, lens, q, logit_softcap=softcap, out=out, return_lse=True)
    ref, ref_lse, vmax = _attention_ref(pools, table, lengths, q, dim**-0.5, softcap, 0, 0)
    assert bool(((got.double() - ref).abs() <= 2.0**-13 * vmax).all()), float((got.double() - ref).abs().max())
    err = (lse.double() - ref_lse).abs()
    assert bool((err <= 2.0**-17 * (1 + ref_lse.abs())).all()), float(err.max())
