"""Units of one row tile (many sequences of few rows) in the forms that change scores before their maximum, and with values that are not
finite.  Against the formula in 64 bits, by the tolerances of test_rows_attention_gpu."""
from __future__ import annotations

import math

import pytest
import torch

from test_rows_attention_gpu import BAD_PAGE, _check, _ints, _reference, _run, _setup, _visible

pytestmark = pytest.mark.gpu


def _idle(table, lengths, new, parents, group):
    """The same sequences with idle ones beside them, so that units are of one row tile."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    idle = max(sum(new) // (128 // group) + 1, sms)
    table = torch.cat((table, torch.full((idle, table.shape[1]), BAD_PAGE, dtype=torch.int32, device="cuda")))
    return table, lengths + [-1] * idle, new + [0] * idle, None if parents is None else parents + [[]] * idle


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale,cap", [(None, 30.0), (None, 5.0), (-0.2, None), (0.0, None), (-0.2, 15.0)])
@pytest.mark.parametrize("dim,kv,group,page,lengths,new,window,sink,tree", [
    (128, 2, 4, 64, [300, 0, 90], [20, 33, 150], 0, 0, False),
    (64, 1, 8, 16, [1000, 3], [16, 129], 70, 3, False),
    (128, 1, 16, 48, [500, 3], [61, 9], 0, 0, True),
    (64, 2, 2, 64, [200], [100], 40, 4, True),
])
def test_scores_that_are_changed(cuda, dtype, scale, cap, dim, kv, group, page, lengths, new, window, sink, tree):
    pools, table, q, parents, seen = _setup(dtype, dim, kv, group, page, lengths, new, window, sink, tree)
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    ref, ref_lse, size = _reference(pools, table, lengths, new, q, scale, cap or 0.0, seen)
    table, lengths, new, parents = _idle(table, lengths, new, parents, group)
    status = _ints([0])
    out, lse = _run(pools, table, lengths, new, parents, q, softmax_scale=scale, logit_softcap=cap, window_size=window or None,
                    sink_tokens=sink, return_lse=True, status=status)
    assert status.item() == 0
    _check(out, lse, ref, ref_lse, size, dtype)


@pytest.mark.parametrize("dtype,dim,group,length,n,tree,window,sink", [
    (torch.bfloat16, 128, 4, 70, 150, False, 0, 0), (torch.float16, 64, 1, 0, 300, False, 0, 0), (torch.float16, 128, 8, 300, 14, False, 0, 0),
    (torch.bfloat16, 128, 4, 400, 100, False, 90, 3), (torch.bfloat16, 128, 4, 77, 60, True, 0, 0), (torch.float16, 64, 16, 1000, 30, True, 0, 0),
])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_odd_values_reach_the_rows_that_see_them(cuda, dtype, dim, group, length, n, tree, window, sink, odd):
    pools, table, q, parents, _ = _setup(dtype, dim, 1, group, 16, [length], [n], window, sink, tree)
    args = _idle(table, [length], [n], parents, group)
    kw = dict(window_size=window or None, sink_tokens=sink, return_lse=True)
    base, base_lse = _run(pools, *args, q, **kw)
    seen = _visible(length, n, window, sink, parents[0] if tree else None)
    for place in sorted({max(0, length - 30), length, length + n // 3, length + n - 1}):
        page, inside = int(table[0, place // 16]), place % 16
        old = pools.v[page, 0, inside].clone()
        pools.v[page, 0, inside, [1, dim - 1]] = odd
        out, lse = _run(pools, *args, q, **kw)
        hit = out[seen[:, place]][:, :, [1, dim - 1]].float()
        assert hit.isnan().all() if math.isnan(odd) else (hit == odd).all()
        assert torch.equal(out[~seen[:, place]], base[~seen[:, place]]) and torch.equal(lse, base_lse)
        rest = [d for d in range(dim) if d not in (1, dim - 1)]
        assert torch.equal(out[:, :, rest], base[:, :, rest])
        pools.v[page, 0, inside] = old
