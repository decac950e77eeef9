"""The attention of many sequences of few rows on average has units of one row tile: the cases of many rows come there beside idle
sequences, and answer as the formula and as without them to the tolerance of two roundings."""
from __future__ import annotations

import math

import pytest
import torch
from test_rows_attention_gpu import BAD_PAGE, CASES, UNIT, _check, _ints, _reference, _run, _setup

pytestmark = pytest.mark.gpu

LARGE = [c for c in CASES if sum(c[6]) > len(c[6]) * (128 // c[3]) and c[1] != 256]


@pytest.mark.parametrize("dtype,dim,kv,group,page,lengths,new,window,sink,softcap,tree", LARGE)
def test_idle_sequences_beside_long_ones(cuda, dtype, dim, kv, group, page, lengths, new, window, sink, softcap, tree):
    pools, table, q, parents, seen = _setup(dtype, dim, kv, group, page, lengths, new, window, sink, tree)
    idle = 2 * max(sum(new) * group // 128 + 1, 80)  # few rows a sequence, and more sequences than SMs
    assert sum(new) <= (len(new) + idle) * (128 // group) and len(new) + idle >= torch.cuda.get_device_properties(0).multi_processor_count
    lengths2, new2 = lengths + [-1, 5] * (idle // 2), new + [0] * idle
    table2 = torch.cat((table, torch.full((idle, table.shape[1]), BAD_PAGE, dtype=torch.int32, device="cuda")))
    parents2 = None if parents is None else parents + [[]] * idle
    status = _ints([0])
    ref, ref_lse, size = _reference(pools, table, lengths, new, q, 1.0 / math.sqrt(dim), softcap, seen)
    kw = dict(window_size=window or None, sink_tokens=sink, logit_softcap=softcap or None, return_lse=True, status=status)
    out, lse = _run(pools, table2, lengths2, new2, parents2, q, **kw)
    assert status.item() == 0
    _check(out, lse, ref, ref_lse, size, dtype)
    again, _ = _run(pools, table2, lengths2, new2, parents2, q, **kw)
    assert torch.equal(out, again)
    other, _ = _run(pools, table, lengths, new, parents, q, **kw)  # units of two row tiles
    gap = (out.double() - other.double()).abs() - 2 * (UNIT[dtype] * ref.abs() + (UNIT[dtype] + 2.0**-13) * size)
    assert gap.max() <= 0
