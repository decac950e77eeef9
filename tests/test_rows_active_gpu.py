"""Idle sequences beside others: a call that is told how many sequences have rows answers as one without the idle ones, to the bit."""
from __future__ import annotations

import math

import pytest
import torch

from test_rows_attention_gpu import BAD_PAGE, UNIT, _ints, _reference, _run, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,kv,group,page,lengths,new,window,sink,tree", [
    (torch.bfloat16, 128, 8, 4, 64, [300], [2500], 0, 0, False),
    (torch.float16, 64, 4, 8, 16, [1000, 3], [1900, 700], 0, 0, False),
    (torch.bfloat16, 128, 8, 8, 64, [0, 900], [1300, 1], 100, 4, False),
    (torch.bfloat16, 128, 8, 16, 64, [500] * 10, [61] * 10, 0, 0, True),
    (torch.bfloat16, 256, 1, 2, 64, [100], [200], 0, 0, False),
])
@pytest.mark.parametrize("given", [False, True])  # the workspace, with which a call takes the longer way
def test_idle_sequences_change_nothing(cuda, dtype, dim, kv, group, page, lengths, new, window, sink, tree, given):
    from asterq.paged_kv import RowsAttentionWorkspace

    pools, table, q, parents, seen = _setup(dtype, dim, kv, group, page, lengths, new, window, sink, tree)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert dim == 256 or sum(new) * kv * group > sms * 4 * 128  # few enough rows are cut alike
    idle = 2 * max(sum(new) * group // 128 + 1, 80)
    table2 = torch.cat((table, torch.full((idle, table.shape[1]), BAD_PAGE, dtype=torch.int32, device="cuda")))
    parents2 = None if parents is None else parents + [[]] * idle
    status = _ints([0])
    kw = dict(window_size=window or None, sink_tokens=sink, return_lse=True, status=status)
    want = _run(pools, table, lengths, new, parents, q, **kw)
    for _ in range(2):  # the second by the short way
        got = _run(pools, table2, lengths + [-1, 5] * (idle // 2), new + [0] * idle, parents2, q, active_seqs=len(new),
                   workspace=RowsAttentionWorkspace() if given else None, **kw)
        assert status.item() == 0
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    # more than there are, and a number too low, are answered too, each to the tolerance of test_rows_attention_gpu
    ref, _, size = _reference(pools, table, lengths, new, q, 1.0 / math.sqrt(dim), 0.0, seen)
    bound = UNIT[dtype] * ref.abs() + (UNIT[dtype] + 2.0**-13) * size
    for active in (len(new) + idle + 9, 1):
        out, _ = _run(pools, table2, lengths + [-1, 5] * (idle // 2), new + [0] * idle, parents2, q, active_seqs=active, **kw)
        assert ((out.double() - ref).abs() - bound).max() <= 0


def test_refusals(cuda):
    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [10], [20], 0, 0, False)
    with pytest.raises(ValueError):
        _run(pools, table, [10], [20], None, q, active_seqs=-1)
