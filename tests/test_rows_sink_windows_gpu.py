"""Trees of drafted tokens under a window that is all sink: a node is seen by its position, and its key may lie behind the sink's
last tile of keys.  Against the formula in 64 bits, by the tolerances of test_rows_attention_gpu."""
from __future__ import annotations

import math

import pytest
import torch

from test_rows_attention_gpu import _check, _ints, _pools, _poison, _reference, _run, _table, _tree, _visible

pytestmark = pytest.mark.gpu


def _bush(n):
    return [-1] + [0] * (n - 1)


@pytest.mark.parametrize("dtype,dim,kv,group,page,lengths,trees,window,sink,softcap", [
    (torch.bfloat16, 128, 1, 4, 64, [120], [_bush(20)], 126, 126, 0.0),  # keys at 120 .. 139, tiles of 128
    (torch.float16, 64, 2, 2, 16, [120], [_bush(30)], 126, 126, 0.0),
    (torch.bfloat16, 256, 1, 2, 16, [60], [_bush(20)], 62, 62, 0.0),  # tiles of 64
    (torch.bfloat16, 128, 1, 4, 64, [120], [_bush(20)], 126, 500, 30.0),
    (torch.bfloat16, 128, 2, 8, 16, [127, 128, 126, 0], [_bush(100), _bush(9), _tree(60, 3), _bush(128)], 128, 128, 0.0),
    (torch.float16, 64, 1, 1, 48, [250, 255, 256, 40], [_tree(128, 1), _bush(40), _bush(3), _tree(30, 2)], 256, 256, 0.0),
    (torch.bfloat16, 128, 1, 4, 64, [0, 0], [_bush(128), _tree(128, 5)], 2, 2, 0.0),
    (torch.float16, 128, 1, 16, 128, [100, 127], [_bush(70), _bush(128)], 101, 101, 0.0),  # roots alone
    (torch.bfloat16, 128, 1, 4, 64, [120, 3000], [_bush(20), _bush(20)], 127, 126, 0.0),  # and one token besides
])
def test_nodes_behind_the_sinks_tiles(cuda, dtype, dim, kv, group, page, lengths, trees, window, sink, softcap):
    new = [len(t) for t in trees]
    table, n_pages = _table([c + n for c, n in zip(lengths, new)], page)
    pools = _pools(n_pages, kv, page, dim, dtype, 1)
    seen = [_visible(c, n, window, sink, t) for c, n, t in zip(lengths, new, trees)]
    _poison(pools, table, lengths, new, seen)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (2 * torch.randn(sum(new), kv * group, dim, device="cuda", generator=g)).to(dtype)
    ref, ref_lse, size = _reference(pools, table, lengths, new, q, 1.0 / math.sqrt(dim), softcap, seen)
    status = _ints([0])
    out, lse = _run(pools, table, lengths, new, trees, q, window_size=window, sink_tokens=sink, logit_softcap=softcap or None,
                    return_lse=True, status=status)
    assert status.item() == 0
    _check(out, lse, ref, ref_lse, size, dtype)
