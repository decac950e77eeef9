"""Steps of PagedKVBatch that fail on the way are abandoned: the batch goes on as if they had not begun."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _batch():
    from asterq.paged_kv import PagedKVBatch

    return PagedKVBatch(2, 1, 64, max_seqs=3, max_tokens=64, page_tokens=16)


def test_an_abandoned_step_leaves_no_trace(cuda):
    torch.manual_seed(32)
    rows = [torch.randn(3, h, 64, device="cuda").bfloat16() for h in (4, 1, 1)]
    prompt = [torch.randn(31, h, 64, device="cuda").bfloat16() for h in (4, 1, 1)]
    outs = []
    for fails in (False, True):
        batch = _batch()
        with pytest.raises(RuntimeError):
            batch.abandon_step()
        a, b = batch.add_sequence(), batch.add_sequence()
        for layer in range(2 if fails else 0):  # a prompt that fails in its second layer, over a page's end
            if layer == 0:
                batch.begin_rows([a], [20])
                batch.append(0, *[torch.randn(20, h, 64, device="cuda").bfloat16() for h in (4, 1, 1)])
            else:
                with pytest.raises(ValueError):
                    batch.append(1, *[x[:1, :, :32] for x in prompt])
                batch.abandon_step()
        batch.begin_rows([b, a], [15, 16])
        for layer in range(2):
            batch.append(layer, *prompt)
        batch.end_step()
        if fails:  # a decode step that needs a new page
            batch.begin_step()
            batch.append(0, *[x.flip(0) for x in rows])
            with pytest.raises(RuntimeError):
                batch.remove_sequence(a)
            batch.abandon_step()
        assert [batch.length(s) for s in (a, b)] == [16, 15] and batch.lengths.tolist()[:2] == [16, 15]
        batch.begin_step()
        for layer in range(2):
            outs.append(batch.attend(layer, batch.append(layer, *rows)))
        batch.end_step()
        batch.raise_if_failed()
        assert batch.lengths.tolist() == [17, 16, -1]
        batch.remove_sequence(a)
        batch.remove_sequence(b)
        assert len(batch._free.free) == batch._free.n_pages  # every page is back
    for x, y in zip(outs[:2], outs[2:]):
        assert torch.equal(x, y)
