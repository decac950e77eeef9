"""Steps of a batch whose window shows nothing but the sink, at the borders of pages that it gives up: every row has its page, and
the answers are those of a batch that keeps all pages, to the bit."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sink", [(4, 4), (16, 16), (20, 30), (1, 0), (5, 4)])
@pytest.mark.parametrize("tokens", [31, 47, 32])
def test_steps_behind_released_pages(cuda, window, sink, tokens):
    from asterq.paged_kv import PagedKVBatch

    def batch():
        b = PagedKVBatch(1, 2, 64, max_seqs=2, max_tokens=100, page_tokens=16, window_size=window, sink_tokens=sink)
        b.add_sequence()
        return b

    give, keep = batch(), batch()
    g = torch.Generator(device="cuda").manual_seed(3)

    def rows(n):
        return [torch.randn(n, h, 64, device="cuda", generator=g).bfloat16() for h in (4, 2, 2)]

    text = rows(tokens)
    for b in (give, keep):
        b.begin_rows([0], [tokens])
        b.append(0, *text)
        b.end_step()
    give.release_behind_window()
    for _ in range(18):
        new = rows(2)
        outs = []
        for b in (give, keep):
            b.begin_step()
            q = b.append(0, *new)
            outs.append((q[:1], b.attend(0, q)[:1]))
            b.end_step()
        assert all(torch.equal(x, y) for x, y in zip(*outs))
        give.release_behind_window()
    give.raise_if_failed()
    keep.raise_if_failed()
