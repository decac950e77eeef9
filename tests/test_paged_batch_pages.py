"""The pages that ``PagedKVBatch`` hands out, shares and gives up, by its host-side lists alone (no GPU needed): the device's
tensors are stand-ins on the CPU, and a slot's tokens are where its table says."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from asterq import paged_kv

PAGE = 16


@pytest.fixture
def batch_of(monkeypatch):
    def empty(n_pages, n_kv_heads, page_tokens, head_dim, *, dtype, device):
        return SimpleNamespace(k=torch.empty(n_pages, n_kv_heads, page_tokens, head_dim, dtype=dtype),
                               v=torch.empty(n_pages, n_kv_heads, page_tokens, head_dim, dtype=dtype))

    monkeypatch.setattr(paged_kv.PagedKVPools, "empty", staticmethod(empty))
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    copied = []
    monkeypatch.setattr(paged_kv, "copy_kv_pages", lambda stack, pairs, status=None: copied.extend(pairs.tolist()))

    def make(**kw):
        kw = dict(max_seqs=3, max_tokens=200, page_tokens=PAGE, pool_pages=8) | kw
        batch = paged_kv.PagedKVBatch(1, 1, 64, device="cpu", **kw)
        batch.copied = copied
        return batch

    return make


def _consistent(batch):
    users = np.zeros(batch._users.size, int)
    for s in range(batch.max_seqs):
        pages = batch._table[s, : batch._held[s]]
        assert (batch._table[s, batch._held[s] :] == -1).all()
        pages = pages[pages >= 0]
        assert len(set(pages.tolist())) == pages.size
        users[pages] += 1
    assert np.array_equal(users, batch._users)
    assert sorted(batch._free.free) == np.nonzero(users == 0)[0].tolist()


def _more(batch, slot, n):
    """n more tokens of a slot; each of their places has a page that no other slot holds."""
    at = batch.length(slot)
    batch.begin_rows([slot], [n])
    pages = batch._table[slot, at // PAGE : -(-(at + n) // PAGE)]
    assert (pages >= 0).all(), f"places {at} to {at + n - 1} are in pages {pages}"
    assert (batch._users[pages] == 1).all()
    assert torch.equal(batch.page_table[slot], torch.from_numpy(batch._table[slot]))
    batch.end_step()
    _consistent(batch)


@pytest.mark.parametrize("window,sink", [(4, 4), (16, 16), (3, 7), (1, 0), (2, 1), (5, 4)])
@pytest.mark.parametrize("tokens", [15, 16, 17, 31, 32, 47, 63])
def test_the_page_of_the_next_token_is_kept(batch_of, window, sink, tokens):
    batch = batch_of(window_size=window, sink_tokens=sink)
    a = batch.add_sequence()
    _more(batch, a, tokens)
    batch.release_behind_window()
    _consistent(batch)
    for n in (1, 1, 20):
        _more(batch, a, n)
        batch.release_behind_window()
        _consistent(batch)


def test_a_page_that_a_fork_holds_is_counted_for_its_holders_alone(batch_of):
    batch = batch_of(window_size=4, sink_tokens=4, pool_pages=4)
    a, c = batch.add_sequence(), batch.add_sequence()
    _more(batch, a, 47)
    _more(batch, c, 10)
    d = batch.fork_sequence(c)
    shared = int(batch._table[c, 0])
    assert batch._users[shared] == 2 and shared == int(batch._table[d, 0])
    batch.release_behind_window()
    _more(batch, a, 1)
    batch.remove_sequence(c)
    _consistent(batch)
    assert batch._users[shared] == 1 and shared not in batch._free.free


@pytest.mark.parametrize("window,sink,tokens,to,fine", [
    (40, 4, 120, 0, True),  # nothing is left that a window could show
    (40, 4, 120, 16, True),  # all of it in the sink's page
    (40, 4, 120, 17, False),  # token 16 has no page any more
    (40, 4, 120, 114, False),  # its window begins at 79
    (40, 4, 120, 115, True),
    (40, 20, 120, 32, True),
    (40, 20, 120, 33, False),
    (4, 4, 63, 40, True),  # the sink alone is seen
    (4, 4, 63, 0, True),
    (1, 0, 63, 40, True),  # a token sees itself alone
])
def test_truncation_needs_what_the_window_shows(batch_of, window, sink, tokens, to, fine):
    batch = batch_of(window_size=window, sink_tokens=sink, pool_pages=16)
    a = batch.add_sequence()
    _more(batch, a, tokens)
    assert batch.release_behind_window() > 0
    if not fine:
        before = batch._table.copy()
        with pytest.raises(ValueError):
            batch.truncate_sequence(a, to)
        assert batch.length(a) == tokens and np.array_equal(before, batch._table)
        return
    batch.truncate_sequence(a, to)
    _consistent(batch)
    assert batch.length(a) == to
    _more(batch, a, 1)
    _more(batch, a, 50)  # and on from there
    batch.truncate_sequence(a, to + 51)
    _consistent(batch)


def test_truncation_behind_a_truncation(batch_of):
    """What was given up before a truncation does not stand in the way of one behind it."""
    batch = batch_of(window_size=40, sink_tokens=4, pool_pages=16)
    a = batch.add_sequence()
    _more(batch, a, 120)
    batch.release_behind_window()
    b = batch.fork_sequence(a)
    batch.truncate_sequence(a, 16)
    _more(batch, a, 60)
    batch.truncate_sequence(a, 40)  # all of its pages are there
    _consistent(batch)
    with pytest.raises(ValueError):
        batch.truncate_sequence(b, 40)
    batch.truncate_sequence(b, 8)
    _consistent(batch)


def test_attention_is_told_how_many_slots_have_rows(batch_of, monkeypatch):
    """A long prompt beside idle slots is not to be cut as many short ones would be."""
    told = []
    monkeypatch.setattr(paged_kv, "paged_prompt_attention", lambda *args, **kw: told.append(kw["active_seqs"]))
    monkeypatch.setattr(paged_kv, "paged_tree_attention", lambda *args, **kw: told.append(kw["active_seqs"]))
    batch = batch_of(max_seqs=5, pool_pages=30)
    slots = [batch.add_sequence() for _ in range(4)]
    for rows in ([30], [30, 1, 1], [30, 0, 1], [30]):
        batch.begin_rows(slots[: len(rows)], rows)
        batch.attend_rows(0, torch.zeros(sum(rows), 1, 64))
        batch.end_step()
    batch.begin_tree(slots[1:3], [[-1, 0], [-1, 0, 0]])
    batch.attend_rows(0, torch.zeros(5, 1, 64))
    batch.abandon_step()
    batch.begin_step()
    batch.abandon_step()
    batch.begin_rows(slots[:1], [7])
    batch.attend_rows(0, torch.zeros(7, 1, 64))
    assert told == [1, 3, 2, 1, 2, 1]
