"""The content of paged pools moved: accepted rows closed up, pages copied, and a batch's forks, truncations and compaction.
Everything is a copy, so everything is compared to the bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _stack(layers, n_pages, kv, page, dim, dtype, seed=0):
    from asterq.paged_kv import PagedKVPools, PagedKVStack

    g = torch.Generator(device="cuda").manual_seed(seed)
    return PagedKVStack([PagedKVPools(*(torch.randn(n_pages, kv, page, dim, device="cuda", generator=g).to(dtype) for _ in range(2)))
                         for _ in range(layers)])


def _all(stack):
    return [x for p in stack.layers for x in (p.k, p.v)]


@pytest.mark.parametrize("dtype,layers,kv,page,dim,lengths,kept", [
    (torch.bfloat16, 1, 1, 16, 64, [0], [[0, 2, 3]]),
    (torch.float16, 3, 2, 16, 128, [15, 16, -1, 5], [[0, 3, 17, 18], [0, 1, 2], [0, 4], []]),
    (torch.bfloat16, 70, 1, 48, 64, [40], [[0, 9, 11, 30]]),  # more layers than a launch takes
    (torch.bfloat16, 2, 8, 64, 256, [60, 3], [list(range(1, 300, 2)), list(range(140))]),  # longer than a run of rows
    (torch.float16, 2, 3, 32, 24, [31], [[5]]),
])
def test_kept_rows_close_up(cuda, dtype, layers, kv, page, dim, lengths, kept):
    from asterq.paged_kv import keep_kv_rows

    new = [(max(k) + 3) if k else 2 for k in kept]
    need = [-(-(max(0, c) + n) // page) for c, n in zip(lengths, new)]
    ids = np.random.RandomState(1).permutation(sum(need) + 2)
    stack = _stack(layers, sum(need) + 2, kv, page, dim, dtype)
    table = np.full((len(lengths), max(need) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at : at + n]
        at += n
    want = [x.clone() for x in _all(stack)]
    for s, rows in enumerate(kept):
        if lengths[s] < 0:
            continue
        for i, k in enumerate(rows):
            a, b = lengths[s] + k, lengths[s] + i
            for x, y in zip(want, _all(stack)):
                x[table[s, b // page], :, b % page] = y[table[s, a // page], :, a % page]
    flat = [k for rows, n in zip(kept, new) for k in rows + [-1] * (n - len(rows))]
    status = _ints([0])
    keep_kv_rows(stack, torch.from_numpy(table).cuda(), _ints(lengths), _ints([0] + np.cumsum(new).tolist()), _ints(flat),
                 _ints([len(k) for k in kept]), status=status)
    assert status.item() == 0
    assert all(torch.equal(x, y) for x, y in zip(want, _all(stack)))


@pytest.mark.parametrize("kept,count", [([0, 2, 2, -1], 3), ([0, 3, 1, -1], 3), ([0, 4, -1, -1], 2), ([-1, 1, 2, 3], 4),
                                        ([0, 1, 2, 3], 5)])
def test_kept_rows_that_do_not_ascend_leave_their_sequence(cuda, kept, count):
    from asterq.paged_kv import keep_kv_rows

    stack = _stack(1, 4, 1, 16, 64, torch.bfloat16)
    before = [x.clone() for x in _all(stack)]
    status = _ints([0])
    keep_kv_rows(stack, _ints([[0, 1], [2, 3]]), _ints([3, 3]), _ints([0, 4, 8]), _ints(kept + [1, 2, -1, -1]), _ints([count, 2]),
                 status=status)
    assert status.item() == 1
    for x, y in zip(_all(stack), before):
        assert torch.equal(x[:2], y[:2])
        assert torch.equal(x[2, :, 3:5], y[2, :, 4:6])  # the other sequence is done


def test_kept_rows_without_a_page_are_left_out(cuda):
    from asterq.paged_kv import keep_kv_rows

    stack = _stack(1, 2, 1, 16, 64, torch.float16)
    before = [x.clone() for x in _all(stack)]
    status = _ints([0])
    keep_kv_rows(stack, _ints([[0, 9]]), _ints([13]), _ints([0, 6]), _ints([1, 2, 4, -1, -1, -1]), _ints([3]), status=status)
    assert status.item() == 1
    for x, y in zip(_all(stack), before):
        assert torch.equal(x[0, :, 13:15], y[0, :, 14:16]) and torch.equal(x[0, :, 15], y[0, :, 15])
    # offsets out of range
    status.zero_()
    keep_kv_rows(stack, _ints([[0, 1]]), _ints([13]), _ints([2, 9]), _ints([1, 2, 4, -1, -1, -1]), _ints([3]), status=status)
    assert status.item() == 1


@pytest.mark.parametrize("layers,kv,page,dim,pairs", [
    (1, 1, 16, 64, [(0, 1)]),
    (2, 2, 48, 128, [(3, 0), (3, 5), (4, 1), (-1, 2), (2, -1), (6, 6)]),
    (66, 1, 16, 8, [(0, 2), (1, 3)]),
    (2, 8, 512, 256, [(1, 0), (1, 2)]),
])
def test_pages_are_copied(cuda, layers, kv, page, dim, pairs):
    from asterq.paged_kv import copy_kv_pages

    stack = _stack(layers, 7, kv, page, dim, torch.bfloat16)
    want = [x.clone() for x in _all(stack)]
    for a, b in pairs:
        if a >= 0 and b >= 0:
            for x, y in zip(want, _all(stack)):
                x[b] = y[a]
    status = _ints([0])
    copy_kv_pages(stack, _ints([list(p) for p in pairs]), status=status)
    assert status.item() == 0
    assert all(torch.equal(x, y) for x, y in zip(want, _all(stack)))


@pytest.mark.parametrize("pairs,done", [
    ([(0, 1), (2, 1), (3, 4)], [(3, 4)]),  # two sources for one page
    ([(0, 1), (1, 2), (3, 4)], [(3, 4)]),  # a page that is written and read
    ([(0, 1), (0, 1)], []),
    ([(0, 7), (9, 2), (3, 4)], [(3, 4)]),  # outside the pools
    ([(5, 5), (5, 2), (3, 4)], [(3, 4)]),
])
def test_pairs_that_depend_on_their_order_are_left_out(cuda, pairs, done):
    from asterq.paged_kv import copy_kv_pages

    stack = _stack(2, 7, 2, 16, 64, torch.bfloat16)
    want = [x.clone() for x in _all(stack)]
    for a, b in done:
        for x in want:
            x[b] = x[a]
    status = _ints([0])
    copy_kv_pages(stack, _ints([list(p) for p in pairs]), status=status)
    assert status.item() == 1
    assert all(torch.equal(x, y) for x, y in zip(want, _all(stack)))


def test_refusals(cuda):
    from asterq.paged_kv import PagedKVPools, PagedKVStack, copy_kv_pages, keep_kv_rows

    stack = _stack(2, 4, 1, 16, 64, torch.bfloat16)
    a, b = stack.layers
    with pytest.raises(ValueError):
        PagedKVStack([])
    with pytest.raises(ValueError):
        PagedKVStack([a, b, a])
    with pytest.raises(ValueError):
        PagedKVStack([a, PagedKVPools(b.k.half(), b.v.half())])
    with pytest.raises(ValueError):
        copy_kv_pages(stack, _ints([[0, 1, 2]]))
    with pytest.raises(ValueError):
        copy_kv_pages(stack, torch.zeros(1, 2, dtype=torch.int32))
    table, lengths, starts, kept, count = _ints([[0, 1]]), _ints([3]), _ints([0, 2]), _ints([0, 1]), _ints([1])
    for bad in ((table[0], lengths, starts, kept, count), (table, _ints([1, 2]), starts, kept, count),
                (table, lengths, _ints([0]), kept, count), (table, lengths, starts, kept.long(), count),
                (table, lengths, starts, kept, _ints([1, 1]))):
        with pytest.raises(ValueError):
            keep_kv_rows(stack, *bad)


# ---------------------------------------------------------------------------------------------------- batches
def _batch(**kw):
    from asterq.paged_kv import PagedKVBatch

    kw = dict(max_seqs=4, max_tokens=200, page_tokens=16, pool_pages=40) | kw
    return PagedKVBatch(2, 1, 64, **kw)


def _text(batch, slot):
    """A sequence's keys and values, layer by layer."""
    t = np.arange(batch.length(slot))
    pg = batch._table[slot][t // batch.page_tokens]
    return [x[torch.from_numpy(pg).long().cuda(), :, torch.from_numpy(t % batch.page_tokens).cuda()].clone()
            for x in _all(batch.stack)]


def _write(batch, slots, tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch.begin_rows(slots, tokens)
    n = sum(tokens)
    rows = [torch.randn(n, 1, 64, device="cuda", generator=g).bfloat16() for _ in range(4)]
    for layer in range(2):
        batch.append(layer, None, rows[2 * layer], rows[2 * layer + 1])
    batch.end_step()
    return rows


def _consistent(batch):
    held = [batch._table[s, : batch._held[s]] for s in range(batch.max_seqs)]
    users = np.zeros(batch._users.size, int)
    for pages in held:
        assert len(set(pages[pages >= 0].tolist())) == (pages >= 0).sum()
        users[pages[pages >= 0]] += 1
    assert np.array_equal(users, batch._users)
    assert sorted(batch._free.free) == np.nonzero(users == 0)[0].tolist()
    batch.raise_if_failed()


def test_forks_share_pages_until_one_writes(cuda):
    batch = _batch()
    a = batch.add_sequence()
    _write(batch, [a], [37], 1)
    old = _text(batch, a)
    free = len(batch._free.free)
    b = batch.fork_sequence(a)
    c = batch.fork_sequence(b, into=3)
    assert c == 3 and len(batch._free.free) == free
    _consistent(batch)
    rows = _write(batch, [a, b, c], [1, 30, 2], 2)
    _consistent(batch)
    assert len(batch._free.free) == free - 2 - 2  # two copies of the last page; b's 67 tokens are five pages, three of them had
    for slot, at, n in ((a, 0, 1), (b, 1, 30), (c, 31, 2)):
        got = _text(batch, slot)
        assert all(torch.equal(x[:37], y) for x, y in zip(got, old))
        assert all(torch.equal(x[37:], y[at : at + n]) for x, y in zip(got, rows))
    d = _text(batch, b)
    batch.remove_sequence(a)
    batch.remove_sequence(c)
    _consistent(batch)
    assert all(torch.equal(x, y) for x, y in zip(_text(batch, b), d))
    batch.remove_sequence(b)
    assert len(batch._free.free) == 40


def test_a_fork_at_a_page_border_copies_nothing(cuda):
    batch = _batch()
    a = batch.add_sequence()
    _write(batch, [a], [32], 1)
    b = batch.fork_sequence(a)
    free = len(batch._free.free)
    old = _text(batch, a)
    _write(batch, [a, b], [1, 1], 2)
    assert len(batch._free.free) == free - 2
    assert all(torch.equal(x[:32], y) for x, y in zip(_text(batch, b), old))
    _consistent(batch)


def test_truncation_gives_pages_up_and_leaves_forks_alone(cuda):
    batch = _batch()
    a = batch.add_sequence()
    _write(batch, [a], [70], 1)
    b = batch.fork_sequence(a)
    old = _text(batch, a)
    batch.truncate_sequence(a, 20)
    _consistent(batch)
    rows = _write(batch, [a], [9], 2)
    _consistent(batch)
    assert all(torch.equal(x, y) for x, y in zip(_text(batch, b), old))
    assert all(torch.equal(x[:20], y[:20]) and torch.equal(x[20:], z) for x, y, z in zip(_text(batch, a), old, rows))
    batch.truncate_sequence(b, 0)
    batch.truncate_sequence(b, 0)
    assert batch.length(b) == 0
    _consistent(batch)
    with pytest.raises(ValueError):
        batch.truncate_sequence(a, 30)
    with pytest.raises(ValueError):
        batch.truncate_sequence(2, 0)


def test_compaction_keeps_the_texts(cuda):
    batch = _batch()
    slots = [batch.add_sequence() for _ in range(4)]
    _write(batch, slots, [50, 60, 17, 90], 1)
    batch.remove_sequence(slots[0])
    batch.remove_sequence(slots[2])
    e = batch.fork_sequence(slots[3])
    texts = {s: _text(batch, s) for s in (slots[1], slots[3], e)}
    n = batch.compact_pages()
    assert n == 4 + 6 and sorted(batch._free.free) == list(range(n, 40))
    _consistent(batch)
    for s, old in texts.items():
        assert all(torch.equal(x, y) for x, y in zip(_text(batch, s), old))
    assert batch.compact_pages() == n
    _write(batch, [e], [3], 5)
    _consistent(batch)
    assert all(torch.equal(x, y) for x, y in zip(_text(batch, slots[3]), texts[slots[3]]))


def test_pages_behind_a_window_are_given_up(cuda):
    batch = _batch(window_size=40, sink_tokens=4)
    a = batch.add_sequence()
    _write(batch, [a], [120], 1)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(4, 1, 64, device="cuda", generator=g).bfloat16() for _ in range(3))

    def step():
        batch.begin_step()
        batch.append(0, None, k, v)
        out = batch.attend(0, q)
        batch.abandon_step()
        batch.begin_rows([a], [3])
        batch.append(0, None, k[:3], v[:3])
        rows = batch.attend_rows(0, q[:3])
        batch.abandon_step()
        return out, rows

    before = step()
    # 120 tokens, 36 newest: places below 120 - 36 + 1 = 85 are passed, so entries 1 .. 4 of 16 tokens
    assert batch.release_behind_window() == 4
    _consistent(batch)
    assert batch.release_behind_window() == 0
    for x, y in zip(before, step()):
        assert torch.equal(x, y)
    batch.raise_if_failed()
    b = batch.fork_sequence(a)
    batch.truncate_sequence(b, 115)
    with pytest.raises(ValueError):
        batch.truncate_sequence(a, 114)  # its window begins at 79, which has no page any more
    batch.remove_sequence(a)
    batch.remove_sequence(b)
    assert len(batch._free.free) == 40
    _consistent(batch)


def test_a_pool_that_runs_out_leaves_the_batch_as_it_was(cuda):
    batch = _batch(pool_pages=5)
    a = batch.add_sequence()
    _write(batch, [a], [70], 1)
    b = batch.fork_sequence(a)
    with pytest.raises(MemoryError):
        batch.begin_rows([a, b], [1, 1])
    _consistent(batch)
    batch.remove_sequence(a)
    _write(batch, [b], [2], 2)
    _consistent(batch)


def test_thousands_of_pages_move(cuda):
    from asterq.paged_kv import PagedKVBatch

    pages = 2700
    batch = PagedKVBatch(2, 1, 64, max_seqs=2, max_tokens=16 * pages + 16, page_tokens=16)
    for _ in range(2):
        batch.begin_rows([batch.add_sequence()], [16 * pages])
        batch.end_step()
    g = torch.Generator(device="cuda").manual_seed(4)
    for pools in batch.layers:
        pools.k.copy_(torch.randn(pools.k.shape, device="cuda", generator=g))
        pools.v.copy_(torch.randn(pools.v.shape, device="cuda", generator=g))
    first = batch.page_table[0, 0].item() < batch.page_table[1, 0].item()
    batch.remove_sequence(0 if first else 1)  # the one in front
    kept = 1 if first else 0
    at = batch.page_table[kept, :pages].long()
    want = [t[at].clone() for pools in batch.layers for t in (pools.k, pools.v)]
    assert at.min().item() >= pages and batch.compact_pages() == pages
    batch.begin_step()
    batch.abandon_step()
    now = batch.page_table[kept, :pages].long()
    assert sorted(now.tolist()) == list(range(pages))
    for x, y in zip(want, [t[now] for pools in batch.layers for t in (pools.k, pools.v)], strict=True):
        assert torch.equal(x, y)
    batch.raise_if_failed()
