"""A prompt, steps of drafted trees and their verification by a batch, together as a server runs them, against a batch that only
ever got the accepted tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LAYERS, KV, HEADS, DIM, VOCAB = 2, 2, 8, 64, 97


class _Model:
    """A toy whose token and position decide a row's projections, and whose outputs decide probabilities."""

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(5)

        def rand(*s):
            return torch.randn(*s, device="cuda", generator=g)

        self.rows = [(rand(VOCAB, HEADS + 2 * KV, DIM)).bfloat16() for _ in range(LAYERS)]
        self.norm = [(1 + 0.2 * rand(DIM), 1 + 0.2 * rand(DIM)) for _ in range(LAYERS)]
        self.head = rand(HEADS * DIM, VOCAB)
        angle = torch.arange(400, device="cuda")[:, None] * 100.0 ** -(torch.arange(DIM // 2, device="cuda") / (DIM // 2))
        self.cos, self.sin = angle.cos(), angle.sin()

    def step(self, batch, tokens, attend):
        """Probabilities behind each row of the open step."""
        tokens = torch.tensor(tokens, device="cuda")
        mixed = 0.0
        for layer in range(LAYERS):
            x = self.rows[layer][tokens]
            q = batch.append(layer, x[:, :HEADS], x[:, HEADS : HEADS + KV], x[:, HEADS + KV :], q_norm=self.norm[layer][0],
                             k_norm=self.norm[layer][1])
            mixed = mixed + attend(layer, q).float()
        return torch.softmax(mixed.flatten(1) @ self.head * 0.1, -1)


def _batch(model, **kw):
    from asterq.paged_kv import PagedKVBatch

    return PagedKVBatch(LAYERS, KV, DIM, max_seqs=5, max_tokens=200, page_tokens=16, cos=model.cos, sin=model.sin, **kw)


@pytest.mark.parametrize("window", [None, 24])
def test_drafted_steps_end_as_plain_ones(cuda, window):
    from asterq.speculative import verify_drafts

    model, rng = _Model(), np.random.RandomState(3)
    batch = _batch(model, window_size=window, sink_tokens=3)
    slots = [batch.add_sequence(s) for s in (0, 2, 3)]
    prompts = {0: rng.randint(0, VOCAB, 37).tolist(), 2: rng.randint(0, VOCAB, 5).tolist(), 3: rng.randint(0, VOCAB, 64).tolist()}
    batch.begin_rows(slots, [len(prompts[s]) for s in slots])
    probs = model.step(batch, [t for s in slots for t in prompts[s]], batch.attend_rows)
    batch.end_step()
    ends = np.cumsum([len(prompts[s]) for s in slots]) - 1
    last = {s: int(probs[e].argmax()) for s, e in zip(slots, ends)}
    texts = {s: list(prompts[s]) for s in slots}
    fork = batch.fork_sequence(2, into=4)
    slots.append(fork)
    last[fork], texts[fork] = (last[2] + 1) % VOCAB, list(texts[2])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    accepted = 0
    g = torch.Generator(device="cuda").manual_seed(8)
    for _ in range(6):
        trees = {s: [-1] + [int(rng.randint(max(0, i - 3), i)) for i in range(1, rng.randint(2, 12))] for s in slots}
        batch.begin_tree(slots, [trees[s] for s in slots])
        tokens = [t for s in sorted(slots) for t in [last[s]] + rng.randint(0, VOCAB, len(trees[s]) - 1).tolist()]
        probs = model.step(batch, tokens, batch.attend_rows)
        kept, count, nxt = verify_drafts(probs, torch.tensor(tokens, dtype=torch.int32, device="cuda"), batch.row_offsets,
                                         batch.parents, torch.rand(len(tokens), device="cuda", generator=g) * 0.02,
                                         torch.rand(5, device="cuda", generator=g),
                                         status=status)
        counts = batch.accept(kept, count)
        flat, starts = kept.tolist(), batch.row_offsets.tolist()
        for s in slots:
            path = flat[starts[s] : starts[s] + counts[s]]
            texts[s] += [tokens[starts[s] + i] for i in path]
            last[s] = int(nxt[s])
            accepted += len(path) - 1
            assert batch.length(s) == len(texts[s]) and path[0] == 0 and -1 not in path
        assert counts[1] == 0 and batch.lengths.tolist()[1] == -1
    assert status.item() == 0 and accepted > 0
    batch.raise_if_failed()
    # the same texts as prompts of another batch: the same keys and values, and the same next step
    plain = _batch(model, window_size=window, sink_tokens=3)
    for s in sorted(slots):
        plain.add_sequence(s)
    plain.begin_rows(sorted(slots), [len(texts[s]) for s in sorted(slots)])
    model.step(plain, [t for s in sorted(slots) for t in texts[s]], plain.attend_rows)
    plain.end_step()
    for s in slots:
        t = np.arange(len(texts[s]))
        for a, b in zip(batch.layers, plain.layers):
            pick = [torch.from_numpy(x._table[s][t // 16]).long().cuda() for x in (batch, plain)]
            at = torch.from_numpy(t % 16).cuda()
            assert torch.equal(a.k[pick[0], :, at], b.k[pick[1], :, at]) and torch.equal(a.v[pick[0], :, at], b.v[pick[1], :, at])
    tokens = [last.get(s, 0) for s in range(5)]
    got = []
    for x in (batch, plain):
        x.begin_step()
        got.append(model.step(x, tokens, x.attend)[slots])
        x.end_step()
        x.raise_if_failed()
    assert torch.equal(got[0], got[1])


def test_a_step_is_closed_in_the_way_it_was_opened(cuda):
    model = _Model()
    batch = _batch(model)
    a = batch.add_sequence()
    with pytest.raises(RuntimeError):
        batch.attend_rows(0, torch.zeros(1, HEADS, DIM, device="cuda").bfloat16())
    for bad in ([[0]], [[-1, -1]], [[-1, 1]], [[]], [[-1] + [0] * 128], [[-1, 0, 5]]):
        with pytest.raises(ValueError):
            batch.begin_tree([a], bad)
    with pytest.raises(ValueError):
        batch.begin_tree([a, a], [[-1], [-1]])
    with pytest.raises(ValueError):
        batch.begin_tree([1], [[-1]])
    batch.begin_tree([a], [[-1, 0, 0]])
    with pytest.raises(RuntimeError):
        batch.end_step()
    with pytest.raises(RuntimeError):
        batch.fork_sequence(a)
    with pytest.raises(RuntimeError):
        batch.compact_pages()
    with pytest.raises(RuntimeError):
        batch.attend(0, torch.zeros(5, HEADS, DIM, device="cuda").bfloat16())
    batch.abandon_step()
    assert batch.length(a) == 0 and batch.parents is None
    # a chain of drafts may go without a tree
    batch.begin_rows([a], [4])
    probs = model.step(batch, [1, 2, 3, 4], batch.attend_rows)
    assert probs.shape == (4, VOCAB)
    kept = torch.tensor([0, 1, -1, -1], dtype=torch.int32, device="cuda")
    assert batch.accept(kept, torch.tensor([2, 0, 0, 0, 0], dtype=torch.int32, device="cuda")) == [2, 0, 0, 0, 0]
    assert batch.length(a) == 2 and batch.lengths.tolist() == [2, -1, -1, -1, -1]
    batch.begin_step()
    with pytest.raises(RuntimeError):
        batch.accept(kept, kept)
    batch.abandon_step()
    batch.raise_if_failed()
