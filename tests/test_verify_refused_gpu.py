"""What a verification leaves for a sequence that it refuses: none of its rows is kept, and its neighbours' answers stand."""
from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _verify(offsets, rows, vocab, fill):
    """The call of the C interface, with what is in the outputs before it."""
    from asterq import _lib

    g = torch.Generator(device="cuda").manual_seed(4)
    target = torch.softmax(torch.randn(rows, vocab, device="cuda", generator=g), -1)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    accept, sample = torch.full((rows,), 1e-6, device="cuda"), torch.rand(len(offsets) - 1, device="cuda", generator=g)
    starts, status = _ints(offsets), _ints([0])
    kept, n_kept, token = _ints([fill] * rows), _ints([fill] * (len(offsets) - 1)), _ints([fill] * (len(offsets) - 1))
    p = _lib.VerifyParams()
    p.dtype, p.n_seqs, p.vocab, p.n_rows, p.target_stride = _lib.DTYPE_F32, len(offsets) - 1, vocab, rows, vocab
    for name, t in dict(target=target, tokens=tokens, row_offsets=starts, accept=accept, sample=sample, kept=kept, n_kept=n_kept,
                        next_token=token, status=status).items():
        setattr(p, name, t.data_ptr())
    assert _lib.load().asterq_verify_drafts(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    return kept.tolist(), n_kept.tolist(), token.tolist(), status.item()


@pytest.mark.parametrize("vocab", [50, 20000])
def test_too_many_nodes(cuda, vocab):
    offsets = [3, 7, 7 + 1030, 7 + 1030 + 5]
    kept, count, token, status = _verify(offsets, 1044, vocab, 77)
    assert status == 1 and count == [4, 0, 5] and token[1] == -1 and 0 <= token[0] < vocab and 0 <= token[2] < vocab
    assert kept[:3] == [77] * 3 and kept[1042:] == [77] * 2  # rows of no sequence
    assert kept[3:7] == [0, 1, 2, 3] and kept[1037:1042] == [0, 1, 2, 3, 4]
    assert kept[7:1037] == [-1] * 1030


@pytest.mark.parametrize("offsets,want", [
    ([0, 4, 20, 20], [0, 1, 2, 3] + [-1] * 8),  # behind the rows
    ([0, 4, 2, 6], [0, 1, None, None, 2, 3] + [77] * 6),  # a sequence that ends before it begins: two others have rows 2 and 3
    ([-3, 5, 9, 12], [-1] * 5 + [0, 1, 2, 3, 0, 1, 2]),
    ([20, 30, 31, 32], [77] * 12),
    ([0, 30, 8, 12], [-1] * 8 + [0, 1, 2, 3]),  # the first would reach into the last one's rows
    ([-(2**31), 2**31 - 1, 6, 8], [-1] * 6 + [0, 1] + [-1] * 4),
])
def test_offsets_out_of_range(cuda, offsets, want):
    kept, count, token, status = _verify(offsets, 12, 40, 77)
    assert status == 1
    for s, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if 0 <= a <= b <= 12:
            assert count[s] == b - a
        else:
            assert count[s] == 0 and token[s] == -1
    assert all(w is None or k == w for k, w in zip(kept, want, strict=True))


def test_many_rows_of_many_refused_sequences(cuda):
    """More rows than one round of the clearing takes, refused and walked sequences in turn."""
    offsets = [5]
    for i in range(120):
        offsets.append(offsets[-1] + (1500 if i % 2 else 3))
    rows = offsets[-1] + 7
    kept, count, token, status = _verify(offsets, rows, 12, 77)
    assert status == 1 and count == [0 if i % 2 else 3 for i in range(120)]
    want = [77] * 5 + ([0, 1, 2] + [-1] * 1500) * 60 + [77] * 7
    assert kept == want


def test_the_python_call_keeps_nothing(cuda):
    from asterq.speculative import verify_drafts

    g = torch.Generator(device="cuda").manual_seed(4)
    target = torch.softmax(torch.randn(1030, 30, device="cuda", generator=g), -1)
    tokens = torch.randint(30, (1030,), device="cuda", generator=g, dtype=torch.int32)
    dirty = torch.full((1030,), 5, dtype=torch.int32, device="cuda")
    del dirty  # what the outputs' memory held before
    status = _ints([0])
    kept, n_kept, token = verify_drafts(target, tokens, _ints([0, 1030]), None, torch.zeros(1030, device="cuda"),
                                        torch.zeros(1, device="cuda"), status=status)
    assert status.item() == 1 and (kept == -1).all() and n_kept.item() == 0 and token.item() == -1
