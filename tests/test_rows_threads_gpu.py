"""Host threads that share a stream and its workspace: attention of prompts takes two launches, and no call's come between those of
another.  Answers are compared to the bit with the same calls made one after the other."""
from __future__ import annotations

import threading

import pytest
import torch

from test_rows_attention_gpu import _ints, _setup, _starts

pytestmark = pytest.mark.gpu


def test_two_threads_on_one_stream(cuda):
    from asterq.paged_kv import RowsAttentionWorkspace, paged_prompt_attention, paged_tree_attention

    ws = RowsAttentionWorkspace()  # given, so that calls leave the interpreter's lock
    work = []
    for dim, kv, group, lengths, new, tree in (
            (128, 4, 4, [9000], [37], False), (128, 1, 8, [40, 5000, 700], [60, 9, 128], True), (64, 2, 2, [3000] * 5, [300] * 5, False),
            (256, 1, 2, [4000], [50], False)):
        pools, table, q, parents, _ = _setup(torch.bfloat16, dim, kv, group, 64, lengths, new, 0, 0, tree)
        args = (pools, table, _ints(lengths), _starts(new))
        flat = _ints([x for p in parents for x in p]) if tree else None

        def call(args=args, flat=flat, q=q):
            if flat is None:
                return paged_prompt_attention(*args, q, workspace=ws)
            return paged_tree_attention(*args, flat, q, workspace=ws)

        work.append((call, call()))
    torch.cuda.synchronize()
    stream, start, got, errors = torch.cuda.Stream(), threading.Barrier(4), [], []

    def thread(i):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for k in range(150):
                    call, want = work[(i + k) % 4]
                    got.append((call(), want))
        except Exception as e:  # shown by the test
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and len(got) == 600
    assert all(torch.equal(a, b) for a, b in got)
