"""Host threads that share a stream and its workspace: prompts of the linear layers take three launches, and no call's come between
those of another.  Answers are compared to the bit with the same calls made one after the other."""
from __future__ import annotations

import threading

import pytest
import torch

from test_linear_attention_gpu import _inputs, _ints, _offsets

pytestmark = pytest.mark.gpu


def test_threads_on_one_stream(cuda):
    from asterq.linear_attention import LinearAttentionWorkspace, linear_attention_prefill

    ws = LinearAttentionWorkspace()  # given, so that calls leave the interpreter's lock
    work = []
    for seed, (new, h, dk, dv) in enumerate([([4000], 4, 128, 128), ([700, 300, 900], 3, 128, 128), ([2000, 1000], 2, 64, 128),
                                             ([3000], 1, 64, 64)]):
        q, k, v, g = _inputs(sum(new), h, dk, dv, torch.bfloat16, seed)
        slots, offsets = _ints(list(range(len(new)))), _ints(_offsets(new))

        def call(args=(slots, None, offsets, q, k, v, g)):
            n, heads, dims = args[0].shape[0], args[3].shape[1], (args[4].shape[2], args[5].shape[2])
            state = torch.zeros(n, heads, *dims, device="cuda")
            return linear_attention_prefill(state, *args, workspace=ws), state

        work.append((call, call()))
    torch.cuda.synchronize()
    stream, start, got, errors = torch.cuda.Stream(), threading.Barrier(4), [], []

    def thread(i):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for k in range(100):
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
    assert not errors and len(got) == 400
    assert all(torch.equal(x, y) for a, b in got for x, y in zip(a, b))
