"""A host thread whose first call on the GPU is one of these: it answers as the thread that made the inputs, to the bit (prompts of the
linear layers would otherwise take their other form, which rounds differently)."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _in_a_thread(call):
    """The call's error or None, in a host thread that has made no other."""
    errors = []

    def run():
        try:
            call()
        except Exception as e:  # shown by the test
            errors.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    return errors


@pytest.mark.parametrize("given", [False, True])  # the workspace, with which a call takes the longer way
def test_attention(cuda, given):
    from asterq.paged_kv import (PagedAttentionWorkspace, RowsAttentionWorkspace, paged_attention, paged_prompt_attention,
                                 paged_tree_attention)
    from test_rows_attention_gpu import _ints, _setup, _starts

    pools, table, q, parents, _ = _setup(torch.bfloat16, 128, 2, 4, 64, [3000, 20], [60, 64], 0, 0, True)
    lengths, starts, up = _ints([3000, 20]), _starts([60, 64]), _ints(parents[0] + parents[1])
    one, rows = (PagedAttentionWorkspace(), RowsAttentionWorkspace()) if given else (None, None)
    for call in (lambda out: paged_prompt_attention(pools, table, lengths, starts, q, out=out, workspace=rows),
                 lambda out: paged_tree_attention(pools, table, lengths, starts, up, q, out=out, workspace=rows),
                 lambda out: paged_attention(pools, table, lengths, q[:2], out=out[:2], workspace=one)):
        want, got = torch.zeros_like(q), torch.zeros_like(q)
        call(want)
        torch.cuda.synchronize()
        assert not _in_a_thread(lambda: call(got))
        assert torch.equal(want, got) and want[:2].any()


def test_linear_prompts(cuda):
    from asterq.linear_attention import LinearAttentionWorkspace, linear_attention_prefill
    from test_linear_attention_gpu import _inputs, _ints, _offsets

    q, k, v, g = _inputs(700, 2, 128, 128, torch.bfloat16, 1)
    slots, offsets = _ints([1, 0]), _ints(_offsets([600, 100]))
    for given in (False, True):
        ws = LinearAttentionWorkspace() if given else None
        states, outs = [torch.zeros(2, 2, 128, 128, device="cuda") for _ in range(2)], [torch.zeros_like(v) for _ in range(2)]

        def call(i):
            linear_attention_prefill(states[i], slots, None, offsets, q, k, v, g, out=outs[i], workspace=ws)

        call(0)
        torch.cuda.synchronize()
        assert not _in_a_thread(lambda: call(1))
        assert torch.equal(*states) and torch.equal(*outs)


def test_latent_decode(cuda):
    from asterq.decode import COLD_TILE_TOKENS, DeviceDecodePlan, latent_decode
    from asterq.plan import build_plan
    from test_decode_gpu import SCALE, single_sequence_workload

    g = torch.Generator().manual_seed(3)
    inp = {name: torch.randn(*shape, generator=g).bfloat16() for name, shape in
           dict(latent=(1501, 512), rope=(1501, 64), q_lat=(1, 16, 512), q_rope=(1, 16, 64)).items()}
    wl = single_sequence_workload(inp, 1500, 200, 1, "cuda")
    plan = DeviceDecodePlan(build_plan(wl.layouts, wl.n_heads, cold_tile=COLD_TILE_TOKENS[wl.pools.cold_scheme]), wl.q_lat.device)
    outs = []

    def call():
        outs.append(latent_decode(wl.pools, plan, wl.q_lat, wl.q_rope, wl.new_latent, wl.new_rope, softmax_scale=SCALE,
                                  out_dtype=torch.float32))

    call()
    torch.cuda.synchronize()
    assert not _in_a_thread(call)
    assert len(outs) == 2 and torch.equal(*outs) and np.isfinite(outs[0].cpu().numpy()).all()
