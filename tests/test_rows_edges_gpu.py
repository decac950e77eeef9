"""Where attention of prompts and drafted trees can go wrong: values that are not finite, strides, rows and offsets out of place,
graphs and streams.  Comparisons are to the bit, or by the tolerances of test_rows_attention_gpu."""
from __future__ import annotations

import math

import pytest
import torch

from test_rows_attention_gpu import _check, _ints, _pools, _reference, _run, _setup, _starts, _table, _tree, _visible

pytestmark = pytest.mark.gpu


def _same(a, b):
    """Equal, NaN to NaN."""
    return torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("dtype,dim,group,length,n", [
    (torch.bfloat16, 128, 4, 70, 200), (torch.float16, 64, 1, 0, 400), (torch.bfloat16, 256, 2, 3, 130), (torch.float16, 128, 8, 300, 14),
    (torch.bfloat16, 128, 4, 5000, 60),
])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_odd_values_reach_the_rows_that_see_them(cuda, dtype, dim, group, length, n, odd):
    """Value dims of one new token: rows before it are as without it, rows from it on have it in these dims."""
    pools, table, q, _, _ = _setup(dtype, dim, 1, group, 16, [length], [n], 0, 0, False)
    base, base_lse = _run(pools, table, [length], [n], None, q, return_lse=True)
    for at in (0, n // 3, n - 1):
        place = length + at
        page, inside = int(table[0, place // 16]), place % 16
        old = pools.v[page, 0, inside].clone()
        pools.v[page, 0, inside, [1, dim - 1]] = odd
        out, lse = _run(pools, table, [length], [n], None, q, return_lse=True)
        assert torch.equal(lse, base_lse)
        want = base.clone()
        want[at:, :, [1, dim - 1]] = odd
        assert _same(out[:at], base[:at])
        hit = out[at:, :, [1, dim - 1]].float()
        assert hit.isnan().all() if math.isnan(odd) else (hit == odd).all()
        rest = [d for d in range(dim) if d not in (1, dim - 1)]
        assert torch.equal(out[:, :, rest], base[:, :, rest])
        pools.v[page, 0, inside] = old


def test_opposite_infinities_are_nan(cuda):
    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [20], [50], 0, 0, False)
    base = _run(pools, table, [20], [50], None, q)
    for place, value in ((30, math.inf), (45, -math.inf)):
        pools.v[int(table[0, place // 16]), 0, place % 16, 5] = value
    out = _run(pools, table, [20], [50], None, q)
    assert torch.equal(out[:10], base[:10])
    assert (out[10:25, :, 5] == math.inf).all() and out[25:, :, 5].isnan().all()


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_odd_keys_reach_the_rows_that_see_them(cuda, odd):
    pools, table, q, _, _ = _setup(torch.bfloat16, 128, 2, 4, 16, [100], [90], 0, 0, False)
    base, base_lse = _run(pools, table, [100], [90], None, q, return_lse=True)
    place = 130
    pools.k[int(table[0, place // 16]), 1, place % 16, 7] = odd
    out, lse = _run(pools, table, [100], [90], None, q, return_lse=True)
    assert torch.equal(out[:30], base[:30]) and torch.equal(lse[:30], base_lse[:30])
    assert torch.equal(out[:, :4], base[:, :4])
    if math.isnan(odd):
        assert out[30:, 4:].isnan().all() and lse[30:, 4:].isnan().all()


def test_odd_queries_stay_in_their_row(cuda):
    pools, table, q, _, _ = _setup(torch.float16, 128, 2, 4, 16, [100], [90], 0, 0, False)
    base = _run(pools, table, [100], [90], None, q)
    q = q.clone()
    q[17, 3, 0] = math.nan
    out = _run(pools, table, [100], [90], None, q)
    assert out[17, 3].isnan().all()
    keep = torch.ones(90, 8, dtype=torch.bool, device="cuda")
    keep[17, 3] = False
    assert torch.equal(out[keep], base[keep])


def test_an_odd_value_of_a_node_reaches_its_descendants_only(cuda):
    length, n = 77, 60
    pools, table, q, parents, _ = _setup(torch.bfloat16, 128, 1, 4, 16, [length], [n], 0, 0, True)
    base = _run(pools, table, [length], [n], parents, q)
    for node in (0, 7, 40):
        seen = _visible(length, n, 0, 0, parents[0])[:, length + node]
        place = length + node
        page, inside = int(table[0, place // 16]), place % 16
        old = pools.v[page, 0, inside].clone()
        pools.v[page, 0, inside, 9] = -math.inf
        out = _run(pools, table, [length], [n], parents, q)
        assert (out[seen][:, :, 9] == -math.inf).all()
        assert torch.equal(out[~seen], base[~seen])
        pools.v[page, 0, inside] = old


def test_an_odd_value_behind_a_window_has_no_part(cuda):
    pools, table, q, _, _ = _setup(torch.bfloat16, 128, 1, 4, 16, [400], [100], 90, 3, False)
    base = _run(pools, table, [400], [100], None, q, window_size=90, sink_tokens=3)
    for place in (1, 350, 420):
        page, inside = int(table[0, place // 16]), place % 16
        old = pools.v[page, 0, inside].clone()
        pools.v[page, 0, inside, 4] = math.inf
        out = _run(pools, table, [400], [100], None, q, window_size=90, sink_tokens=3)
        seen = _visible(400, 100, 90, 3)[:, place]
        assert (out[seen][:, :, 4] == math.inf).all() and torch.equal(out[~seen], base[~seen])
        pools.v[page, 0, inside] = old


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-3])
@pytest.mark.parametrize("cap", [None, 15.0])
def test_scales(cuda, scale, cap):
    args = (torch.bfloat16, 64, 2, 2, 16, [50], [70], 0, 0)
    pools, table, q, _, seen = _setup(*args, False)
    q = q / 4 if scale == 3.0 else q
    ref, ref_lse, size = _reference(pools, table, [50], [70], q, scale, cap or 0.0, seen)
    out, lse = _run(pools, table, [50], [70], None, q, softmax_scale=scale, logit_softcap=cap, return_lse=True)
    _check(out, lse, ref, ref_lse, size, torch.bfloat16)


def test_maxima_that_rise_and_fall(cuda):
    """Scores that grow tile by tile by more and by less than what O keeps its scale over, and large ones at the start."""
    for order in (1, -1):
        pools, table, q, _, seen = _setup(torch.float16, 128, 1, 4, 64, [2000], [64], 0, 0, False)
        ramp = torch.linspace(0.05, 3.0, 2064, device="cuda")[::order] if order == 1 else torch.linspace(3.0, 0.05, 2064, device="cuda")
        t = torch.arange(2064, device="cuda")
        pg = table[0].long()[t // 64]
        pools.k[pg, :, t % 64] = (pools.k[pg, :, t % 64].float() * ramp[:, None, None]).half()
        ref, ref_lse, size = _reference(pools, table, [2000], [64], q, 128**-0.5, 0.0, seen)
        out, lse = _run(pools, table, [2000], [64], None, q, return_lse=True)
        _check(out, lse, ref, ref_lse, size, torch.float16)


def test_queries_of_any_layout(cuda):
    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 2, 3, 16, [30], [45], 0, 0, False)
    want = _run(pools, table, [30], [45], None, q)
    fused = torch.randn(45, 11, 64, device="cuda").bfloat16()
    fused[:, 2:8] = q
    odd = torch.zeros(45 * 6 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(45, 6, 64)
    odd.copy_(q)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (fused[:, 2:8], odd, heads_first):
        assert torch.equal(_run(pools, table, [30], [45], None, x), want)
    one = q[:, :1].expand(45, 6, 64)
    assert torch.equal(_run(pools, table, [30], [45], None, one), _run(pools, table, [30], [45], None, one.contiguous()))
    row = q[:1].expand(45, 6, 64)
    assert torch.equal(_run(pools, table, [30], [45], None, row), _run(pools, table, [30], [45], None, row.contiguous()))


def test_single_row_and_single_head(cuda):
    pools, table, q, _, seen = _setup(torch.bfloat16, 128, 1, 1, 16, [30], [1], 0, 0, False)
    ref, ref_lse, size = _reference(pools, table, [30], [1], q, 128**-0.5, 0.0, seen)
    wide = torch.zeros(1, 3, 128, dtype=q.dtype, device="cuda")
    wide[:, 1:2] = q
    for x in (q, wide[:, 1:2]):
        out, lse = _run(pools, table, [30], [1], None, x, return_lse=True)
        _check(out, lse, ref, ref_lse, size, torch.bfloat16)


def test_rows_of_no_sequence_and_of_no_place(cuda):
    from asterq.paged_kv import paged_prompt_attention

    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [10, 0], [20, 30], 0, 0, False)
    status = _ints([0])
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    paged_prompt_attention(pools, table, _ints([10, 0]), _ints([3, 20, 44]), q, out=out, status=status)
    assert status.item() == 0 and (out[:3] == 5.0).all() and (out[44:] == 5.0).all() and (out[3:44] != 5.0).any(-1).all()
    # a table of one page: places from 16 on have none
    out.fill_(5.0)
    got, lse = paged_prompt_attention(pools, table[:, :1].contiguous(), _ints([10, -1]), _ints([0, 20, 50]), q, out=out,
                                      return_lse=True, status=status)
    assert status.item() == 1
    assert (out[6:] == 0).all() and (lse[6:] == -math.inf).all() and torch.isfinite(lse[:6]).all()
    want = _run(pools, table, [10, 0], [20, 30], None, q)
    assert (out[:6].float() - want[:6].float()).abs().max() < 0.05
    # nothing at all
    out.fill_(5.0)
    status.zero_()
    paged_prompt_attention(pools, table, _ints([-1, -1]), _ints([0, 20, 50]), q, out=out, status=status)
    assert status.item() == 0 and (out == 0).all()
    far = _ints([2**31 - 1, 0])
    paged_prompt_attention(pools, table, far, _ints([0, 20, 50]), q, out=out, status=status)
    assert status.item() == 1 and (out[:20] == 0).all() and (out[20:] != 0).any()


@pytest.mark.parametrize("starts", [[0, 30, 20], [-1, 20, 50], [0, 20, 51], [0, 60, 50]])
def test_offsets_out_of_order_leave_the_call_undone(cuda, starts):
    from asterq.paged_kv import paged_prompt_attention

    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [10, 0], [20, 30], 0, 0, False)
    status = _ints([0])
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    paged_prompt_attention(pools, table, _ints([10, 0]), _ints(starts), q, out=out, status=status)
    assert status.item() == 1 and (out == 5.0).all()


def test_trees_out_of_bounds(cuda):
    from asterq.paged_kv import paged_tree_attention

    pools, table, q, parents, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [10, 5], [100, 29], 0, 0, True)
    flat = parents[0] + parents[1]
    status = _ints([0])
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    # 129 nodes of one sequence
    paged_tree_attention(pools, table, _ints([10, 5]), _ints([0, 129, 129]), _ints(flat), q, out=out, status=status)
    assert status.item() == 1 and (out == 5.0).all()
    # parents that are not before their node: roots
    status.zero_()
    bad = list(flat)
    bad[3], bad[50], bad[99], bad[100 + 7] = 3, 90, -5, 2**31 - 1
    good = list(flat)
    for i in (3, 50, 99, 107):
        good[i] = -1
    a = paged_tree_attention(pools, table, _ints([10, 5]), _starts([100, 29]), _ints(bad), q, status=status)
    assert status.item() == 1
    status.zero_()
    b = paged_tree_attention(pools, table, _ints([10, 5]), _starts([100, 29]), _ints(good), q, status=status)
    assert status.item() == 0 and torch.equal(a, b)


def test_pages_out_of_range_are_reported(cuda):
    from asterq.paged_kv import paged_prompt_attention

    pools, table, q, _, _ = _setup(torch.bfloat16, 64, 1, 2, 16, [10, 0], [20, 30], 0, 0, False)
    for page in (-1, pools.k.shape[0], 2**31 - 1):
        bad = table.clone()
        bad[0, 1] = page
        status = _ints([0])
        out = paged_prompt_attention(pools, bad, _ints([10, 0]), _starts([20, 30]), q, status=status)
        assert status.item() == 1
        assert torch.equal(out[20:], _run(pools, table, [10, 0], [20, 30], None, q)[20:])


def test_a_chain_is_a_prompt(cuda):
    """A tree whose nodes have one child each sees what a prompt chunk of its tokens sees."""
    pools, table, q, _, _ = _setup(torch.bfloat16, 128, 2, 4, 64, [300, 0], [90, 128], 0, 0, False)
    chain = [list(range(-1, 89)), list(range(-1, 127))]
    for kw in ({}, dict(window_size=40, sink_tokens=3)):
        a, la = _run(pools, table, [300, 0], [90, 128], None, q, return_lse=True, **kw)
        b, lb = _run(pools, table, [300, 0], [90, 128], chain, q, return_lse=True, **kw)
        assert (a.float() - b.float()).abs().max() <= 2.0**-6 and (la - lb).abs().max() <= 2.0**-14


def test_one_row_is_the_single_token_call(cuda):
    from asterq.paged_kv import paged_attention

    pools, table, q, _, _ = _setup(torch.bfloat16, 128, 2, 4, 64, [299, 8, 0], [1, 1, 1], 0, 0, False)
    for kw in ({}, dict(window_size=40, sink_tokens=3), dict(logit_softcap=20.0)):
        a, la = _run(pools, table, [299, 8, 0], [1, 1, 1], None, q, return_lse=True, **kw)
        b, lb = paged_attention(pools, table, _ints([299, 8, 0]), q, n_new=1, return_lse=True, **kw)
        assert (a.float() - b.float()).abs().max() <= 2.0**-6 and (la - lb).abs().max() <= 2.0**-14


def test_the_same_bits_every_time(cuda):
    args = (torch.bfloat16, 128, 2, 4, 64, [3000, 10, 700], [100, 300, 7], 0, 0, False)
    pools, table, q, _, _ = _setup(*args)
    first = _run(pools, table, args[5], args[6], None, q, return_lse=True)
    for _ in range(10):
        again = _run(pools, table, args[5], args[6], None, q, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits(cuda):
    """Pools of more than 2^31 values, the pages in use at their end."""
    from asterq.paged_kv import PagedKVPools

    n = 2**31 // (512 * 128) + 8
    pools = PagedKVPools.empty(n, 1, 512, 128)
    small = _pools(4, 1, 512, 128, torch.bfloat16, 5)
    pools.k[n - 4 :], pools.v[n - 4 :] = small.k, small.v
    q = torch.randn(40, 4, 128, device="cuda").bfloat16()
    a = _run(pools, _ints([[n - 2, n - 4, n - 1, n - 3]]), [1500], [40], None, q)
    b = _run(small, _ints([[2, 0, 3, 1]]), [1500], [40], None, q)
    assert torch.equal(a, b)


def test_captured_calls_follow_their_inputs(cuda):
    from asterq.paged_kv import RowsAttentionWorkspace, paged_prompt_attention, paged_tree_attention

    pools, table, q, parents, _ = _setup(torch.bfloat16, 128, 2, 4, 64, [500, 20], [30, 64], 0, 0, True)
    lengths, starts, up = _ints([500, 20]), _starts([30, 64]), _ints(parents[0] + parents[1])
    for own in (None, RowsAttentionWorkspace()):
        graph = torch.cuda.CUDAGraph()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            a = paged_prompt_attention(pools, table, lengths, starts, q, workspace=own)
            b = paged_tree_attention(pools, table, lengths, starts, up, q, workspace=own)
        other = torch.randn_like(q)
        keep = q.clone()
        for x, row in ((keep, [500, 20]), (other, [500, 20]), (other, [200, 3])):
            q.copy_(x)
            lengths.copy_(_ints(row))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, _run(pools, table, row, [30, 64], None, q))
            assert torch.equal(b, _run(pools, table, row, [30, 64], parents, q))
        q.copy_(keep)
        lengths.copy_(_ints([500, 20]))


def test_calls_on_two_streams_do_not_meet(cuda):
    pools, table, q, _, _ = _setup(torch.bfloat16, 128, 2, 4, 64, [5000], [64], 0, 0, False)
    want = _run(pools, table, [5000], [64], None, q)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_run(pools, table, [5000], [64], None, q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_refusals(cuda):
    from asterq.paged_kv import paged_prompt_attention, paged_tree_attention

    pools, table, q, parents, _ = _setup(torch.bfloat16, 64, 2, 2, 16, [10], [20], 0, 0, True)
    lengths, starts, up = _ints([10]), _starts([20]), _ints(parents[0])
    for exc, args, kw in (
            (ValueError, (pools, table, lengths, starts, q[0]), {}), (ValueError, (pools, table[0], lengths, starts, q), {}),
            (ValueError, (pools, table, lengths, _ints([0]), q), {}), (ValueError, (pools, table, _ints([1, 2]), starts, q), {}),
            (TypeError, (pools, table, lengths, starts, q.half()), {}), (ValueError, (pools, table, lengths, starts, q[:, :3]), {}),
            (ValueError, (pools, table, lengths, starts, q[:, :, :32]), {}), (RuntimeError, (pools, table, lengths, starts, q.cpu()), {}),
            (ValueError, (pools, table, lengths, starts, q), dict(window_size=0)),
            (ValueError, (pools, table, lengths, starts, q), dict(sink_tokens=-1)),
            (ValueError, (pools, table, lengths, starts, q), dict(out=torch.empty_like(q)[:, :2])),
            (RuntimeError, (pools, table, lengths, starts, q), dict(out=torch.empty_like(q, dtype=torch.float16))),
            (ValueError, (pools, table, lengths, starts, q), dict(status=torch.zeros(1, device="cuda"))),
            (RuntimeError, (pools, table, lengths, starts, q.clone().requires_grad_()), {})):
        with pytest.raises(exc):
            paged_prompt_attention(*args, **kw)
    with torch.no_grad():
        paged_prompt_attention(pools, table, lengths, starts, q.clone().requires_grad_())
    for bad in (None, up[:19], up.long(), up.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            paged_tree_attention(pools, table, lengths, starts, bad, q)
