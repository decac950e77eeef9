"""Linear attention with decays on the GPU, prompts and single tokens, against the recurrence in 64 bits.

Tolerances, fixed before the first run.  With B the recurrence run on absolute values (B_t = e^g B_{t-1}
+ |k| |v|^T), n the tokens of the sequence and u the output type's unit roundoff:
  state   |err| <= 8 sqrt(n + 4) 2^-24 B: a few fp32 roundings a token, adding up like a random walk
  output  |err| <= u |ref| + (2^-14 + 8 sqrt(n + 4) 2^-24) scale |q| B: products may take operands in two
          16-bit parts (2^-16 each), fp32 sums
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}


def _recurrence(s0, g, q, k, v):
    """(outputs, last state) of one sequence; q, k [n, h, dk], v [n, h, dv], g [n, h], s0 [h, dk, dv], all double."""
    s, out = s0.clone(), []
    for t in range(q.shape[0]):
        s = g[t].exp()[:, None, None] * s + k[t][:, :, None] * v[t][:, None, :]
        out.append((q[t][:, :, None] * s).sum(1))
    return torch.stack(out) if out else v.new_zeros(v.shape), s


def _check(state0, state, out, slots, lengths, offsets, q, k, v, g, scale):
    """Compare a call's outputs and states; untouched slots keep their bits."""
    touched = set()
    gd = g.double() if g.dim() == 2 else g.double().expand(q.shape[0], -1)
    for s, slot in enumerate(slots):
        a, b = offsets[s], offsets[s + 1]
        if a == b:
            continue
        if slot < 0:
            assert bool((out[a:b] == 0).all())
            continue
        touched.add(slot)
        s0 = state0[slot].double()
        if lengths is not None and lengths[s] <= 0:
            s0 = torch.zeros_like(s0)
        x = [t[a:b].double() for t in (q, k, v)]
        ref, last = _recurrence(s0, gd[a:b], *x)
        bound, size = _recurrence(s0.abs(), gd[a:b], *[t.abs() for t in x])
        walk = 8 * math.sqrt(b - a + 4) * 2.0**-24
        err = (state[slot].double() - last).abs()
        assert bool((err <= walk * size).all()), ("state", s, float((err / (walk * size + 1e-300)).max()))
        ref, bound = ref * scale, bound * scale
        err = (out[a:b].double() - ref).abs()
        assert bool((err <= UNIT[out.dtype] * ref.abs() + (2.0**-14 + walk) * bound + 1e-30).all()), \
            ("out", s, float(err.max()))
    for slot in range(state.shape[0]):
        if slot not in touched:
            assert torch.equal(state[slot], state0[slot])


def _inputs(rows, h, dk, dv, dtype, seed, decay="token"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, h * (2 * dk + dv), device="cuda", generator=gen).to(dtype)
    q, k, v = (t.view(rows, h, t.shape[1] // h) for t in x.split([h * dk, h * dk, h * dv], 1))
    if decay == "head":
        g = torch.log1p(-torch.exp2(-4.0 - 5.0 * torch.arange(h, device="cuda") / h))
    else:
        g = -torch.nn.functional.softplus(torch.randn(rows, h, device="cuda", generator=gen) * 2 - 3)
    return q, k, v, g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _offsets(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


PROMPTS = [[1], [2, 0, 1, 15, 16, 17], [63, 64, 65], [127, 128, 129, 0], [255, 256, 257], [700, 1, 31, 0, 96], [2050]]


@pytest.mark.parametrize("new", PROMPTS)
@pytest.mark.parametrize("dk,dv,h", [(128, 128, 3), (64, 64, 2), (128, 64, 1), (64, 128, 5)])
@pytest.mark.parametrize("decay", ["token", "head"])
def test_prefill_matches_the_recurrence(cuda, new, dk, dv, h, decay):
    from asterq.linear_attention import linear_attention_prefill

    n = len(new)
    q, k, v, g = _inputs(sum(new), h, dk, dv, torch.bfloat16, 1, decay)
    slots = [(3 * i + 1) % (n + 2) for i in range(n)] if (n + 2) % 3 else list(range(n))
    lengths = [7 * (i % 2) for i in range(n)]
    state = torch.randn(n + 2, h, dk, dv, device="cuda")
    for s in range(n):
        if lengths[s] == 0 and new[s]:
            state[slots[s]] = math.nan  # a fresh sequence does not read its slot
    state0 = state.clone()
    offsets = _offsets(new)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = linear_attention_prefill(state, _ints(slots), _ints(lengths), _ints(offsets), q, k, v, g, status=status)
    assert int(status) == 0
    _check(state0, state, out, slots, lengths, offsets, q, k, v, g, dk**-0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prefill_of_other_types(cuda, dtype):
    from asterq.linear_attention import linear_attention_prefill

    new = [130, 0, 65, 1]
    q, k, v, g = _inputs(sum(new), 2, 64, 128, dtype, 2)
    state = torch.randn(4, 2, 64, 128, device="cuda")
    state0 = state.clone()
    out = linear_attention_prefill(state, _ints([3, 2, 1, 0]), None, _ints(_offsets(new)), q, k, v, g, scale=0.3)
    _check(state0, state, out, [3, 2, 1, 0], None, _offsets(new), q, k, v, g, 0.3)


def test_prefill_in_pieces_is_the_whole_prompt(cuda):
    """Chunks of a prompt carried through the pool, against the same prompt at once (within both errors)."""
    from asterq.linear_attention import linear_attention_prefill

    n, h, dk, dv = 1000, 4, 128, 128
    q, k, v, g = _inputs(n, h, dk, dv, torch.bfloat16, 3)
    state = torch.randn(1, h, dk, dv, device="cuda")
    state0, outs, at = state.clone(), [], 0
    for m in (1, 300, 64, 128, 507):
        part = slice(at, at + m)
        outs.append(linear_attention_prefill(state, _ints([0]), _ints([at]), _ints([0, m]), q[part], k[part], v[part],
                                             g[part]))
        at += m
    _check(state0, state, torch.cat(outs), [0], [0], [0, n], q, k, v, g, dk**-0.5)


@pytest.mark.parametrize("strength", ["none", "reset", "infinite"])
def test_prefill_with_extreme_decays(cuda, strength):
    """No decay at all; a nearly full reset between slow decays; a decay of exactly zero."""
    from asterq.linear_attention import linear_attention_prefill

    n, h, dk, dv = 400, 2, 128, 64
    q, k, v, _ = _inputs(n, h, dk, dv, torch.bfloat16, 4)
    g = torch.zeros(n, h, device="cuda")
    if strength != "none":
        g += -1e-3
        for t in (0, 1, 70, 128, 129, 255, 256, 383, 399):
            g[t] = -1e4 if strength == "reset" else -math.inf
    state = torch.randn(1, h, dk, dv, device="cuda")
    state0 = state.clone()
    out = linear_attention_prefill(state, _ints([0]), None, _ints([0, n]), q, k, v, g)
    _check(state0, state, out, [0], None, [0, n], q, k, v, g, dk**-0.5)


def test_prefill_keeps_to_its_sequence(cuda):
    """NaN and infinities in one sequence's rows and in an empty slot's do not reach its neighbours."""
    from asterq.linear_attention import linear_attention_prefill

    new = [100, 70, 200, 40]
    q, k, v, g = _inputs(sum(new), 2, 128, 128, torch.bfloat16, 5)
    offsets = _offsets(new)
    for x in (q, k, v):
        x[offsets[1] : offsets[2]] = math.nan
        x[offsets[3] :] = math.inf
    state = torch.randn(4, 2, 128, 128, device="cuda")
    state0 = state.clone()
    out = linear_attention_prefill(state, _ints([0, 1, 2, -1]), None, _ints(offsets), q, k, v, g)
    assert bool(out[offsets[1] : offsets[2]].isnan().all()) and bool(state[1].isnan().all())
    keep = [0, 2, 3]
    assert bool((out[offsets[3] :] == 0).all()) and torch.equal(state[3], state0[3])
    for s in (0, 2):
        a, b = offsets[s], offsets[s + 1]
        part = [t[a:b] for t in (q, k, v, g)]
        _check(state0[[s]], state[[s]], out[a:b], [0], None, [0, b - a], *part, 128**-0.5)
    assert bool(state[keep].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,h,dk,dv", [(1, 1, 128, 128), (5, 3, 64, 128), (300, 2, 128, 64), (33, 16, 64, 64),
                                          (40, 16, 128, 128)])
def test_step_matches_the_recurrence(cuda, dtype, rows, h, dk, dv):
    from asterq.linear_attention import linear_attention_step

    q, k, v, g = _inputs(rows, h, dk, dv, dtype, 6, "token" if rows % 2 else "head")
    perm = torch.randperm(rows + 2, generator=torch.Generator().manual_seed(7)).tolist()
    slots = [-1 if i % 5 == 3 else perm[i] for i in range(rows)]
    state = torch.randn(rows + 2, h, dk, dv, device="cuda")
    state0 = state.clone()
    out = linear_attention_step(state, _ints(slots), q, k, v, g)
    _check(state0, state, out, slots, None, list(range(rows + 1)), q, k, v, g, dk**-0.5)


def test_step_starts_fresh_sequences_from_zeros(cuda):
    from asterq.linear_attention import linear_attention_step

    q, k, v, g = _inputs(3, 2, 64, 64, torch.bfloat16, 8)
    state = torch.full((3, 2, 64, 64), math.nan, device="cuda")
    state[1] = 1.0
    state0 = state.clone()
    out = linear_attention_step(state, _ints([0, 1, 2]), q, k, v, g, lengths=_ints([0, 5, 0]))
    _check(state0, state, out, [0, 1, 2], [0, 5, 0], [0, 1, 2, 3], q, k, v, g, 0.125)


def test_steps_follow_a_prompt(cuda):
    """A prompt and then single tokens, as a server runs them, against the recurrence over all of it."""
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step

    n, h, dk, dv = 150, 4, 128, 128
    q, k, v, g = _inputs(n + 20, h, dk, dv, torch.bfloat16, 9)
    state = torch.empty(2, h, dk, dv, device="cuda").fill_(math.nan)
    state[0] = 0.0
    outs = [linear_attention_prefill(state, _ints([1]), _ints([0]), _ints([0, n]), q[:n], k[:n], v[:n], g[:n])]
    for t in range(n, n + 20):
        outs.append(linear_attention_step(state, _ints([1]), q[t : t + 1], k[t : t + 1], v[t : t + 1], g[t : t + 1]))
    state0 = torch.zeros_like(state)
    _check(state0, state, torch.cat(outs), [1], None, [0, n + 20], q, k, v, g, dk**-0.5)


def test_bad_slots_and_offsets_are_reported(cuda):
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step

    q, k, v, g = _inputs(4, 2, 64, 64, torch.bfloat16, 10)
    state = torch.randn(3, 2, 64, 64, device="cuda")
    state0 = state.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = linear_attention_step(state, _ints([0, 3, 2**31 - 1, -5]), q, k, v, g, status=status)
    assert int(status) == 1 and bool((out[1:] == 0).all())
    _check(state0, state, out, [0, -1, -1, -1], None, [0, 1, 2, 3, 4], q, k, v, g, 0.125)
    for offsets in ([0, 5], [-1, 3], [2, 2**31 - 1]):
        status.zero_()
        before = state.clone()
        linear_attention_prefill(state, _ints([1]), None, _ints(offsets), q, k, v, g, status=status)
        assert int(status) == 1 and torch.equal(before, state)


def test_outputs_are_the_same_every_time(cuda):
    from asterq.linear_attention import linear_attention_prefill

    new = [3000, 1, 777]
    q, k, v, g = _inputs(sum(new), 4, 128, 128, torch.bfloat16, 11)
    state0 = torch.randn(3, 4, 128, 128, device="cuda")
    first = None
    for _ in range(5):
        state = state0.clone()
        out = linear_attention_prefill(state, _ints([2, 0, 1]), None, _ints(_offsets(new)), q, k, v, g)
        if first is None:
            first = (out, state)
        assert torch.equal(out, first[0]) and torch.equal(state, first[1])


def test_side_stream_and_graph(cuda):
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step

    new = [300, 65]
    q, k, v, g = _inputs(sum(new), 4, 128, 128, torch.bfloat16, 12)
    state0 = torch.randn(2, 4, 128, 128, device="cuda")
    slots, offsets = _ints([1, 0]), _ints(_offsets(new))

    def both(state):
        return (linear_attention_prefill(state, slots, None, offsets, q, k, v, g),
                linear_attention_step(state, slots, q[:2], k[:2], v[:2], g[:2]))

    plain = state0.clone()
    want = both(plain)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = state0.clone()
    with torch.cuda.stream(side):
        got = both(other)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and torch.equal(plain, other)
    third = state0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = both(third)
    third.copy_(state0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, captured)) and torch.equal(plain, third)


def test_nothing_to_do(cuda):
    from asterq.linear_attention import linear_attention_prefill

    q, k, v, g = _inputs(0, 2, 64, 64, torch.bfloat16, 13)
    state = torch.randn(1, 2, 64, 64, device="cuda")
    before = state.clone()
    assert linear_attention_prefill(state, _ints([0]), None, _ints([0, 0]), q, k, v, g).shape == (0, 2, 64)
    assert torch.equal(before, state)


def test_refusals(cuda):
    from asterq import _lib
    from asterq.linear_attention import linear_attention_prefill, linear_attention_step

    q, k, v, g = _inputs(2, 2, 64, 64, torch.bfloat16, 14)
    state, slots = torch.zeros(2, 2, 64, 64, device="cuda"), _ints([0, 1])
    for bad in ((q, k[:1], v, g), (q, k, v[:, :1], g), (q, k, v, g[:1]), (q, k, v, g.half())):
        with pytest.raises(ValueError):
            linear_attention_step(state, slots, *bad)
    with pytest.raises(TypeError):
        linear_attention_step(state, slots, q, k.half(), v, g)
    with pytest.raises(TypeError):
        linear_attention_step(state, slots, q.double(), k.double(), v.double(), g)
    with pytest.raises(RuntimeError):
        linear_attention_step(state, slots, q.cpu(), k, v, g)
    with pytest.raises(ValueError):
        linear_attention_step(state.half(), slots, q, k, v, g)
    with pytest.raises(ValueError):
        linear_attention_step(state[:, :1], slots, q, k, v, g)
    with pytest.raises(ValueError):
        linear_attention_step(state, slots[:1], q, k, v, g)
    with pytest.raises(ValueError):
        linear_attention_prefill(state, slots, None, _ints([0, 2]), q, k, v, g)
    with pytest.raises(ValueError):
        linear_attention_prefill(state, slots.long(), None, _ints([0, 1, 2]), q, k, v, g)
    with pytest.raises(_lib.AsterqError):
        linear_attention_step(torch.zeros(2, 2, 32, 32, device="cuda"), slots, q[..., :32], k[..., :32], v[..., :32], g)
