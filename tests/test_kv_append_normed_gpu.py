"""Append with norms of queries and keys and with positions of the rows' own, against the formula in 64 bits.

Tolerances, fixed before the first run.  u is the type's half step (2^-8 bfloat16, 2^-11 float16; below TINY = 2^-14 float16
is subnormal, its step u TINY).
  q, k  |err| <= u max(|ref|, TINY) + 2^-19 (|x| + |y|) for a pair (x, y) of normed values: a sum of 512 squares in fp32 carries at
        most 2^-24 log2(512) + .. < 2^-20 of itself, its root half of that, the root's reciprocal 2^-22, four products 2^-22
  v     equal
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-14}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _inputs(dtype, dim, heads, kv, rotary, page, lengths, new, fused, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(new)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if fused:
        x = (rand(total, heads + 2 * kv, dim) * 1.7).to(dtype)
        q, k, v = x[:, :heads], x[:, heads : heads + kv], x[:, heads + kv :]
    else:
        q, k, v = ((rand(total, n, dim) * 1.7).to(dtype) for n in (heads, kv, kv))
    need = [-(-(max(0, c) + n) // page) for c, n in zip(lengths, new)]
    ids = torch.randperm(sum(need) + 1, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    from asterq.paged_kv import PagedKVPools

    pools = PagedKVPools(*(rand(sum(need) + 1, kv, page, dim).to(dtype) for _ in range(2)))
    angle = rand(max(max(0, c) + n for c, n in zip(lengths, new)) + 40, rotary // 2) * 3
    return q, k, v, pools, table.cuda(), angle.cos(), angle.sin()


def _formula(x, w, eps, cos, sin, interleaved):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    n = cos.shape[-1]
    a, b = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if interleaved else (x[..., :n], x[..., n : 2 * n])
    c, s = cos.double()[:, None], sin.double()[:, None]
    turned = x.clone()
    size = x.abs().clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    turned[..., first], turned[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return turned, size


def _near(got, ref, size, dtype):
    bound = UNIT[dtype] * ref.abs().clamp(min=TINY[dtype]) + 2.0**-19 * size
    worst = ((got.double() - ref).abs() - bound).max()
    assert worst <= 0, f"{worst} above the bound"


@pytest.mark.parametrize("dtype,dim,heads,kv,rotary,interleaved,page,lengths,new,weights,tree,fused", [
    (torch.bfloat16, 128, 8, 2, 128, False, 64, [0, 63, 64, 200], [1, 1, 1, 1], "f32", False, True),
    (torch.float16, 64, 12, 4, 32, True, 16, [5, 0, -1, 100], [7, 0, 3, 20], "own", False, False),
    (torch.bfloat16, 256, 4, 1, 256, False, 48, [10, 47], [30, 2], "f32", True, True),
    (torch.float16, 96, 3, 1, 96, False, 16, [9], [50], "f32", False, True),
    (torch.bfloat16, 80, 5, 5, 16, True, 64, [1, 2], [9, 9], "own", True, False),
    (torch.float16, 512, 2, 2, 64, False, 16, [0], [33], "f32", False, False),
    (torch.bfloat16, 16, 7, 1, 16, False, 16, [3, 3], [40, 1], "f32", True, True),
    (torch.bfloat16, 128, 8, 2, 128, False, 64, [20], [40], "none", True, True),
    (torch.bfloat16, 128, 8, 2, 0, False, 64, [20], [40], "f32", False, True),
    (torch.bfloat16, 128, 16, 8, 128, False, 64, [0, 100, 7], [1900, 3, 1201], "f32", False, True),  # CTAs of several rows
])
def test_append_matches_the_formula(cuda, dtype, dim, heads, kv, rotary, interleaved, page, lengths, new, weights, tree, fused):
    from asterq.paged_kv import append_kv

    q, k, v, pools, table, cos, sin = _inputs(dtype, dim, heads, kv, max(rotary, 2), page, lengths, new, fused)
    g = torch.Generator(device="cuda").manual_seed(9)
    w = [None, None] if weights == "none" else [
        (1 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(dtype if weights == "own" else torch.float32) for _ in range(2)]
    place = [max(0, c) + i for c, n in zip(lengths, new) for i in range(n)]
    at = [max(0, c) + (i * 5 // 7) for c, n in zip(lengths, new) for i in range(n)] if tree else place
    before = pools.k.clone(), pools.v.clone()
    status = _ints([0])
    starts = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    kw = dict(cos=cos, sin=sin, interleaved=interleaved) if rotary else {}
    q_out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    got = append_kv(pools, table, _ints(lengths), starts, k, v, q=q, q_norm=w[0], k_norm=w[1], norm_eps=1e-5, q_out=q_out,
                    positions=_ints(at) if tree else None, status=status, **kw)
    assert got is q_out and status.item() == 0
    angle = torch.tensor(at, device="cuda")
    c, s = (cos[angle], sin[angle]) if rotary else (torch.ones(len(at), 0, device="cuda"), torch.zeros(len(at), 0, device="cuda"))
    live = torch.tensor([s_ for s_, n in enumerate(new) for _ in range(n)], device="cuda")
    on = _ints(lengths)[live] >= 0
    ref, size = _formula(q, w[0], 1e-5, c, s, interleaved)
    _near(got[on], ref[on], size[on], dtype)
    assert (got[~on] == 7.0).all()  # rows of an empty slot are left out
    ref, size = _formula(k, w[1], 1e-5, c, s, interleaved)
    where = torch.tensor(place, device="cuda")
    pg = table[live, where // page].long()
    _near(pools.k[pg, :, where % page][on], ref[on], size[on], dtype)
    assert torch.equal(pools.v[pg, :, where % page][on], v[on])
    rest = torch.ones(pools.k.shape[0], page, dtype=torch.bool, device="cuda")
    rest[pg[on], (where % page)[on]] = False
    for pool, old in zip((pools.k, pools.v), before):
        assert torch.equal(pool.transpose(1, 2)[rest], old.transpose(1, 2)[rest])


def test_without_weights_or_positions_it_is_the_plain_append(cuda):
    """Positions that are the places change no bit of it."""
    from asterq.paged_kv import PagedKVPools, append_kv

    q, k, v, pools, table, cos, sin = _inputs(torch.bfloat16, 128, 8, 2, 128, 64, [3, 70], [5, 60], True)
    other = PagedKVPools(pools.k.clone(), pools.v.clone())
    lengths, starts = _ints([3, 70]), _ints([0, 5, 65])
    a = append_kv(pools, table, lengths, starts, k, v, q=q, cos=cos, sin=sin)
    b = append_kv(other, table, lengths, starts, k, v, q=q, cos=cos, sin=sin,
                  positions=_ints(list(range(3, 8)) + list(range(70, 130))))
    assert torch.equal(a, b) and torch.equal(pools.k, other.k) and torch.equal(pools.v, other.v)


def test_rows_without_a_place_or_position_are_left_out(cuda):
    from asterq.paged_kv import append_kv

    q, k, v, pools, table, cos, sin = _inputs(torch.bfloat16, 64, 4, 2, 64, 16, [10], [6], True)
    before = pools.k.clone()
    status = _ints([0])
    w = torch.ones(64, device="cuda")
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    at = _ints([10, -1, 12, cos.shape[0], 14, 15])
    append_kv(pools, table, _ints([10]), _ints([0, 6]), k, v, q=q, cos=cos, sin=sin, q_norm=w, k_norm=w, positions=at, q_out=out,
              status=status)
    assert status.item() == 1
    assert (out[[1, 3]] == 7.0).all() and (out[[0, 2, 4, 5]] != 7.0).any()
    page = int(table[0, 0])
    assert torch.equal(pools.k[page, :, [11, 13]], before[page, :, [11, 13]])
    bad = table.clone()
    bad[0, 0] = pools.k.shape[0]
    status.zero_()
    before = pools.k.clone()
    append_kv(pools, bad, _ints([10]), _ints([0, 6]), k, v, q_norm=None, k_norm=w, cos=cos, sin=sin, status=status)
    assert status.item() == 1 and torch.equal(pools.k, before)


def test_refusals(cuda):
    from asterq.paged_kv import append_kv

    q, k, v, pools, table, cos, sin = _inputs(torch.bfloat16, 64, 4, 2, 64, 16, [10], [6], True)
    args = (pools, table, _ints([10]), _ints([0, 6]), k, v)
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError):
        append_kv(*args, q=q, q_norm=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        append_kv(*args, q=q, q_norm=torch.ones(64))
    with pytest.raises(TypeError):
        append_kv(*args, q=q, q_norm=w.half())
    with pytest.raises(TypeError):
        append_kv(*args, q=q, q_norm=w, k_norm=w.bfloat16())
    with pytest.raises(ValueError):
        append_kv(*args, q_norm=w)
    with pytest.raises(ValueError):
        append_kv(*args, q=q, q_norm=w, norm_eps=-1.0)
    with pytest.raises(ValueError):
        append_kv(*args, q=q, positions=_ints([0] * 6))
    with pytest.raises(ValueError):
        append_kv(*args, q=q, cos=cos, sin=sin, positions=_ints([0] * 5))
    with pytest.raises(RuntimeError):
        append_kv(*args, q=q, q_norm=w.clone().requires_grad_())
