"""Attention of prompt chunks and of trees of drafted tokens over paged keys and values, against the formula in 64 bits.

Tolerances, fixed before the first run.  u is the pools' type's half step (2^-8 bfloat16, 2^-11 float16), A the sum of a
row's weights times |v| in a dim (at most max|v|), o the unit of the output's type (0 for float32).
  out  |err| <= o |ref| + (u + 2^-13) A: each weight enters its product rounded once (u of it); scores of magnitude <= 40 carry
       fp32 errors of some 2^-18 (a dot of 256 products, the scale, exp2 at 2^-22), the sum of weights 2^-16
  lse  |err| <= 2^-17 (1 + |ref|), the same score errors
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
BAD_PAGE = -7


def _pools(n_pages, kv, page, dim, dtype, seed):
    from asterq.paged_kv import PagedKVPools

    g = torch.Generator(device="cuda").manual_seed(seed)
    return PagedKVPools(*[torch.randn(n_pages, kv, page, dim, device="cuda", generator=g).to(dtype) for _ in range(2)])


def _table(totals, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, n) // page) for n in totals]
    ids = torch.randperm(sum(need) + 2, generator=g).tolist()
    table = torch.full((len(totals), max(need + [1]) + 1), BAD_PAGE, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(ids[at : at + n], dtype=torch.int32)
        at += n
    return table.cuda(), sum(need) + 2


def _tree(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [-1] + [int(torch.randint(max(0, i - 9), i, (1,), generator=g)) for i in range(1, n)]


def _visible(length, n, window, sink, parents=None):
    """[n, length + n]: what the rows of one sequence see."""
    seen = torch.zeros(n, length + n, dtype=torch.bool)
    depth = []
    sk = min(sink, window) if window else 0
    for i in range(n):
        if parents is None:
            line, pos = list(range(length + i + 1)), {j: j for j in range(length + i + 1)}
            at = length + i
        else:
            depth.append(0 if parents[i] < 0 else depth[parents[i]] + 1)
            up, j = [], i
            while j >= 0:
                up.append(j)
                j = parents[j]
            line = list(range(length)) + [length + j for j in up]
            pos = {j: j for j in range(length)} | {length + j: length + depth[j] for j in up}
            at = length + depth[i]
        seen[i, [j for j in line if not window or pos[j] < sk or pos[j] > at - (window - sk)]] = True
    return seen.cuda()


def _reference(pools, table, lengths, new, q, scale, softcap, seen):
    rows, h, d = q.shape
    kv, page = pools.k.shape[1], pools.k.shape[2]
    out = torch.zeros(rows, h, d, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    lse = torch.full((rows, h), -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for s, (length, n) in enumerate(zip(lengths, new)):
        if length >= 0 and n:
            t = torch.arange(length + n, device="cuda")
            pg = table[s].long()[t // page]
            k, v = pools.k[pg, :, t % page].double(), pools.v[pg, :, t % page].double()
            any_ = seen[s].any(0)
            k, v = k * any_[:, None, None], torch.where(any_[:, None, None], v, 0.0)
            k = torch.where(any_[:, None, None], pools.k[pg, :, t % page].double(), 0.0)
            score = torch.einsum("ikgd,tkd->kgit", q[row : row + n].double().view(n, kv, h // kv, d), k) * scale
            if softcap:
                score = softcap * torch.tanh(score / softcap)
            score = score.masked_fill(~seen[s], -math.inf)
            lse[row : row + n] = torch.logsumexp(score, -1).permute(2, 0, 1).reshape(n, h)
            w = torch.softmax(score, -1)
            out[row : row + n] = torch.einsum("kgit,tkd->ikgd", w, v).reshape(n, h, d)
            size[row : row + n] = torch.einsum("kgit,tkd->ikgd", w, v.abs()).reshape(n, h, d)
        row += n
    return out, lse, size


def _poison(pools, table, lengths, new, seen):
    """NaN and infinities into every place of the pools that no row sees."""
    page = pools.k.shape[2]
    used = torch.zeros(pools.k.shape[0], page, dtype=torch.bool, device="cuda")
    for s, (length, n) in enumerate(zip(lengths, new)):
        if length >= 0 and n:
            t = seen[s].any(0).nonzero()[:, 0]
            used[table[s].long()[t // page], t % page] = True
    for pool in (pools.k, pools.v):
        pool.masked_fill_(~used[:, None, :, None], math.nan)
        pool[..., 1::2].masked_fill_(~used[:, None, :, None].expand_as(pool[..., 1::2]), math.inf)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    return _ints([0] + torch.tensor(new).cumsum(0).tolist())


def _setup(dtype, dim, kv, group, page, lengths, new, window, sink, tree, seed=1, poison=True):
    table, n_pages = _table([max(0, c) + n for c, n in zip(lengths, new)], page)
    pools = _pools(n_pages, kv, page, dim, dtype, seed)
    parents = [_tree(n, 7 + s) if n else [] for s, n in enumerate(new)] if tree else None
    seen = [_visible(max(0, c), n, window, sink, parents[s] if tree else None) if n else None
            for s, (c, n) in enumerate(zip(lengths, new))]
    if poison:
        _poison(pools, table, lengths, new, seen)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (2 * torch.randn(sum(new), kv * group, dim, device="cuda", generator=g)).to(dtype)
    return pools, table, q, parents, seen


def _run(pools, table, lengths, new, parents, q, **kw):
    from asterq.paged_kv import paged_prompt_attention, paged_tree_attention

    if parents is None:
        return paged_prompt_attention(pools, table, _ints(lengths), _starts(new), q, **kw)
    flat = _ints([x for p in parents for x in p])
    return paged_tree_attention(pools, table, _ints(lengths), _starts(new), flat, q, **kw)


def _check(out, lse, ref, ref_lse, size, dtype):
    o = UNIT[out.dtype]
    bound = o * ref.abs() + (UNIT[dtype] + 2.0**-13) * size
    assert torch.isfinite(out).all()
    worst = ((out.double() - ref).abs() - bound).max()
    assert worst <= 0, f"{worst} above the bound"
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    err = (lse.double() - ref_lse).abs()[~empty]
    assert not err.numel() or (err <= 2.0**-17 * (1 + ref_lse.abs()[~empty])).all()


CASES = [
    # dtype, head_dim, kv, group, page, lengths, new, window, sink, softcap, tree
    (torch.bfloat16, 128, 1, 4, 64, [0], [1], 0, 0, 0.0, False),
    (torch.bfloat16, 128, 2, 4, 64, [0], [150], 0, 0, 0.0, False),
    (torch.float16, 128, 1, 1, 16, [5], [300], 0, 0, 0.0, False),
    (torch.bfloat16, 128, 2, 2, 48, [0, 100, 0, -1, 300], [1, 40, 0, 9, 200], 0, 0, 0.0, False),
    (torch.float16, 64, 2, 8, 16, [1000, 3, 127, 128, 129], [129, 16, 15, 17, 1], 0, 0, 0.0, False),
    (torch.bfloat16, 64, 1, 5, 512, [700], [260], 0, 0, 0.0, False),
    (torch.bfloat16, 256, 1, 2, 64, [100, 0], [200, 63], 0, 0, 0.0, False),
    (torch.float16, 256, 2, 7, 32, [64, 500], [20, 70], 0, 0, 30.0, False),
    (torch.bfloat16, 128, 1, 3, 64, [0, 50, 600], [400, 300, 5], 100, 4, 0.0, False),
    (torch.float16, 64, 2, 1, 16, [300, 0], [600, 700], 513, 130, 0.0, False),
    (torch.bfloat16, 128, 1, 8, 64, [1000, 3], [90, 30], 8, 8, 0.0, False),  # nothing but the sink
    (torch.bfloat16, 128, 1, 8, 64, [1000, 3], [90, 30], 1, 0, 0.0, False),  # nothing but itself
    (torch.bfloat16, 256, 1, 3, 16, [400], [100], 70, 3, 20.0, False),
    (torch.bfloat16, 128, 1, 128, 64, [33], [5], 0, 0, 0.0, False),
    (torch.bfloat16, 128, 4, 4, 512, [20000], [37], 0, 0, 0.0, False),
    (torch.float16, 128, 2, 4, 64, [7000], [1500], 0, 0, 0.0, False),  # units cut over many SMs
    (torch.bfloat16, 64, 8, 4, 64, [0] * 40, [33 + 7 * i for i in range(40)], 0, 0, 0.0, False),
    (torch.bfloat16, 128, 1, 4, 64, [10], [1], 0, 0, 0.0, True),
    (torch.bfloat16, 128, 2, 4, 64, [0, 127, 128, 500, -1, 90], [8, 30, 2, 64, 5, 0], 0, 0, 0.0, True),
    (torch.float16, 128, 1, 16, 128, [3000, 77], [61, 128], 0, 0, 0.0, True),
    (torch.bfloat16, 64, 4, 1, 16, [100, 33, 1], [128, 127, 3], 0, 0, 30.0, True),
    (torch.float16, 256, 1, 5, 48, [200, 9], [40, 33], 0, 0, 0.0, True),
    (torch.bfloat16, 128, 2, 2, 64, [500, 3, 60], [60, 70, 20], 9, 4, 0.0, True),  # windows shorter than the trees are deep
    (torch.float16, 64, 1, 8, 16, [1000, 129], [30, 100], 200, 131, 0.0, True),
    (torch.bfloat16, 128, 1, 4, 64, [40, 2], [30, 9], 6, 6, 0.0, True),
    (torch.bfloat16, 128, 8, 4, 64, [4000] * 3, [16] * 3, 0, 0, 0.0, True),
]


@pytest.mark.parametrize("dtype,dim,kv,group,page,lengths,new,window,sink,softcap,tree", CASES)
def test_rows_match_the_formula(cuda, dtype, dim, kv, group, page, lengths, new, window, sink, softcap, tree):
    pools, table, q, parents, seen = _setup(dtype, dim, kv, group, page, lengths, new, window, sink, tree)
    status = _ints([0])
    scale = 1.0 / math.sqrt(dim)
    ref, ref_lse, size = _reference(pools, table, lengths, new, q, scale, softcap, seen)
    kw = dict(window_size=window or None, sink_tokens=sink, logit_softcap=softcap or None, return_lse=True, status=status)
    out, lse = _run(pools, table, lengths, new, parents, q, **kw)
    assert status.item() == 0
    _check(out, lse, ref, ref_lse, size, dtype)
    wide, lse32 = _run(pools, table, lengths, new, parents, q, out=torch.full(q.shape, 9.0, device="cuda"), **kw)
    _check(wide, lse32, ref, ref_lse, size, dtype)
    assert torch.equal(wide.to(dtype), out) and torch.equal(lse, lse32)
