"""Paged grouped-query cache on the GPU: append with rotation and attention of one new token, against
plain implementations in 64 bits.

Tolerances, fixed before the first run.  u is the output type's unit roundoff (2^-8 bfloat16, 2^-11
float16, 0 for float32 outputs); where float16 is subnormal, below TINY = 2^-14, its roundoff is u TINY.
  append     |err| <= u max(|ref|, TINY) + 2^-22 (|x| + |y|): three fp32 operations on values of the pair,
             one rounding
  attention  |err| <= u |ref| + 2^-13 max|v|: scores of magnitude <= 40 carry fp32 errors of some 2^-18
             (a dot of 256 products, the scale, exp2 at 2^-22), the weights' two 16-bit parts 2^-16
  lse        |err| <= 2^-17 (1 + |ref|), the same score errors
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-14}
BAD_PAGE = -7


def _pools(n_pages, kv, page, dim, dtype, seed):
    from asterq.paged_kv import PagedKVPools

    g = torch.Generator(device="cuda").manual_seed(seed)
    return PagedKVPools(*[torch.randn(n_pages, kv, page, dim, device="cuda", generator=g).to(dtype) for _ in range(2)])


def _table(lengths, page, n_extra=2, seed=0):
    """Shuffled pages, table entries past a sequence's end not valid; the pools need n pages."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, n) // page) for n in lengths]
    ids = torch.randperm(sum(need) + n_extra, generator=g).tolist()
    width = max(need + [1]) + 1
    table = torch.full((len(lengths), width), BAD_PAGE, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(ids[at : at + n], dtype=torch.int32)
        at += n
    return table.cuda(), sum(need) + n_extra


def _visible(n, window, sink):
    if not window or n <= window:
        return list(range(n))
    sink = min(sink, window)
    return list(range(sink)) + list(range(n - (window - sink), n))


def _attention_ref(pools, table, lengths, q, scale, softcap, window, sink):
    rows, h, d = q.shape
    kv, page = pools.k.shape[1], pools.k.shape[2]
    out = torch.zeros(rows, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, h), -math.inf, dtype=torch.float64, device="cuda")
    vmax = 0.0
    for r, n in enumerate(lengths):
        if n <= 0:
            continue
        t = torch.tensor(_visible(n, window, sink), device="cuda")
        pg = table[r].long()[t // page]
        k, v = pools.k[pg, :, t % page].double(), pools.v[pg, :, t % page].double()  # [t, kv, d]
        score = torch.einsum("kgd,tkd->kgt", q[r].double().view(kv, h // kv, d), k) * scale
        if softcap:
            score = softcap * torch.tanh(score / softcap)
        lse[r] = torch.logsumexp(score, -1).reshape(h)
        out[r] = torch.einsum("kgt,tkd->kgd", torch.softmax(score, -1), v).reshape(h, d)
        vmax = max(vmax, float(v.abs().max()))
    return out, lse, vmax


def _poison(pools, table, lengths, window, sink):
    """NaN and infinities into every place of the pools that no row sees."""
    kv, page = pools.k.shape[1], pools.k.shape[2]
    seen = torch.zeros(pools.k.shape[0], page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(lengths):
        if n > 0:
            t = torch.tensor(_visible(n, window, sink), device="cuda")
            seen[table[r].long()[t // page], t % page] = True
    for pool in (pools.k, pools.v):
        pool.masked_fill_(~seen[:, None, :, None], math.nan)
        pool[..., 1::2].masked_fill_(~seen[:, None, :, None].expand_as(pool[..., 1::2]), math.inf)


CASES = [
    # dtype, head_dim, kv, group, page, lengths, window, sink, softcap
    (torch.bfloat16, 128, 2, 4, 64, [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000], 0, 0, 0.0),
    (torch.float16, 128, 1, 8, 16, [5, 0, 333, -1, 64], 0, 0, 0.0),
    (torch.bfloat16, 64, 4, 1, 48, [47, 48, 49, 95, 96, 97, 700], 0, 0, 30.0),
    (torch.float16, 64, 1, 16, 512, [511, 513, 4097], 0, 0, 0.0),
    (torch.bfloat16, 256, 2, 7, 64, [1, 31, 32, 33, 500], 0, 0, 0.0),
    (torch.float16, 256, 1, 12, 32, [1025, 3], 0, 0, 20.0),
    (torch.bfloat16, 128, 1, 40, 64, [200, 1], 0, 0, 0.0),  # more heads a kv head than a row block holds
    (torch.bfloat16, 128, 2, 2, 16, [300, 512, 513, 600, 1111, 40, 64], 512, 0, 0.0),
    (torch.bfloat16, 64, 2, 4, 16, [300, 97, 100, 101, 1111, 40, 228], 100, 4, 30.0),
    (torch.float16, 128, 1, 3, 64, [1000, 70, 71, 64], 70, 65, 0.0),  # sink and recent tokens in neighbouring tiles
    (torch.bfloat16, 128, 1, 3, 64, [1000, 10], 8, 8, 0.0),  # nothing but the sink
    (torch.bfloat16, 256, 1, 3, 16, [1000, 10, 33], 1, 0, 0.0),  # nothing but the newest token
    (torch.bfloat16, 128, 4, 4, 512, [20000], 0, 0, 0.0),  # pieces of a few tiles on every SM
    (torch.float16, 128, 1, 16, 512, [50001], 0, 0, 0.0),  # one unit over all SMs
]


@pytest.mark.parametrize("dtype,dim,kv,group,page,lengths,window,sink,softcap", CASES)
def test_attention_matches_the_formula(cuda, dtype, dim, kv, group, page, lengths, window, sink, softcap):
    from asterq.paged_kv import paged_attention

    table, n_pages = _table(lengths, page)
    pools = _pools(n_pages, kv, page, dim, dtype, 1)
    _poison(pools, table, lengths, window, sink)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (2 * torch.randn(len(lengths), kv * group, dim, device="cuda", generator=g)).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = 1.0 / math.sqrt(dim)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ref, ref_lse, vmax = _attention_ref(pools, table, lengths, q, scale, softcap, window, sink)
    for out_dtype in (dtype, torch.float32):
        out = torch.full(q.shape, math.nan, dtype=out_dtype, device="cuda")
        got, lse = paged_attention(pools, table, lens, q, logit_softcap=softcap or None, window_size=window or None,
                                   sink_tokens=sink, out=out, return_lse=True, status=status)
        assert got is out and int(status) == 0
        err = (got.double() - ref).abs()
        assert bool((err <= UNIT[out_dtype] * ref.abs() + 2.0**-13 * vmax).all()), float(err.max())
        empty = ref_lse == -math.inf
        assert bool((lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
        lerr = (lse.double() - ref_lse)[~empty].abs()
        assert bool((lerr <= 2.0**-17 * (1 + ref_lse[~empty].abs())).all()), float(lerr.max())


def test_attention_is_the_same_every_time(cuda):
    """Pieces of a sequence join in a fixed order, whichever CTA comes last."""
    from asterq.paged_kv import paged_attention

    lengths = [9000, 17, 3000]
    table, n_pages = _table(lengths, 64)
    pools = _pools(n_pages, 2, 64, 128, torch.bfloat16, 3)
    q = torch.randn(3, 16, 128, device="cuda").bfloat16()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    first = paged_attention(pools, table, lens, q)
    for _ in range(20):
        assert torch.equal(first, paged_attention(pools, table, lens, q))


def test_attention_n_new_and_strided_queries(cuda):
    from asterq.paged_kv import paged_attention

    table, n_pages = _table([130, 64, 1], 64)
    pools = _pools(n_pages, 2, 64, 128, torch.bfloat16, 4)
    wide = torch.randn(3, 24, 128, device="cuda").bfloat16()
    q = wide[:, 4:12]
    a = paged_attention(pools, table, torch.tensor([129, 63, 0], dtype=torch.int32, device="cuda"), q, n_new=1)
    b = paged_attention(pools, table, torch.tensor([130, 64, 1], dtype=torch.int32, device="cuda"), q.contiguous())
    assert torch.equal(a, b)
    # a stride that 16-byte loads cannot follow is copied first
    odd = torch.randn(3, 8, 129, device="cuda").bfloat16()[..., :128]
    c = paged_attention(pools, table, torch.tensor([130, 64, 1], dtype=torch.int32, device="cuda"), odd)
    d = paged_attention(pools, table, torch.tensor([130, 64, 1], dtype=torch.int32, device="cuda"), odd.contiguous())
    assert torch.equal(c, d)


def test_attention_nan_where_the_formula_has_one(cuda):
    """A visible key with an infinite score makes the row NaN, as inf - inf does in the formula."""
    from asterq.paged_kv import paged_attention

    table, n_pages = _table([100, 100], 64)
    pools = _pools(n_pages, 1, 64, 128, torch.bfloat16, 5)
    pools.k[table[0, 0].long(), 0, 5] = math.inf
    q = torch.rand(2, 4, 128, device="cuda").bfloat16() + 0.1
    out = paged_attention(pools, table, torch.tensor([100, 100], dtype=torch.int32, device="cuda"), q)
    assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())


def test_attention_reports_a_bad_page_and_stays_in_bounds(cuda):
    from asterq.paged_kv import paged_attention

    table, n_pages = _table([200, 100], 64)
    pools = _pools(n_pages, 1, 64, 64, torch.bfloat16, 6)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    lens = torch.tensor([200, 100], dtype=torch.int32, device="cuda")
    good = paged_attention(pools, table, lens, q)
    for bad in (-1, n_pages, 2**31 - 1):
        broken = table.clone()
        broken[0, 1] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = paged_attention(pools, broken, lens, q, status=status)
        assert int(status) == 1 and torch.equal(out[1], good[1])
    # lengths past the table end with the table
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    full = table[1:, :2].contiguous()
    over = paged_attention(pools, full, torch.tensor([2**31 - 1], dtype=torch.int32, device="cuda"), q[1:], status=status)
    assert torch.equal(over, paged_attention(pools, full, torch.tensor([128], dtype=torch.int32, device="cuda"), q[1:]))


def test_attention_of_no_rows_and_empty_pools(cuda):
    from asterq.paged_kv import PagedKVPools, paged_attention

    pools = _pools(3, 1, 16, 64, torch.float16, 7)
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert paged_attention(pools, none, none[:, 0].contiguous(), torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")).shape == (0, 2, 64)
    empty = PagedKVPools.empty(0, 1, 16, 64, dtype=torch.float16)
    out, lse = paged_attention(empty, torch.empty(2, 0, dtype=torch.int32, device="cuda"),
                               torch.zeros(2, dtype=torch.int32, device="cuda"),
                               torch.ones(2, 2, 64, dtype=torch.float16, device="cuda"), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_many_rows_of_few_tokens(cuda):
    """More sequences than a CTA has threads, many of them empty."""
    from asterq.paged_kv import paged_attention

    lengths = [(7 * i) % 19 - 1 for i in range(1501)]
    table, n_pages = _table(lengths, 16)
    pools = _pools(n_pages, 1, 16, 64, torch.bfloat16, 8)
    q = torch.randn(len(lengths), 2, 64, device="cuda").bfloat16()
    out = paged_attention(pools, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), q)
    ref, _, vmax = _attention_ref(pools, table, lengths, q, 0.125, 0.0, 0, 0)
    assert bool(((out.double() - ref).abs() <= 2.0**-8 * ref.abs() + 2.0**-13 * vmax).all())


def test_pools_past_32_bit_offsets(cuda):
    """Append to and attend over pages whose element offsets pass 2^31."""
    from asterq.paged_kv import PagedKVPools, append_kv, paged_attention

    page, kv, dim = 512, 4, 128
    n_pages = 2**31 // (page * kv * dim) + 8
    k = torch.zeros(n_pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    pools = PagedKVPools(k, v)
    table = torch.tensor([[n_pages - 1, n_pages - 3, 0]], dtype=torch.int32, device="cuda")
    n = 700
    g = torch.Generator(device="cuda").manual_seed(9)
    new_k, new_v = (torch.randn(n, kv, dim, device="cuda", generator=g).bfloat16() for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    append_kv(pools, table, zero, torch.tensor([0, n], dtype=torch.int32, device="cuda"), new_k, new_v)
    assert torch.equal(pools.k[n_pages - 1].transpose(0, 1), new_k[:page])
    assert torch.equal(pools.v[n_pages - 3].transpose(0, 1)[: n - page], new_v[page:])
    q = torch.randn(1, 8, dim, device="cuda", generator=g).bfloat16()
    out = paged_attention(pools, table, zero, q, n_new=n)
    ref, _, vmax = _attention_ref(pools, table, [n], q, dim**-0.5, 0.0, 0, 0)
    assert bool(((out.double() - ref).abs() <= 2.0**-8 * ref.abs() + 2.0**-13 * vmax).all())


# --------------------------------------------------------------------------------------------- append
def _rotate_ref(x, cos, sin, interleaved):
    """(rotated, |x| + |y| of each value's pair) in 64 bits."""
    x = x.double()
    half = cos.shape[1]
    first = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
    second = first + (1 if interleaved else half)
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., first], x[..., second]
    out, size = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 64, True), (64, 16, False), (256, 256, True),
                                                    (96, 32, False), (512, 512, False), (80, 80, True), (64, 0, False)])
@pytest.mark.parametrize("new", [[1] * 7, [0, 130, 1, 0, 0, 17, 64], [4500, 3]])
def test_append_matches_the_formula(cuda, dtype, dim, rotary, interleaved, new):
    from asterq.paged_kv import append_kv

    heads, kv, page = 6, 2, 48
    cached = [(37 * i) % 101 for i in range(len(new))]
    total = sum(new)
    table, n_pages = _table([c + n for c, n in zip(cached, new)], page)
    pools = _pools(n_pages, kv, page, dim, dtype, 10)
    before_k, before_v = pools.k.clone(), pools.v.clone()
    g = torch.Generator(device="cuda").manual_seed(11)
    fused = torch.randn(total, (heads + 2 * kv) * dim, device="cuda", generator=g).to(dtype)
    q, k, v = (x.view(total, -1, dim) for x in fused.split([heads * dim, kv * dim, kv * dim], 1))
    positions = max(c + n for c, n in zip(cached, new))
    cos = sin = None
    if rotary:
        angle = torch.arange(positions, device="cuda")[:, None] * 1000.0 ** (-torch.arange(rotary // 2, device="cuda") / rotary)
        cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    ints = dict(dtype=torch.int32, device="cuda")
    status = torch.zeros(1, **ints)
    got = append_kv(pools, table, torch.tensor(cached, **ints), torch.tensor(offsets, **ints), k, v, q=q, cos=cos, sin=sin,
                    interleaved=interleaved, status=status)
    assert int(status) == 0
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).cuda()
    seq = torch.cat([torch.full((n,), s, dtype=torch.long) for s, n in enumerate(new)]).cuda()
    pg, at = table.long()[seq, pos // page], pos % page
    for name, x, y in (("q", q, got), ("k", k, pools.k[pg, :, at])):
        if rotary:
            ref, size = _rotate_ref(x, cos[pos], sin[pos], interleaved)
            err = (y.double() - ref).abs()
            assert bool((err <= UNIT[dtype] * ref.abs().clamp(min=TINY[dtype]) + 2.0**-22 * size).all()), (name, float(err.max()))
            assert torch.equal(y[..., rotary:], x[..., rotary:])
        else:
            assert torch.equal(y, x)
    assert torch.equal(pools.v[pg, :, at], v)
    # nothing else is written
    before_k[pg, :, at], before_v[pg, :, at] = pools.k[pg, :, at], pools.v[pg, :, at]
    assert torch.equal(before_k, pools.k) and torch.equal(before_v, pools.v)


def test_append_without_queries_and_with_many_sequences(cuda):
    from asterq.paged_kv import append_kv

    n = 1300
    new = [(i * 5) % 3 for i in range(n)]
    table, n_pages = _table([20 + x for x in new], 16)
    pools = _pools(n_pages, 1, 16, 64, torch.bfloat16, 12)
    offsets = torch.cat([torch.zeros(1), torch.tensor(new).cumsum(0)]).int().cuda()
    rows = sum(new)
    k, v = (torch.randn(rows, 1, 64, device="cuda").bfloat16() for _ in range(2))
    assert append_kv(pools, table, torch.full((n,), 20, dtype=torch.int32, device="cuda"), offsets, k, v) is None
    seq = torch.cat([torch.full((x,), s, dtype=torch.long) for s, x in enumerate(new)]).cuda()
    pos = 20 + torch.arange(rows, device="cuda") - offsets.long()[seq]
    assert torch.equal(pools.k[table.long()[seq, pos // 16], :, pos % 16], k)


def test_append_leaves_out_what_has_no_place(cuda):
    """Empty slots, a bad page, a position past the table and one past cos: those rows alone are left out."""
    from asterq.paged_kv import append_kv

    ints = dict(dtype=torch.int32, device="cuda")
    pools = _pools(6, 1, 16, 64, torch.bfloat16, 13)
    k0, v0 = pools.k.clone(), pools.v.clone()
    table = torch.tensor([[0, 1], [2, 6], [3, 4], [5, -1], [-1, -1]], **ints)
    lengths = torch.tensor([-1, 15, 31, 3, 0], **ints)  # empty; 2nd page bad; past the table; fine; no page
    offsets = torch.tensor([0, 2, 4, 6, 8, 9], **ints)
    x = torch.randn(12, 3, 64, device="cuda").bfloat16()  # three rows of no sequence at the end
    q_out = torch.full((12, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cos, sin = torch.ones(40, 32, device="cuda"), torch.zeros(40, 32, device="cuda")
    status = torch.zeros(1, **ints)
    append_kv(pools, table, lengths, offsets, x[:, :1], x[:, 1:2], q=x[:, 2:], cos=cos, sin=sin, q_out=q_out, status=status)
    assert int(status) == 1
    written = {2: (2, 15), 4: (4, 15), 6: (5, 3), 7: (5, 4)}
    for row, (pg, at) in written.items():
        k0[pg, 0, at], v0[pg, 0, at] = x[row, 0], x[row, 1]
        assert torch.equal(q_out[row, 0], x[row, 2])
    assert torch.equal(pools.k, k0) and torch.equal(pools.v, v0)
    rest = [r for r in range(12) if r not in written]
    assert bool((q_out[rest] == 7.0).all())
    status.zero_()  # row 7 is at position 4: out of a table of four positions
    append_kv(pools, table, lengths, offsets, x[:, :1], x[:, 1:2], cos=cos[:4], sin=sin[:4], status=status)
    assert int(status) == 1


def test_refusals(cuda):
    from asterq import _lib
    from asterq.paged_kv import PagedKVBatch, PagedKVPools, append_kv, paged_attention

    pools = _pools(4, 2, 16, 64, torch.bfloat16, 14)
    ints = dict(dtype=torch.int32, device="cuda")
    table, lens, offs = torch.zeros(2, 2, **ints), torch.zeros(2, **ints), torch.tensor([0, 1, 2], **ints)
    q, kv = torch.zeros(2, 4, 64, device="cuda").bfloat16(), torch.zeros(2, 2, 64, device="cuda").bfloat16()
    for bad in (q[:, :3], q[..., :32], q[0]):
        with pytest.raises(ValueError):
            paged_attention(pools, table, lens, bad)
    with pytest.raises(TypeError):
        paged_attention(pools, table, lens, q.half())
    with pytest.raises(RuntimeError):
        paged_attention(pools, table, lens, q.cpu())
    for kw in (dict(window_size=0), dict(sink_tokens=-1), dict(n_new=-1)):
        with pytest.raises(ValueError):
            paged_attention(pools, table, lens, q, **kw)
    with pytest.raises(ValueError):
        paged_attention(pools, table.long(), lens, q)
    with pytest.raises(ValueError):
        paged_attention(pools, table, lens[:1], q)
    with pytest.raises(_lib.AsterqError):
        paged_attention(_pools(4, 2, 24, 64, torch.bfloat16, 0), table, lens, q)  # pages of 24 tokens
    with pytest.raises(_lib.AsterqError):
        paged_attention(_pools(4, 2, 16, 96, torch.bfloat16, 0), table, lens, torch.zeros(2, 4, 96, device="cuda").bfloat16())
    with pytest.raises(ValueError):
        append_kv(pools, table, lens, offs, kv, kv[:1])
    with pytest.raises(TypeError):
        append_kv(pools, table, lens, offs, kv.half(), kv)
    with pytest.raises(ValueError):
        append_kv(pools, table, lens, offs, kv, kv, cos=torch.zeros(4, 32, device="cuda"))
    with pytest.raises(TypeError):
        append_kv(pools, table, lens, offs, kv, kv, cos=torch.zeros(4, 32).cuda().half(), sin=torch.zeros(4, 32).cuda().half())
    with pytest.raises(_lib.AsterqError):
        append_kv(pools, table, lens, offs, kv, kv, cos=torch.zeros(4, 36, device="cuda"), sin=torch.zeros(4, 36, device="cuda"))
    with pytest.raises(ValueError):
        append_kv(pools, table, lens, offs[:2], kv, kv)
    with pytest.raises(TypeError):
        PagedKVPools(pools.k.float(), pools.v.float())
    with pytest.raises(ValueError):
        PagedKVPools(pools.k, pools.v[:, :, :, ::2])
    with pytest.raises(NotImplementedError):
        PagedKVBatch(1, 1, 96, max_seqs=1, max_tokens=16)
    batch = PagedKVBatch(1, 1, 64, max_seqs=1, max_tokens=16)
    with pytest.raises(RuntimeError):
        batch.append(0, None, kv, kv)
    batch.add_sequence()
    with pytest.raises(RuntimeError):
        batch.add_sequence()
    with pytest.raises(ValueError):
        batch.begin_rows([0], [17])


def test_workspace_too_small_is_refused(cuda):
    from asterq.paged_kv import PagedAttentionWorkspace, paged_attention

    pools = _pools(4, 2, 16, 64, torch.bfloat16, 15)
    ints = dict(dtype=torch.int32, device="cuda")
    ws = PagedAttentionWorkspace()
    ws.nbytes = 64
    with pytest.raises(ValueError, match="workspace"):
        paged_attention(pools, torch.zeros(1, 1, **ints), torch.ones(1, **ints),
                        torch.zeros(1, 4, 64, device="cuda").bfloat16(), workspace=ws)


# --------------------------------------------------------------------------------------------- the batch
def test_batch_serves_prompts_steps_and_removals(cuda):
    """Prompt chunks and decode steps of two layers over shared pages, sequences coming and going, against a
    plain cache kept on the side; a decode step is captured and replayed as a CUDA graph as well."""
    from asterq.paged_kv import PagedKVBatch

    torch.manual_seed(20)
    heads, kv, dim, layers, window = 8, 2, 64, 2, 70
    angle = torch.arange(400, device="cuda")[:, None] * 100.0 ** (-torch.arange(32, device="cuda") / 32)
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    batch = PagedKVBatch(layers, kv, dim, max_seqs=4, max_tokens=400, page_tokens=16, cos=cos, sin=sin,
                         window_size=window, sink_tokens=3)
    kept = {}  # slot -> per layer (k, v) lists, rotated in 64 bits and rounded

    def new_rows(n):
        return [[torch.randn(n, h, dim, device="cuda").bfloat16() for h in (heads, kv, kv)] for _ in range(layers)]

    def keep(slot, layer, k, v, pos):
        turned = _rotate_ref(k, cos[pos], sin[pos], False)[0].bfloat16()
        ks, vs = kept[slot][layer]
        kept[slot][layer] = (torch.cat((ks, turned)), torch.cat((vs, v)))

    def prompt(slots, tokens):
        rows = new_rows(sum(tokens))
        batch.begin_rows(slots, tokens)
        for layer in range(layers):
            batch.append(layer, *rows[layer])
            at = 0
            for s, n in sorted(zip(slots, tokens)):
                pos = torch.arange(batch.length(s), batch.length(s) + n, device="cuda")
                keep(s, layer, rows[layer][1][at : at + n], rows[layer][2][at : at + n], pos)
                at += n
        batch.end_step()

    def step():
        rows = new_rows(4)
        batch.begin_step()
        for layer in range(layers):
            q = batch.append(layer, *rows[layer])
            out = batch.attend(layer, q)
            for s in range(4):
                if s not in kept:
                    assert bool((out[s] == 0).all())
                    continue
                keep(s, layer, rows[layer][1][s : s + 1], rows[layer][2][s : s + 1],
                     torch.tensor([batch.length(s)], device="cuda"))
                k, v = kept[s][layer]
                t = torch.tensor(_visible(k.shape[0], window, 3), device="cuda")
                score = torch.einsum("kgd,tkd->kgt", q[s].double().view(kv, -1, dim), k[t].double()) * dim**-0.5
                ref = torch.einsum("kgt,tkd->kgd", torch.softmax(score, -1), v[t].double()).reshape(heads, dim)
                # the kept keys were rounded from 64 bits, the cache's from 32: half a bf16 step apart at times
                assert float((out[s].double() - ref).abs().max()) < 2.0**-5
        batch.end_step()

    def admit():
        s = batch.add_sequence()
        kept[s] = [(torch.zeros(0, kv, dim, device="cuda").bfloat16(),) * 2 for _ in range(layers)]
        return s

    a, b = admit(), admit()
    prompt([a, b], [33, 90])
    for _ in range(3):
        step()
    c = admit()
    prompt([c, a], [1, 47])
    step()
    batch.remove_sequence(b)
    del kept[b]
    step()
    b = admit()
    step()  # decodes a sequence without a prompt
    batch.raise_if_failed()
    assert [batch.length(s) for s in (a, b, c)] == [33 + 3 + 47 + 3, 1, 4]
    assert batch.lengths.tolist() == [batch.length(s) for s in range(4)]

    # a captured step replays with the lengths it finds on the device
    rows = new_rows(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    batch.begin_step()
    with torch.cuda.stream(side):
        eager = [batch.attend(i, batch.append(i, *rows[i])) for i in range(layers)]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = [batch.attend(i, batch.append(i, *rows[i])) for i in range(layers)]
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(eager, captured):
        assert torch.equal(x, y)
    batch.end_step()
