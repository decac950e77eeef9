"""Workloads of the operators that serve a hybrid model's other layers.

Beside its latent-attention layers a hybrid model has layers of grouped-query attention over a
paged key/value cache and layers of linear attention with a fixed-size state.  One decode step or
one prompt chunk of such layers is four operators:

  append         new keys and values into their pages, keys and queries rotated on the way
  attention      one new token a sequence over its pages
  prompt         linear attention of prompt chunks, state carried from and to its pool
  step           linear attention of one new token a sequence

``run`` computes them in plain torch (``own`` false) or calls the package's kernels (``own`` true).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_BASE = 10000.0
CHUNK = 64  # tokens of a chunk of the plain form of the prompt operator


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asterlm-frontier_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from asterq import linear_attention, paged_kv

    return paged_kv, linear_attention


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the smallest decode steps: a handful of sequences, where the launch is what counts
        dict(name="append, 8 single tokens", op="append", seqs=8, tokens=0, context=1024, heads=16, kv_heads=2,
             head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", page_tokens=64),
        # an ordinary decode step of a full batch, half of each head rotated in interleaved pairs
        dict(name="append, 256 single tokens", op="append", seqs=256, tokens=0, context=700, heads=32, kv_heads=8,
             head_dim=64, rotary_dim=32, interleaved=True, dtype="f16", page_tokens=16),
        # prompt chunks of a few requests admitted together, ragged, on top of what they have cached
        dict(name="append, ragged prompts", op="append", seqs=13, tokens=16411, context=2048, heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", page_tokens=512),
        # one interactive sequence: latency, the cache split over all SMs
        dict(name="attention, one of 8192", op="attention", rows=1, min_len=8192, max_len=8192, empty=0, heads=16,
             kv_heads=4, head_dim=128, dtype="bf16", page_tokens=512, window=0, sink=0, softcap=0.0),
        # continuous batching of ragged contexts, 1k to 32k tokens: the bandwidth case
        dict(name="attention, 64 ragged to 32k", op="attention", rows=64, min_len=1024, max_len=32768, empty=0,
             heads=32, kv_heads=8, head_dim=128, dtype="bf16", page_tokens=64, window=0, sink=0, softcap=0.0),
        # one long document, one key/value head for all query heads
        dict(name="attention, one of 131072", op="attention", rows=1, min_len=131072, max_len=131072, empty=0,
             heads=16, kv_heads=1, head_dim=128, dtype="f16", page_tokens=512, window=0, sink=0, softcap=0.0),
        # many short chats with a head of keys for each query head, sliding window and sink, empty slots
        dict(name="attention, 256 short, window", op="attention", rows=256, min_len=1, max_len=2047, empty=9,
             heads=16, kv_heads=16, head_dim=64, dtype="bf16", page_tokens=16, window=512, sink=4, softcap=30.0),
        # one prompt of an interactive request: few heads, so the work has to be split over its length
        dict(name="prompt, one of 8192", op="prompt", seqs=1, tokens=8192, carried=0, heads=16, dk=128, dv=128,
             decay="token"),
        # prompts admitted together, ragged, some of them continuing from a state
        dict(name="prompt, ragged 32k", op="prompt", seqs=12, tokens=32777, carried=5, heads=32, dk=128, dv=128,
             decay="token"),
        # smaller heads with one constant decay each, short ragged prompts
        dict(name="prompt, 40 short of 64 wide", op="prompt", seqs=40, tokens=9001, carried=0, heads=12, dk=64, dv=64,
             decay="head"),
        # a decode step of a few sequences
        dict(name="step, 4 rows", op="step", rows=4, empty=0, heads=16, dk=128, dv=128, decay="token", dtype="bf16"),
        # a decode step of a full batch with idle slots: the states' traffic
        dict(name="step, 256 rows", op="step", rows=256, empty=3, heads=32, dk=128, dv=128, decay="head",
             dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm; sizes met nowhere in use are stepped over."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    return n + 1 if n % 1024 == 0 and n % 3 == 0 else n


def _odd_width(n):
    return n != 3072


def draw(rng):
    while True:
        case = _draw(rng)
        if case is not None:
            return case


def _draw(rng):
    op = rng.choice(["append", "attention", "prompt", "step"])
    if op == "append":
        d = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        rotary = rng.choice([d, d, d // 2])
        prompt = rng.random() < 0.5
        seqs = _spread(rng, 1, 24) if prompt else _spread(rng, 1, 256)
        tokens = _spread(rng, 2 * seqs, 12000) if prompt else 0
        context = _spread(rng, 1, 1500)
        if heads * (tokens or seqs) * d > 32 * 16000 * 128 or (seqs * (context + 64) + tokens) * kv * d > 1 << 28:
            return None
        if not (_odd_width(heads * d) and _odd_width((heads + 2 * kv) * d)):
            return None
        return dict(op=op, seqs=seqs, tokens=tokens, context=context, heads=heads, kv_heads=kv, head_dim=d,
                    rotary_dim=rotary, interleaved=rng.random() < 0.4, dtype=rng.choice(["bf16", "f16"]),
                    page_tokens=rng.choice([16, 48, 64, 256, 512]))
    if op == "attention":
        d = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 7, 8, 16])
        rows = _spread(rng, 1, 256)
        max_len = _spread(rng, 1, 131072)
        min_len = max(1, int(max_len * rng.choice([0.02, 0.1, 0.5, 1.0])))
        if rows * max_len * kv * d > 64 * 32768 * 8 * 128 // 2 or not _odd_width(kv * group * d):
            return None
        window = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
        return dict(op=op, rows=rows, min_len=min_len, max_len=max_len, empty=rng.choice([0, 0, rows // 9]),
                    heads=kv * group, kv_heads=kv, head_dim=d, dtype=rng.choice(["bf16", "f16"]),
                    page_tokens=rng.choice([16, 48, 64, 128, 512]), window=window,
                    sink=rng.choice([0, 4, 13]) if window else 0, softcap=rng.choice([0.0, 0.0, 30.0]))
    heads = rng.choice([1, 3, 4, 8, 12, 16, 32])
    dk, dv = rng.choice([64, 128]), rng.choice([64, 128])
    decay = rng.choice(["token", "head"])
    if not (_odd_width(heads * dk) and _odd_width(heads * dv) and _odd_width(heads * (2 * dk + dv))):
        return None
    if op == "prompt":
        seqs = _spread(rng, 1, 32)
        tokens = _spread(rng, seqs, 16384)
        return dict(op=op, seqs=seqs, tokens=tokens, carried=rng.choice([0, seqs // 2, seqs]), heads=heads, dk=dk, dv=dv,
                    decay=decay)
    rows = _spread(rng, 1, 256)
    return dict(op=op, rows=rows, empty=rng.choice([0, rows // 8]), heads=heads, dk=dk, dv=dv, decay=decay,
                dtype=rng.choice(["bf16", "f16"]))


# ---------------------------------------------------------------------------------------------
# lengths: fixed by the case, in an order that the seed sets
# ---------------------------------------------------------------------------------------------
def _row_lengths(case):
    """Cached tokens of an attention case's rows, the new one counted; -1 for an empty slot."""
    n, lo, hi = case["rows"], case["min_len"], case["max_len"]
    got = [max(lo, min(hi, int(round(lo * (hi / lo) ** ((i + 0.5) / n))))) for i in range(n)]
    if n > 1:
        got[0], got[-1] = lo, hi
    for i in range(case["empty"]):
        got[(i * n) // case["empty"]] = -1
    return got


def _ragged(total, parts):
    """`total` split into `parts` sizes that fall off from long ones to short ones, one of them 0 if there are many."""
    weights = [1.0 / (1 + i) for i in range(parts)]
    if parts > 8:
        weights[parts // 2] = 0.0
    scale = total / sum(weights)
    sizes = [int(w * scale) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def _new_tokens(case):
    return _ragged(case["tokens"], case["seqs"]) if case["tokens"] else [1] * case["seqs"]


def _visible(length, window, sink):
    if length <= 0 or not window or length <= window:
        return max(0, length)
    return window


def _page_table(lengths, page_tokens, rng, device):
    """Pages for sequences of these lengths, handed out in a shuffled order as a long-running server has them."""
    need = [-(-max(0, n) // page_tokens) for n in lengths]
    ids = list(range(sum(need)))
    rng.shuffle(ids)
    table = np.full((len(lengths), max(1, max(need))), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at : at + n]
        at += n
    return torch.from_numpy(table).to(device), max(1, len(ids))


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _starts(sizes):
    return [0] + [int(x) for x in np.cumsum(sizes)]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    rng = random.Random(int(seed))
    return {"append": _prepare_append, "attention": _prepare_attention, "prompt": _prepare_prompt,
            "step": _prepare_step}[case["op"]](case, dev, gen, rng)


def _randn(shape, dtype, dev, gen):
    return torch.randn(shape, dtype=torch.float32, device=dev, generator=gen).to(dtype) if math.prod(shape) < 1 << 26 \
        else torch.randn(shape, dtype=dtype, device=dev, generator=gen)


def _prepare_append(case, dev, gen, rng):
    dtype, d, h, kv, p = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"], case["page_tokens"]
    new = _new_tokens(case)
    rng.shuffle(new)
    cached = [rng.randint(0, case["context"]) for _ in new]
    total = sum(new)
    table, pages = _page_table([c + n for c, n in zip(cached, new)], p, rng, dev)
    # the pools have pages for every sequence's full context, as a server sets them up once
    pages = max(pages, case["seqs"] * (-(-case["context"] // p)) + -(-total // p))
    positions = max(c + n for c, n in zip(cached, new))
    angle = torch.arange(positions, device=dev, dtype=torch.float32)[:, None] * ROPE_BASE ** (
        -torch.arange(0, case["rotary_dim"], 2, device=dev, dtype=torch.float32) / case["rotary_dim"])
    # queries, keys and values as one projection leaves them: slices of its rows
    fused = _randn((total, (h + 2 * kv) * d), dtype, dev, gen)
    q, k, v = fused[:, : h * d], fused[:, h * d : (h + kv) * d], fused[:, (h + kv) * d :]
    return dict(case=case, q=q.view(total, h, d), k=k.view(total, kv, d), v=v.view(total, kv, d), cos=angle.cos(),
                sin=angle.sin(), k_pool=_randn((pages, kv, p, d), dtype, dev, gen),
                v_pool=_randn((pages, kv, p, d), dtype, dev, gen), table=table, lengths=_ints(cached, dev),
                starts=_ints(_starts(new), dev))


def _prepare_attention(case, dev, gen, rng):
    dtype, d, h, kv, p = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"], case["page_tokens"]
    lengths = _row_lengths(case)
    rng.shuffle(lengths)
    table, pages = _page_table(lengths, p, rng, dev)
    return dict(case=case, q=_randn((case["rows"], h, d), dtype, dev, gen) * 1.5,
                k_pool=_randn((pages, kv, p, d), dtype, dev, gen), v_pool=_randn((pages, kv, p, d), dtype, dev, gen),
                table=table, lengths=_ints(lengths, dev))


def _decays(case, tokens, dev, gen):
    """Logarithms of the decays: a constant for each head that spreads memories from tens to thousands of tokens, or a
    gate's for each token and head, from a hardly felt decay to one that forgets nearly all."""
    h = case["heads"]
    if case["decay"] == "head":
        return torch.log1p(-torch.exp2(-5.0 - 6.0 * torch.arange(h, device=dev, dtype=torch.float32) / h))
    gate = torch.randn((tokens, h), device=dev, generator=gen) * 2.0 - 3.0
    return -torch.nn.functional.softplus(gate)


def _projected(case, tokens, dtype, dev, gen):
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    fused = _randn((tokens, h * (2 * dk + dv)), dtype, dev, gen)
    q, k, v = fused[:, : h * dk], fused[:, h * dk : 2 * h * dk], fused[:, 2 * h * dk :]
    return q.view(tokens, h, dk), k.view(tokens, h, dk), v.view(tokens, h, dv)


def _prepare_prompt(case, dev, gen, rng):
    new = _ragged(case["tokens"], case["seqs"])
    rng.shuffle(new)
    n, total = case["seqs"], sum(new)
    q, k, v = _projected(case, total, torch.bfloat16, dev, gen)
    slots = list(range(n + 3))
    rng.shuffle(slots)
    cached = [17] * case["carried"] + [0] * (n - case["carried"])
    rng.shuffle(cached)
    return dict(case=case, q=q, k=k, v=v, decay=_decays(case, total, dev, gen), slots=_ints(slots[:n], dev),
                lengths=_ints(cached, dev), starts=_ints(_starts(new), dev), longest=max(new),
                state=torch.randn((n + 3, case["heads"], case["dk"], case["dv"]), device=dev, generator=gen))


def _prepare_step(case, dev, gen, rng):
    n = case["rows"]
    q, k, v = _projected(case, n, DTYPES[case["dtype"]], dev, gen)
    slots = list(range(n + 2))
    rng.shuffle(slots)
    slots = slots[:n]
    for i in range(case["empty"]):
        slots[(i * n) // case["empty"]] = -1
    live = torch.tensor([r for r, slot in enumerate(slots) if slot >= 0], device=dev)
    return dict(case=case, q=q, k=k, v=v, decay=_decays(case, n, dev, gen), slots=_ints(slots, dev), live=live,
                state=torch.randn((n + 2, case["heads"], case["dk"], case["dv"]), device=dev, generator=gen))


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "prompt": _own_prompt, "step": _own_step}[op](state)
    return {"append": _plain_append, "attention": _plain_attention, "prompt": _plain_prompt,
            "step": _plain_step}[op](state)


def _own_append(s):
    paged_kv, _ = _package()
    pools = paged_kv.PagedKVPools(s["k_pool"], s["v_pool"])
    q = paged_kv.append_kv(pools, s["table"], s["lengths"], s["starts"], s["k"], s["v"], q=s["q"], cos=s["cos"],
                           sin=s["sin"], interleaved=s["case"]["interleaved"])
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_attention(s):
    paged_kv, _ = _package()
    c = s["case"]
    pools = paged_kv.PagedKVPools(s["k_pool"], s["v_pool"])
    out, lse = paged_kv.paged_attention(pools, s["table"], s["lengths"], s["q"], logit_softcap=c["softcap"] or None,
                                        window_size=c["window"] or None, sink_tokens=c["sink"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_prompt(s):
    _, linear = _package()
    out = linear.linear_attention_prefill(s["state"], s["slots"], s["lengths"], s["starts"], s["q"], s["k"], s["v"],
                                          s["decay"])
    return {"out": out, "state": s["state"]}


def _own_step(s):
    _, linear = _package()
    out = linear.linear_attention_step(s["state"], s["slots"], s["q"], s["k"], s["v"], s["decay"])
    return {"out": out, "state": s["state"]}


def _rotate(x, cos, sin, interleaved):
    """The rotation of the first dims of each head; cos and sin [tokens, 1, pairs]."""
    pairs = cos.shape[-1]
    x = x.float()
    turn, rest = x[..., : 2 * pairs], x[..., 2 * pairs :]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turn[..., :pairs], turn[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s):
    c, p = s["case"], s["case"]["page_tokens"]
    rows = torch.arange(s["k"].shape[0], device=s["k"].device)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), rows.int(), right=True)
    pos = s["lengths"][seq].long() + rows - s["starts"][seq].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    page, at = s["table"][seq, pos // p].long(), pos % p
    dtype = s["k"].dtype
    s["k_pool"][page, :, at] = _rotate(s["k"], cos, sin, c["interleaved"]).to(dtype)
    s["v_pool"][page, :, at] = s["v"]
    return {"q": _rotate(s["q"], cos, sin, c["interleaved"]).to(dtype), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attention(s):
    c = s["case"]
    rows, h, d = s["q"].shape
    kv, p = c["kv_heads"], c["page_tokens"]
    table = s["table"].long().clamp(min=0)
    n = table.shape[1] * p
    k = s["k_pool"][table].transpose(1, 2).reshape(rows, kv, n, d).float()  # [rows, pages, kv, p, d] before
    v = s["v_pool"][table].transpose(1, 2).reshape(rows, kv, n, d).float()
    q = s["q"].view(rows, kv, h // kv, d).float()
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    at, length = torch.arange(n, device=q.device)[None], s["lengths"][:, None]
    seen = at < length
    if c["window"]:
        sink = min(c["sink"], c["window"])
        seen = seen & ((at < sink) | (at >= length - (c["window"] - sink)))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    v = v * seen[:, None, :, None]
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))
    return {"out": out.reshape(rows, h, d).to(s["q"].dtype), "lse": lse.reshape(rows, h)}


def _plain_prompt(s):
    """Chunks of all sequences side by side; the states between chunks by one product with the decays between them."""
    c = s["case"]
    n, h, dk, dv = c["seqs"], c["heads"], c["dk"], c["dv"]
    chunks = -(-s["longest"] // CHUNK)
    start, size = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    at = torch.arange(chunks * CHUNK, device=start.device)
    real = at[None] < size[:, None]
    row = torch.where(real, start[:, None] + at[None], 0)

    def laid_out(x):  # [tokens, h, ...] -> [n, h, chunks, CHUNK, ...], zero beyond a sequence's end
        x = x[row].float() * real.view(n, -1, *([1] * (x.dim() - 1)))
        return x.view(n, chunks, CHUNK, *x.shape[2:]).movedim(3, 1)

    g = s["decay"] if s["decay"].dim() == 2 else s["decay"].expand(s["q"].shape[0], h)
    q, k, v, g = laid_out(s["q"]), laid_out(s["k"]), laid_out(s["v"]), laid_out(g)
    b = g.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device=b.device).tril().bool()
    gap = (b[..., :, None] - b[..., None, :]).masked_fill(~lower, -math.inf)
    out = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * torch.exp(gap), v)
    own_part = torch.matmul((k * torch.exp(b[..., -1:] - b)[..., None]).transpose(-1, -2), v)
    # the decay from the end of chunk j up to the start of chunk i, summed from chunk j on: a difference of two sums from
    # the sequence's start would lose what a long sequence's sums have in common
    later = torch.ones(chunks + 1, chunks, device=b.device).tril(-1).bool()
    whole = torch.nn.functional.pad(b[..., -1], (1, 0))
    gap = (whole[..., :, None] * later.tril(-2)).cumsum(-2).masked_fill(~later, -math.inf)
    between = torch.matmul(torch.exp(gap), own_part.flatten(-2)).view(n, h, chunks + 1, dk, dv)
    whole = whole.cumsum(-1)
    slots = s["slots"].long()
    first = s["state"][slots] * (s["lengths"] > 0).view(n, 1, 1, 1)
    between = between + torch.exp(whole)[..., None, None] * first[:, :, None]
    out = out + torch.exp(b)[..., None] * torch.matmul(q, between[:, :, :-1])
    out = (out / math.sqrt(dk)).movedim(1, 3).reshape(n, chunks * CHUNK, h, dv)
    rows = torch.arange(s["q"].shape[0], device=row.device)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), rows.int(), right=True)
    got = out[seq, rows - start[seq]].to(s["q"].dtype)
    last = torch.where((size > 0).view(n, 1, 1, 1), between[:, :, -1], s["state"][slots])
    s["state"][slots] = last
    return {"out": got, "state": s["state"]}


def _plain_step(s):
    live, slots = s["live"], s["slots"].long()[s["live"]]
    g = s["decay"][live] if s["decay"].dim() == 2 else s["decay"].expand(live.shape[0], -1)
    q, k, v = s["q"][live].float(), s["k"][live].float(), s["v"][live].float()
    new = torch.exp(g)[..., None, None] * s["state"][slots] + k[..., :, None] * v[..., None, :]
    s["state"].index_copy_(0, slots, new)
    got = torch.matmul(q[..., None, :], new)[..., 0, :] / math.sqrt(k.shape[-1])
    out = torch.zeros(s["v"].shape, dtype=s["q"].dtype, device=got.device).index_copy_(0, live, got.to(s["q"].dtype))
    return {"out": out, "state": s["state"]}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "append":
        d, h, kv, t = case["head_dim"], case["heads"], case["kv_heads"], sum(_new_tokens(case))
        values = t * (h + 2 * kv) * d
        turned = t * (h + kv) * case["rotary_dim"]
        return {"bytes": 2 * 2 * values + 2 * 4 * t * (case["rotary_dim"] // 2), "flops": 3 * turned}
    if op == "attention":
        d, h, kv = case["head_dim"], case["heads"], case["kv_heads"]
        seen = sum(_visible(n, case["window"], case["sink"]) for n in _row_lengths(case))
        return {"bytes": seen * kv * d * 2 * 2 + case["rows"] * h * (2 * d * 2 + 4), "flops": 4 * h * d * seen}
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    if op == "prompt":
        t, n = case["tokens"], case["seqs"]
        decays = 4 * t * h if case["decay"] == "token" else 4 * h
        return {"bytes": 2 * t * h * (2 * dk + 2 * dv) + decays + 4 * h * dk * dv * (n + case["carried"]),
                "flops": 4 * t * h * dk * dv}
    live = case["rows"] - case["empty"]
    return {"bytes": live * h * (8 * dk * dv + 2 * (2 * dk + 2 * dv) + (4 if case["decay"] == "token" else 0)),
            "flops": 5 * live * h * dk * dv}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "prompt": _exact_prompt,
            "step": _exact_step}[case["op"]](case, s)


def _turn_exact(x, cos, sin, interleaved):
    """Each pair as a complex number, times the rotation's."""
    x, pairs = x.double(), cos.shape[-1]
    first = torch.arange(0, 2 * pairs, 2, device=x.device) if interleaved else torch.arange(pairs, device=x.device)
    second = first + (1 if interleaved else pairs)
    turned = torch.complex(x[..., first], x[..., second]) * torch.complex(cos.double(), sin.double())[:, None]
    x[..., first], x[..., second] = turned.real, turned.imag
    return x


def _exact_append(case, s):
    p, starts, cached, table = case["page_tokens"], s["starts"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    k_pool, v_pool, q = s["k_pool"].double(), s["v_pool"].double(), torch.zeros_like(s["q"], dtype=torch.float64)
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        pos, row = cached[i], a
        while row < b:
            n = min(b - row, p - pos % p)
            cos, sin = s["cos"][pos : pos + n], s["sin"][pos : pos + n]
            q[row : row + n] = _turn_exact(s["q"][row : row + n], cos, sin, case["interleaved"])
            page, at = table[i][pos // p], pos % p
            k_pool[page, :, at : at + n] = _turn_exact(s["k"][row : row + n], cos, sin, case["interleaved"]).transpose(0, 1)
            v_pool[page, :, at : at + n] = s["v"][row : row + n].double().transpose(0, 1)
            row, pos = row + n, pos + n
    return {"q": q, "k_pool": k_pool, "v_pool": v_pool}


def _exact_attention(case, s):
    h, kv, p, d = case["heads"], case["kv_heads"], case["page_tokens"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=s["q"].device)
    table = s["table"].tolist()
    for r, n in enumerate(s["lengths"].tolist()):
        if n <= 0:
            continue
        seen = list(range(n))
        if case["window"] and n > case["window"]:
            sink = min(case["sink"], case["window"])
            seen = seen[:sink] + seen[n - (case["window"] - sink) :]
        seen = torch.tensor(seen, device=out.device)
        page = torch.tensor(table[r], device=out.device)[seen // p]
        for j in range(kv):
            k, v = s["k_pool"][page, j, seen % p].double(), s["v_pool"][page, j, seen % p].double()
            group = slice(j * h // kv, (j + 1) * h // kv)
            score = s["q"][r, group].double() @ k.T * d ** -0.5
            if case["softcap"]:
                score = case["softcap"] * torch.tanh(score / case["softcap"])
            lse[r, group] = torch.logsumexp(score, -1)
            out[r, group] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}


def _recurrence(state, g, q, k, v):
    """One token of all rows: the new states and their outputs."""
    state = torch.exp(g)[..., None, None] * state + k[..., :, None] * v[..., None, :]
    return state, (q[..., None] * state).sum(-2) * q.shape[-1] ** -0.5


def _exact_prompt(case, s):
    if s["longest"] * case["seqs"] * case["heads"] * case["dk"] * case["dv"] > 1 << 40:
        return None
    starts = s["starts"].tolist()
    size = [b - a for a, b in zip(starts, starts[1:])]
    order = sorted(range(case["seqs"]), key=lambda i: -size[i])
    first = torch.tensor([starts[i] for i in order], device=s["q"].device)
    slots = s["slots"].long()[order]
    state = s["state"].double()
    now = state[slots] * (s["lengths"][order] > 0).double().view(-1, 1, 1, 1)
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=now.device)
    g = s["decay"].double()
    for t in range(s["longest"]):
        n = sum(x > t for x in size)
        row = first[:n] + t
        now[:n], out[row] = _recurrence(now[:n], g[row] if g.dim() == 2 else g.expand(n, -1), s["q"][row].double(),
                                        s["k"][row].double(), s["v"][row].double())
    some = torch.tensor([size[i] > 0 for i in order], device=now.device)
    state[slots[some]] = now[some]
    return {"out": out, "state": state}


def _exact_step(case, s):
    state, out = s["state"].double(), torch.zeros(s["v"].shape, dtype=torch.float64, device=s["v"].device)
    g = s["decay"].double()
    rows = torch.tensor([r for r, slot in enumerate(s["slots"].tolist()) if slot >= 0], device=out.device)
    slots = s["slots"].long()[rows]
    state[slots], out[rows] = _recurrence(state[slots], g[rows] if g.dim() == 2 else g.expand(len(rows), -1),
                                          s["q"][rows].double(), s["k"][rows].double(), s["v"][rows].double())
    return {"out": out, "state": state}
