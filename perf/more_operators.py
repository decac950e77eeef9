"""Workloads of the operators that serve prompts and drafted tokens over a paged key/value cache.

Grouped-query layers answer a prompt chunk, or a tree of drafted tokens, over the pages that hold their keys and
values; drafted tokens are then checked against the target's probabilities, and what was accepted is kept:

  append         new keys and values into their pages, keys and queries normed by head and rotated on the way
  prompt         attention of prompt chunks over their pages (sliding window with sinks where a layer has one)
  tree           attention of trees of drafted tokens over their pages
  verify         drafted tokens accepted or rejected by given random numbers, and the next token drawn
  pages          the cache's content moved: accepted rows closed up (keep), pages copied for forks (copy)

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
EPS = 1e-6
SCORES = 1 << 27  # scores of the plain form held at a time


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asterlm-frontier_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from asterq import paged_kv, speculative

    return paged_kv, speculative


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the drafted tree of a few interactive requests: eight nodes each, where the launch is what counts
        dict(name="append 4 trees of 8", op="append", seqs=4, tokens=32, tree=True, context=1500, heads=16, kv_heads=4,
             head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", page_tokens=64),
        # prompt chunks of a few requests admitted together, ragged, on top of what they have cached
        dict(name="append ragged prompts", op="append", seqs=11, tokens=16387, tree=False, context=2048, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=64, interleaved=True, dtype="f16", page_tokens=64),
        # a short follow-up question in a chat: few rows over a cached conversation
        dict(name="prompt one of 150", op="prompt", seqs=1, tokens=150, min_context=1111, max_context=1111, heads=16,
             kv_heads=4, head_dim=128, dtype="bf16", page_tokens=64, window=0, sink=0, softcap=0.0),
        # prompts admitted together, ragged, in a layer with a sliding window whose first tokens stay visible
        dict(name="prompt 9 ragged with window", op="prompt", seqs=9, tokens=16393, min_context=0, max_context=4096,
             heads=16, kv_heads=8, head_dim=64, dtype="f16", page_tokens=16, window=1024, sink=4, softcap=0.0),
        # a chunk of a long document over what is cached of it: the matrix products' case
        dict(name="prompt 8192 over 24576", op="prompt", seqs=1, tokens=8192, min_context=24576, max_context=24576,
             heads=32, kv_heads=8, head_dim=128, dtype="bf16", page_tokens=512, window=0, sink=0, softcap=0.0),
        # the drafted tree of one interactive request: latency, the cache split over all SMs
        dict(name="tree one of 8", op="tree", seqs=1, nodes=8, min_context=2011, max_context=2011, heads=16, kv_heads=4,
             head_dim=128, dtype="bf16", page_tokens=64, window=0, sink=0, softcap=0.0),
        # an ordinary batch with trees of 16 nodes
        dict(name="tree 32 of 16", op="tree", seqs=32, nodes=16, min_context=500, max_context=8192, heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", page_tokens=64, window=0, sink=0, softcap=0.0),
        # wide trees over long contexts, sixteen query heads for each key/value head
        dict(name="tree 24 of 61 long", op="tree", seqs=24, nodes=61, min_context=2048, max_context=32768, heads=32,
             kv_heads=2, head_dim=128, dtype="f16", page_tokens=128, window=0, sink=0, softcap=0.0),
        # a chain of drafted tokens of a few requests, drafted greedily (no probabilities of the drafts)
        dict(name="verify 4 chains of 6", op="verify", seqs=4, nodes=6, tree=False, vocab=32000, drafted=False),
        # a full batch of drafted trees with the draft's probabilities, a large vocabulary
        dict(name="verify 96 trees of 12", op="verify", seqs=96, nodes=12, tree=True, vocab=128256, drafted=True),
        # a batch's accepted paths closed up behind their contexts, in all layers
        dict(name="pages keep of 48 trees", op="pages", kind="keep", layers=16, seqs=48, nodes=32, context=300,
             kv_heads=8, head_dim=128, dtype="bf16", page_tokens=64),
        # pages copied where forked sequences part, in all layers
        dict(name="pages copy of 60", op="pages", kind="copy", layers=24, pages=200, pairs=60, kv_heads=8, head_dim=128,
             dtype="f16", page_tokens=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = {"append": _draw_append, "prompt": _draw_prompt, "tree": _draw_tree, "verify": _draw_verify,
                "pages": _draw_pages}[rng.choice(["append", "prompt", "prompt", "tree", "tree", "verify", "pages"])](rng)
        if case is not None:
            return case


def _draw_append(rng):
    d, kv = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8])
    heads, seqs, tree = kv * rng.choice([1, 2, 3, 4, 8]), _spread(rng, 1, 64), rng.random() < 0.4
    tokens = seqs * rng.randint(2, 48) if tree else _spread(rng, seqs, 12000)
    context = _spread(rng, 1, 1500)
    if heads * tokens * d > 32 * 16000 * 128 or (seqs * (context + 64) + tokens) * kv * d > 1 << 28:
        return None
    return dict(op="append", seqs=seqs, tokens=tokens, tree=tree, context=context, heads=heads, kv_heads=kv, head_dim=d,
                rotary_dim=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.4,
                dtype=rng.choice(["bf16", "f16"]), page_tokens=rng.choice([16, 48, 64, 256, 512]))


def _window(rng):
    window = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
    return dict(window=window, sink=rng.choice([0, 4, 13]) if window else 0, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))


def _draw_prompt(rng):
    d, kv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    heads, seqs = kv * rng.choice([1, 2, 4, 7, 8]), _spread(rng, 1, 24)
    tokens, most = _spread(rng, seqs, 12000), _spread(rng, 1, 24576)
    case = dict(op="prompt", seqs=seqs, tokens=tokens, min_context=rng.choice([0, most // 8, most]), max_context=most,
                heads=heads, kv_heads=kv, head_dim=d, dtype=rng.choice(["bf16", "f16"]),
                page_tokens=rng.choice([16, 48, 64, 128, 512]), **_window(rng))
    if 4 * d * heads * tokens * (most + tokens) > 2e12 or seqs * most * kv * d > 1 << 28:
        return None
    return case


def _draw_tree(rng):
    d, kv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    group, seqs = rng.choice([1, 2, 4, 5, 8, 16]), _spread(rng, 1, 128)
    nodes, most = _spread(rng, 2, 100), _spread(rng, 1, 65536)
    if seqs * most * kv * d > 1 << 27 or seqs * nodes * kv * group * most * d > 24 * 61 * 32 * 16384 * 128:
        return None
    return dict(op="tree", seqs=seqs, nodes=nodes, min_context=max(1, most // rng.choice([1, 2, 16])), max_context=most,
                heads=kv * group, kv_heads=kv, head_dim=d, dtype=rng.choice(["bf16", "f16"]),
                page_tokens=rng.choice([16, 48, 64, 128, 512]), **_window(rng))


def _draw_verify(rng):
    seqs, nodes, vocab = _spread(rng, 1, 160), _spread(rng, 2, 64), _spread(rng, 100, 150000)
    if seqs * nodes * vocab > 96 * 12 * 128256:
        return None
    return dict(op="verify", seqs=seqs, nodes=nodes, tree=rng.random() < 0.6, vocab=vocab, drafted=rng.random() < 0.6)


def _draw_pages(rng):
    layers, kv, d, p = rng.randint(1, 32), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.choice([16, 48, 64, 256])
    case = dict(op="pages", layers=layers, kv_heads=kv, head_dim=d, dtype=rng.choice(["bf16", "f16"]), page_tokens=p)
    if rng.random() < 0.5:
        seqs, nodes, context = _spread(rng, 1, 128), _spread(rng, 2, 64), _spread(rng, 1, 500)
        pages, more = seqs * (-(-(context + nodes) // p)), dict(kind="keep", seqs=seqs, nodes=nodes, context=context)
    else:
        pairs = _spread(rng, 1, 120)
        pages = 3 * pairs + 5
        more = dict(kind="copy", pages=pages, pairs=pairs)
    return None if layers * pages * kv * p * d > 1 << 30 else {**case, **more}


# ---------------------------------------------------------------------------------------------
# sizes: fixed by the case, in an order that the seed sets
# ---------------------------------------------------------------------------------------------
def _ragged(total, parts):
    """`total` split into `parts` sizes that fall off from long ones to short ones, one of them 0 if there are many."""
    weights = [1.0 / (1 + i) for i in range(parts)]
    if parts > 8:
        weights[parts // 2] = 0.0
    scale = total / sum(weights)
    sizes = [int(w * scale) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def _contexts(case):
    """Cached tokens of the sequences, from the least to the most."""
    n, lo, hi = case["seqs"], case["min_context"], case["max_context"]
    got = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** ((i + 0.5) / n))) - 1 for i in range(n)]
    got[0], got[-1] = lo, hi
    return got


def _nodes(case):
    """Nodes of the sequences' trees: up to a quarter are smaller, as where a draft stopped early."""
    n = case["nodes"]
    return [n if i % 4 else max(1, n - i % (n // 2 + 1)) for i in range(case["seqs"])]


def _parents(n, chain, rng):
    """The parent of each node, -1 for the root: a chain, or a tree whose early nodes have several children."""
    if chain:
        return list(range(-1, n - 1))
    return [-1] + [max(0, min(i - 1, int(i * rng.random() ** 0.7 * 0.9))) for i in range(1, n)]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


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
    return {"append": _prepare_append, "prompt": _prepare_rows, "tree": _prepare_rows, "verify": _prepare_verify,
            "pages": _prepare_pages}[case["op"]](case, dev, gen, rng)


def _randn(shape, dtype, dev, gen):
    return torch.randn(shape, dtype=torch.float32, device=dev, generator=gen).to(dtype) if math.prod(shape) < 1 << 26 \
        else torch.randn(shape, dtype=dtype, device=dev, generator=gen)


def _prepare_append(case, dev, gen, rng):
    dtype, d, h, kv, p = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"], case["page_tokens"]
    new = [case["tokens"] // case["seqs"]] * case["seqs"] if case["tree"] else _ragged(case["tokens"], case["seqs"])
    rng.shuffle(new)
    cached = [rng.randint(0, case["context"]) for _ in new]
    total = sum(new)
    table, pages = _page_table([c + n for c, n in zip(cached, new)], p, rng, dev)
    # the pools have pages for every sequence's full context, as a server sets them up once
    pages = max(pages, case["seqs"] * (-(-case["context"] // p)) + -(-total // p))
    # a drafted node's position goes by its depth, a prompt's token's by its row
    at = [c + j for c, n in zip(cached, new) for j in (_depths(_parents(n, False, rng)) if case["tree"] else range(n))]
    positions = max(c + n for c, n in zip(cached, new))
    angle = torch.arange(positions, device=dev, dtype=torch.float32)[:, None] * ROPE_BASE ** (
        -torch.arange(0, case["rotary_dim"], 2, device=dev, dtype=torch.float32) / case["rotary_dim"])
    # queries, keys and values as one projection leaves them: slices of its rows
    fused = _randn((total, (h + 2 * kv) * d), dtype, dev, gen) * 1.3
    q, k, v = fused[:, : h * d], fused[:, h * d : (h + kv) * d], fused[:, (h + kv) * d :]
    return dict(case=case, q=q.view(total, h, d), k=k.view(total, kv, d), v=v.view(total, kv, d), cos=angle.cos(),
                sin=angle.sin(), q_norm=1 + 0.2 * torch.randn(d, device=dev, generator=gen),
                k_norm=1 + 0.2 * torch.randn(d, device=dev, generator=gen), positions=_ints(at, dev) if case["tree"] else None,
                k_pool=_randn((pages, kv, p, d), dtype, dev, gen), v_pool=_randn((pages, kv, p, d), dtype, dev, gen),
                table=table, lengths=_ints(cached, dev), starts=_ints(_starts(new), dev))


def _new_rows(case):
    return _ragged(case["tokens"], case["seqs"]) if case["op"] == "prompt" else _nodes(case)


def _prepare_rows(case, dev, gen, rng):
    dtype, d, h, kv, p = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"], case["page_tokens"]
    both = list(zip(_contexts(case), _new_rows(case)))
    rng.shuffle(both)
    cached, new = [c for c, _ in both], [n for _, n in both]
    total = sum(new)
    table, pages = _page_table([c + n for c, n in both], p, rng, dev)
    state = dict(case=case, q=_randn((total, h, d), dtype, dev, gen) * 1.5, cached=cached, new=new,
                 k_pool=_randn((pages, kv, p, d), dtype, dev, gen), v_pool=_randn((pages, kv, p, d), dtype, dev, gen),
                 table=table, lengths=_ints(cached, dev), starts=_ints(_starts(new), dev))
    if case["op"] == "tree":
        state["parents"] = _ints([x for n in new for x in _parents(n, False, rng)], dev)
    return state


def _prepare_verify(case, dev, gen, rng):
    new = _nodes(case)
    rng.shuffle(new)
    rows, vocab = sum(new), case["vocab"]
    trees = [_parents(n, not case["tree"], rng) for n in new]
    # the target's distributions, and a draft's that are near them
    logits = torch.randn((rows, vocab), device=dev, generator=gen) * 2.5
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits.add_(torch.randn((rows, vocab), device=dev, generator=gen) * 0.7), -1)
    starts = _starts(new)
    above = torch.tensor([starts[s] + max(x, 0) for s, t in enumerate(trees) for x in t], device=dev)
    if case["drafted"]:  # each node's token is drawn from the draft's distribution at its parent
        pick = torch.rand((rows, 1), device=dev, generator=gen, dtype=torch.float64)
        sums = torch.cat([draft[above[i : i + 256]].double().cumsum(-1) for i in range(0, rows, 256)]) if rows * vocab < 1 << 24 \
            else None
        tokens = torch.searchsorted(sums, pick * sums[:, -1:]) if sums is not None else torch.cat(
            [torch.searchsorted(c, pick[i : i + 256] * c[:, -1:]) for i in range(0, rows, 256)
             for c in [draft[above[i : i + 256]].double().cumsum(-1)]])
        tokens = tokens[:, 0].clamp(max=vocab - 1)
    else:  # the draft's best token, its second best for a second child, and so on
        rank, seen = [], {}
        for s, t in enumerate(trees):
            for x in t:
                rank.append(seen.get((s, x), 0))
                seen[(s, x)] = rank[-1] + 1
        best = draft.topk(min(vocab, max(rank) + 1), -1).indices
        tokens = best[above, torch.tensor(rank, device=dev).clamp(max=best.shape[1] - 1)]
    return dict(case=case, target=target, draft=draft if case["drafted"] else None, tokens=tokens.int(), new=new,
                parents=None if not case["tree"] else _ints([x for t in trees for x in t], dev), starts=_ints(starts, dev),
                accept=torch.rand(rows, device=dev, generator=gen), sample=torch.rand(case["seqs"], device=dev, generator=gen))


def _prepare_pages(case, dev, gen, rng):
    dtype, shape = DTYPES[case["dtype"]], (case["kv_heads"], case["page_tokens"], case["head_dim"])
    state = dict(case=case)
    if case["kind"] == "keep":
        new = _nodes(case)
        cached = [rng.randint(0, case["context"]) for _ in new]
        state["table"], pages = _page_table([c + n for c, n in zip(cached, new)], case["page_tokens"], rng, dev)
        pages = max(pages, case["seqs"] * (-(-(case["context"] + case["nodes"]) // case["page_tokens"])))
        kept, count = [], []
        for n in new:  # a path from the root down, as long as a verification leaves it
            path, parents = [0], _parents(n, False, rng)
            for i in range(1, n):
                if parents[i] == path[-1] and rng.random() < 0.8:
                    path.append(i)
            count.append(len(path))
            kept += path + [-1] * (n - len(path))
        state.update(lengths=_ints(cached, dev), starts=_ints(_starts(new), dev), kept=_ints(kept, dev), count=_ints(count, dev))
    else:
        pages = case["pages"]
        ids = list(range(pages))
        rng.shuffle(ids)
        n = case["pairs"]
        # the pages of the forks are free ones; one page may have several copies
        state["pairs"] = _ints([[rng.choice(ids[n:]), ids[i]] for i in range(n)], dev)
    state["k_pools"], state["v_pools"] = ([_randn((pages, *shape), dtype, dev, gen) for _ in range(case["layers"])] for _ in range(2))
    if own:  # a server makes the stack of its layers once
        paged_kv, _ = _package()
        state["stack"] = paged_kv.PagedKVStack([paged_kv.PagedKVPools(k, v) for k, v in zip(state["k_pools"], state["v_pools"])])
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "prompt": _own_prompt, "tree": _own_tree, "verify": _own_verify,
                "pages": _own_pages}[op](state)
    return {"append": _plain_append, "prompt": _plain_rows, "tree": _plain_rows, "verify": _plain_verify,
            "pages": _plain_pages}[op](state)


def _own_append(s):
    paged_kv, _ = _package()
    pools = paged_kv.PagedKVPools(s["k_pool"], s["v_pool"])
    q = paged_kv.append_kv(pools, s["table"], s["lengths"], s["starts"], s["k"], s["v"], q=s["q"], cos=s["cos"],
                           sin=s["sin"], interleaved=s["case"]["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                           norm_eps=EPS, positions=s["positions"])
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _layer(c):
    return dict(logit_softcap=c["softcap"] or None, window_size=c["window"] or None, sink_tokens=c["sink"], return_lse=True)


def _own_prompt(s):
    paged_kv, _ = _package()
    pools = paged_kv.PagedKVPools(s["k_pool"], s["v_pool"])
    out, lse = paged_kv.paged_prompt_attention(pools, s["table"], s["lengths"], s["starts"], s["q"], **_layer(s["case"]))
    return {"out": out, "lse": lse}


def _own_tree(s):
    paged_kv, _ = _package()
    pools = paged_kv.PagedKVPools(s["k_pool"], s["v_pool"])
    out, lse = paged_kv.paged_tree_attention(pools, s["table"], s["lengths"], s["starts"], s["parents"], s["q"],
                                             **_layer(s["case"]))
    return {"out": out, "lse": lse}


def _own_verify(s):
    _, speculative = _package()
    kept, count, token = speculative.verify_drafts(s["target"], s["tokens"], s["starts"], s["parents"], s["accept"],
                                                   s["sample"], draft_probs=s["draft"])
    return {"kept": kept, "count": count, "token": token}


def _own_pages(s):
    paged_kv, _ = _package()
    if s["case"]["kind"] == "keep":
        paged_kv.keep_kv_rows(s["stack"], s["table"], s["lengths"], s["starts"], s["kept"], s["count"])
    else:
        paged_kv.copy_kv_pages(s["stack"], s["pairs"])
    return {"k": s["k_pools"], "v": s["v_pools"]}


def _rotate(x, cos, sin, interleaved):
    """The rotation of the first dims of each head; cos and sin [tokens, 1, pairs]."""
    pairs = cos.shape[-1]
    turn, rest = x[..., : 2 * pairs], x[..., 2 * pairs :]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turn[..., :pairs], turn[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _plain_append(s):
    c, p = s["case"], s["case"]["page_tokens"]
    rows = torch.arange(s["k"].shape[0], device=s["k"].device)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), rows.int(), right=True)
    place = s["lengths"][seq].long() + rows - s["starts"][seq].long()
    at = place if s["positions"] is None else s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    page, inside = s["table"][seq, place // p].long(), place % p
    dtype = s["k"].dtype
    s["k_pool"][page, :, inside] = _rotate(_normed(s["k"], s["k_norm"]), cos, sin, c["interleaved"]).to(dtype)
    s["v_pool"][page, :, inside] = s["v"]
    return {"q": _rotate(_normed(s["q"], s["q_norm"]), cos, sin, c["interleaved"]).to(dtype), "k_pool": s["k_pool"],
            "v_pool": s["v_pool"]}


def _ancestors(parents):
    """[n, n]: whether column j is row i or above it in the tree, and the rows' depths."""
    n = parents.shape[0]
    seen = torch.eye(n + 1, device=parents.device)
    seen[torch.arange(n, device=parents.device), torch.where(parents < 0, n, parents).long()] = 1.0
    for _ in range(max(1, (n - 1).bit_length())):  # steps of one, two, four, .. generations
        seen = (torch.matmul(seen, seen) > 0).float()
    seen = seen[:n, :n] > 0
    return seen, seen.sum(-1) - 1


def _plain_rows(s):
    """Sequence by sequence, as many rows at a time as the scores' memory allows."""
    c = s["case"]
    total, h, d = s["q"].shape
    kv, p = c["kv_heads"], c["page_tokens"]
    sink = min(c["sink"], c["window"])
    out = torch.empty_like(s["q"])
    lse = torch.empty((total, h), dtype=torch.float32, device=out.device)
    row = 0
    for i, (cached, new) in enumerate(zip(s["cached"], s["new"])):
        n = cached + new
        pages = s["table"][i, : -(-n // p)].long()
        k = s["k_pool"][pages].transpose(0, 1).reshape(kv, -1, d)[:, :n].float()
        v = s["v_pool"][pages].transpose(0, 1).reshape(kv, -1, d)[:, :n].float()
        key = torch.arange(n, device=out.device)
        if c["op"] == "tree":
            seen, depth = _ancestors(s["parents"][row : row + new])
            position = cached + depth
            key_at = torch.cat((key[:cached], position))
            tree = torch.cat((torch.ones((new, cached), dtype=torch.bool, device=out.device), seen), 1)
        else:
            position, key_at, tree = cached + torch.arange(new, device=out.device), key, None
        step = max(1, SCORES // (h * n)) if new else 1
        for a in range(0, new, step):
            b = min(new, a + step)
            q = s["q"][row + a : row + b].float().view(b - a, kv, h // kv, d).permute(1, 2, 0, 3)
            score = torch.matmul(q, k.transpose(1, 2)[:, None]) / math.sqrt(d)  # [kv, group, rows, n]
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            at = position[a:b, None]
            visible = key_at <= at
            if c["window"]:
                visible = visible & ((key_at < sink) | (key_at > at - (c["window"] - sink)))
            if tree is not None:
                visible = visible & tree[a:b]
            score = score.masked_fill(~visible, -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = torch.exp(score - top)
            all_ = weight.sum(-1, keepdim=True)
            got = torch.matmul(weight, v[:, None]) / all_
            out[row + a : row + b] = got.permute(2, 0, 1, 3).reshape(b - a, h, d).to(out.dtype)
            lse[row + a : row + b] = (top + torch.log(all_)).squeeze(-1).permute(2, 0, 1).reshape(b - a, h)
        row += new
    return {"out": out, "lse": lse}


def _plain_verify(s):
    """All sequences side by side, node by node; what is left of the target after rejections, and its mass, in 64 bits:
    a random number next to a border between two tokens goes by their last bits."""
    new = torch.tensor(s["new"], device=s["tokens"].device)
    seqs, most, vocab = new.shape[0], max(s["new"]), s["target"].shape[1]
    start = s["starts"][:-1].long()
    each = torch.arange(seqs, device=new.device)
    cur = torch.zeros(seqs, dtype=torch.long, device=new.device)
    count = torch.ones_like(cur)
    kept = torch.full((s["tokens"].shape[0] + 1,), -1, dtype=torch.int32, device=new.device)
    kept[start] = 0
    left, mass = s["target"][start].double(), torch.ones(seqs, dtype=torch.float64, device=new.device)
    for i in range(1, most):
        row = torch.where(i < new, start + i, 0)
        above = torch.full_like(cur, i - 1) if s["parents"] is None else s["parents"][row].long()
        tried = (i < new) & (above == cur)
        token = s["tokens"][row].long()
        chance = left[each, token]
        if s["draft"] is None:
            drafted = torch.ones_like(mass)
        else:
            q = s["draft"][start + cur]
            drafted = q[each, token].double()
        taken = tried & (s["accept"][row].double() * drafted * mass < chance)
        lost = tried & ~taken
        if s["draft"] is None:
            left[each, token] = torch.where(lost, 0.0, chance)
            mass = torch.where(lost, mass - chance, mass)
        else:
            rest = (left - mass[:, None] * q.double()).clamp_(min=0)
            more = rest.sum(-1)
            none = lost & (more == 0)  # nothing is left: the target itself
            left = torch.where((lost & ~none)[:, None], rest, left)
            left = torch.where(none[:, None], s["target"][start + cur].double(), left)
            mass = torch.where(none, 1.0, torch.where(lost, more, mass))
        cur = torch.where(taken, i, cur)
        kept[torch.where(taken, start + count, kept.shape[0] - 1)] = i
        kept[-1] = -1
        count += taken
        left = torch.where(taken[:, None], s["target"][start + cur].double(), left)
        mass = torch.where(taken, 1.0, mass)
    sums = left.cumsum(-1)
    token = (sums <= s["sample"].double()[:, None] * sums[:, -1:]).sum(-1).clamp(max=vocab - 1)
    return {"kept": kept[:-1], "count": count.int(), "token": token.int()}


def _plain_pages(s):
    c, p = s["case"], s["case"]["page_tokens"]
    if c["kind"] == "keep":
        rows = torch.arange(s["kept"].shape[0], device=s["kept"].device)
        seq = torch.searchsorted(s["starts"][1:].contiguous(), rows.int(), right=True)
        place, length = rows - s["starts"][seq].long(), s["lengths"][seq].long()
        live = place < s["count"][seq]
        seq, to, source = seq[live], (length + place)[live], (length + s["kept"].long())[live]
        to_page, from_page = s["table"][seq, to // p].long(), s["table"][seq, source // p].long()
        for pool in s["k_pools"] + s["v_pools"]:
            pool[to_page, :, to % p] = pool[from_page, :, source % p]
    else:
        source, to = s["pairs"].long().unbind(1)
        for pool in s["k_pools"] + s["v_pools"]:
            pool[to] = pool[source]
    return {"k": s["k_pools"], "v": s["v_pools"]}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _pairs(cached, new, window, sink):
    """Visible (query, key) pairs of a prompt chunk, and its keys that some query sees."""
    if not window:
        return cached * new + new * (new + 1) // 2, cached + new
    sink = min(sink, window)
    recent = window - sink
    at = np.arange(cached, cached + new, dtype=np.int64)
    pairs = np.minimum(at + 1, window)
    first = max(0, cached + 1 - recent)
    return int(pairs.sum()), cached + new - first + min(sink, first)


def work(case):
    op = case["op"]
    if op == "append":
        rows, d = case["tokens"], case["head_dim"]
        heads = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": 4 * rows * heads * d + 4 * rows * case["rotary_dim"], "flops": 8 * rows * heads * d}
    if op in ("prompt", "tree"):
        pairs = keys = rows = 0
        for cached, new in zip(_contexts(case), _new_rows(case)):
            if op == "prompt":
                a, b = _pairs(cached, new, case["window"], case["sink"])
            else:  # the nodes above one another are few beside the cached tokens
                a, b = new * (min(cached, case["window"] or cached) + 1), min(cached, case["window"] or cached) + new
            pairs, keys, rows = pairs + a, keys + b, rows + new
        d = case["head_dim"]
        return {"bytes": 4 * keys * case["kv_heads"] * d + rows * case["heads"] * (4 * d + 4),
                "flops": 4 * pairs * case["heads"] * d}
    if op == "verify":
        # one distribution a sequence to draw from, and the draft's where a token may have been rejected
        each = 8 if case["drafted"] else 4
        return {"bytes": case["seqs"] * (each * case["vocab"] + 24 * case["nodes"]), "flops": 3 * case["seqs"] * case["vocab"]}
    row = 2 * case["kv_heads"] * case["head_dim"] * 2 * case["layers"]  # keys and values of a token in all layers
    tokens = 4 * case["seqs"] if case["kind"] == "keep" else case["pairs"] * case["page_tokens"]
    return {"bytes": 2 * tokens * row, "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] in ("prompt", "tree"):
        return _exact_rows(s)
    if case["op"] == "pages":
        return _exact_pages(s)
    return None  # whole numbers


def _exact_append(s):
    c, p = s["case"], s["case"]["page_tokens"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    place = np.concatenate([np.arange(a, a + y - x) for a, x, y in zip(lengths, starts, starts[1:])]).astype(np.int64)
    seq = np.repeat(np.arange(len(lengths)), np.diff(starts))
    page = torch.from_numpy(s["table"].cpu().numpy()[seq, place // p]).long().cuda()
    at = torch.from_numpy(place % p).cuda()
    turn = torch.from_numpy(place).cuda() if s["positions"] is None else s["positions"].long()
    phase = torch.complex(s["cos"].double(), s["sin"].double())[turn][:, None]
    n = c["rotary_dim"]

    def turned(x, weight):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
        left = x[..., :n]
        z = torch.view_as_complex(left.unflatten(-1, (-1, 2)).contiguous()) if c["interleaved"] else \
            torch.complex(left[..., : n // 2].contiguous(), left[..., n // 2 :].contiguous())
        z = z * phase
        left = torch.view_as_real(z).flatten(-2) if c["interleaved"] else torch.cat((z.real, z.imag), -1)
        return torch.cat((left, x[..., n:]), -1)

    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    k_pool[page, :, at] = turned(s["k"], s["k_norm"])
    v_pool[page, :, at] = s["v"].double()
    return {"q": turned(s["q"], s["q_norm"]), "k_pool": k_pool, "v_pool": v_pool}


def _exact_rows(s):
    """A key/value head at a time, over the keys of each sequence in the order of their positions."""
    c = s["case"]
    total, h, d = s["q"].shape
    kv, p, group = c["kv_heads"], c["page_tokens"], h // c["kv_heads"]
    out = torch.zeros((total, h, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((total, h), dtype=torch.float64, device="cuda")
    reach = c["window"] - min(c["sink"], c["window"])
    row = 0
    for i, (cached, new) in enumerate(zip(s["cached"], s["new"])):
        n = cached + new
        where = torch.arange(n, device="cuda")
        page = s["table"][i].long()[where // p]
        if c["op"] == "tree":
            up = s["parents"][row : row + new].tolist()
            line = np.zeros((new, new), bool)  # line[i, j]: j is i or above it
            for j in range(new):
                if up[j] >= 0:
                    line[j] = line[up[j]]
                line[j, j] = True
            position = torch.from_numpy(cached + line.sum(1) - 1).cuda()
            line = torch.from_numpy(line).cuda()
        else:
            position, line = torch.arange(cached, n, device="cuda"), None
        for g in range(kv):
            k, v = s["k_pool"][page, g, where % p].double(), s["v_pool"][page, g, where % p].double()
            for a in range(0, new, 512):
                rows = slice(a, min(new, a + 512))
                q = s["q"][row + a : row + rows.stop, g * group : (g + 1) * group].double()
                score = (q.reshape(-1, d) @ k.t()).view(rows.stop - a, group, n) * d ** -0.5
                if c["softcap"]:
                    score = torch.tanh(score / c["softcap"]) * c["softcap"]
                hidden = torch.zeros((rows.stop - a, n), dtype=torch.bool, device="cuda")
                if line is None:
                    hidden |= where[None] > position[rows, None]
                    if c["window"]:
                        hidden |= (position[rows, None] - where[None] >= reach) & (where[None] >= c["sink"])
                else:
                    hidden[:, cached:] = ~line[rows]
                    if c["window"]:
                        at = torch.cat((where[:cached], position))
                        hidden |= (position[rows, None] - at[None] >= reach) & (at[None] >= c["sink"])
                score[hidden[:, None].expand_as(score)] = -math.inf
                total_ = torch.logsumexp(score, -1)
                lse[row + a : row + rows.stop, g * group : (g + 1) * group] = total_
                weight = (score - total_[..., None]).exp_()
                out[row + a : row + rows.stop, g * group : (g + 1) * group] = (weight.view(-1, n) @ v).view(-1, group, d)
        row += new
    return {"out": out, "lse": lse}


def _exact_pages(s):
    c, p = s["case"], s["case"]["page_tokens"]
    pools = {"k": [x.clone() for x in s["k_pools"]], "v": [x.clone() for x in s["v_pools"]]}
    if c["kind"] == "keep":
        table, kept = s["table"].tolist(), s["kept"].tolist()
        moves = []
        for i, (start, length, count) in enumerate(zip(s["starts"].tolist(), s["lengths"].tolist(), s["count"].tolist())):
            for j in range(count):
                a, b = length + kept[start + j], length + j
                moves.append((table[i][a // p], a % p, table[i][b // p], b % p))
        fp, fa, tp, ta = (torch.tensor(x, device="cuda") for x in zip(*moves))
        old = {"k": s["k_pools"], "v": s["v_pools"]}
        for name, xs in pools.items():
            for x, y in zip(xs, old[name]):
                x.index_put_((tp[:, None], torch.arange(x.shape[1], device="cuda")[None], ta[:, None]),
                             y[fp[:, None], torch.arange(x.shape[1], device="cuda")[None], fa[:, None]])
    else:
        for xs, ys in ((pools["k"], s["k_pools"]), (pools["v"], s["v_pools"])):
            for x, y in zip(xs, ys):
                for a, b in s["pairs"].tolist():
                    x[b].copy_(y[a])
    return pools
