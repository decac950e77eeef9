"""Serving a small hybrid model: linear, grouped-query and latent attention layers by the same slots.

Two requests with prompts of different lengths are admitted and decoded together; a third joins while
they run, one leaves.  Each layer mixes tokens with one of the package's operators:

  linear   a fixed-size state a slot (asterq.linear_attention: prompt chunks, then single tokens)
  kv       keys and values in pages, rotated by position (asterq.paged_kv)
  latent   the compressed latent cache (asterq.batch.PagedLatentBatch)

and the projections around them are plain products of random bf16 weights.  At the end each request is
compared with the same model run over its whole text at once in fp32.

  python examples/hybrid_decode.py [--steps N]
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT / "asterlm-frontier_b200") not in sys.path:
    sys.path.insert(0, str(ROOT / "asterlm-frontier_b200"))

from asterq.batch import PagedLatentBatch  # noqa: E402
from asterq.linear_attention import linear_attention_prefill, linear_attention_step  # noqa: E402
from asterq.paged_kv import PagedKVBatch  # noqa: E402

WIDTH, HEADS, DIM, KV_HEADS, LATENT, ROPE = 256, 4, 64, 2, 512, 64
LATENT_HEADS = 16
LAYERS = ("linear", "linear", "kv", "linear", "latent")  # three linear layers to one that attends to all tokens
MAX_SEQS, MAX_TOKENS = 4, 512
BF16 = torch.bfloat16


def rotary_tables(device):
    angle = torch.arange(MAX_TOKENS, device=device)[:, None] * 10000.0 ** (-torch.arange(DIM // 2, device=device) / (DIM // 2))
    return angle.cos().contiguous(), angle.sin().contiguous()


class Weights:
    """Random projections of each layer, and how its inputs come out of them."""

    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, device=device, generator=g) / math.sqrt(rows)).to(BF16)

        widths = {"linear": HEADS * 3 * DIM + HEADS, "kv": (HEADS + 2 * KV_HEADS) * DIM,
                  "latent": LATENT_HEADS * (LATENT + ROPE) + LATENT + ROPE}
        outs = {"linear": HEADS * DIM, "kv": HEADS * DIM, "latent": LATENT_HEADS * LATENT}
        self.layers = [(kind, matrix(WIDTH, widths[kind]), matrix(outs[kind], WIDTH)) for kind in LAYERS]

    @staticmethod
    def split(kind, y):
        n = y.shape[0]
        if kind == "linear":
            q, k, v, gate = y.split([HEADS * DIM, HEADS * DIM, HEADS * DIM, HEADS], 1)
            decay = -torch.nn.functional.softplus(gate.float() - 3.0)
            return q.view(n, HEADS, DIM), k.view(n, HEADS, DIM), v.view(n, HEADS, DIM), decay
        if kind == "kv":
            q, k, v = y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1)
            return q.view(n, HEADS, DIM), k.view(n, KV_HEADS, DIM), v.view(n, KV_HEADS, DIM)
        q, qr, latent, rope = y.split([LATENT_HEADS * LATENT, LATENT_HEADS * ROPE, LATENT, ROPE], 1)
        return q.view(n, LATENT_HEADS, LATENT) / 8, qr.view(n, LATENT_HEADS, ROPE), latent, rope


def normed(x):
    """x at unit root mean square, each row: what a layer's projections read."""
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def causal(q, k, v, scale):
    """Plain attention of a whole text: q [n, h, d], k and v [n, kv, d], in fp32."""
    n, h = q.shape[:2]
    group = h // k.shape[1]
    k, v = (x.float().repeat_interleave(group, 1) for x in (k, v))
    score = torch.einsum("qhd,khd->hqk", q.float(), k) * scale
    score = score.masked_fill(torch.ones(n, n, device=q.device).triu(1).bool(), -math.inf)
    return torch.einsum("hqk,khd->qhd", score.softmax(-1), v)


def rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    c, s = cos[: x.shape[0], None], sin[: x.shape[0], None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


class Server:
    """The caches of all layers, by slot."""

    def __init__(self, weights, device):
        self.w, self.device = weights, device
        self.cos, self.sin = rotary_tables(device)
        self.kv = PagedKVBatch(LAYERS.count("kv"), KV_HEADS, DIM, max_seqs=MAX_SEQS, max_tokens=MAX_TOKENS, page_tokens=64,
                               cos=self.cos, sin=self.sin, device=device)
        self.states = [torch.empty(MAX_SEQS, HEADS, DIM, DIM, device=device) for _ in range(LAYERS.count("linear"))]
        self.latent = [PagedLatentBatch(LATENT_HEADS, max_seqs=MAX_SEQS, page_tokens=128, recent_tokens=128,
                                        max_cold_pages=8, device=device) for _ in range(LAYERS.count("latent"))]

    def _ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def admit(self, x):
        """Run a prompt [n, WIDTH] through the layers into a free slot; returns (slot, outputs)."""
        n, slot = x.shape[0], self.kv.add_sequence()
        self.kv.begin_rows([slot], [n])
        at = {kind: 0 for kind in LAYERS}
        for kind, w_in, w_out in self.w.layers:
            i, at[kind] = at[kind], at[kind] + 1
            parts = Weights.split(kind, normed(x) @ w_in)
            if kind == "linear":
                q, k, v, decay = parts
                y = linear_attention_prefill(self.states[i], self._ints([slot]), self._ints([0]), self._ints([0, n]), q, k, v,
                                             decay)
            elif kind == "kv":
                q, k, v = parts
                y = causal(self.kv.append(i, q, k, v), rotate(k, self.cos, self.sin).to(BF16), v, DIM**-0.5)
            else:
                q, qr, latent, rope = parts
                assert self.latent[i].add_sequence(latent.contiguous(), rope.contiguous()) == slot
                key = torch.cat((latent, rope), -1)[:, None]
                y = causal(torch.cat((q, qr), -1), key, latent[:, None], (LATENT + ROPE) ** -0.5)
            x = x + y.reshape(n, -1).to(BF16) @ w_out
        self.kv.end_step()
        return slot, x

    def step(self, x):
        """One token for every open slot: x [MAX_SEQS, WIDTH], row s for slot s (rows of free slots are ignored)."""
        self.kv.begin_step()  # brings the lengths on the GPU up to date
        open_slots = self.kv.lengths >= 0
        slots = torch.where(open_slots, torch.arange(MAX_SEQS, dtype=torch.int32, device=self.device), -1).int()
        at = {kind: 0 for kind in LAYERS}
        for kind, w_in, w_out in self.w.layers:
            i, at[kind] = at[kind], at[kind] + 1
            parts = Weights.split(kind, normed(x) @ w_in)
            if kind == "linear":
                q, k, v, decay = parts
                y = linear_attention_step(self.states[i], slots, q, k, v, decay)
            elif kind == "kv":
                y = self.kv.attend(i, self.kv.append(i, *parts))
            else:
                q, qr, latent, rope = (p.contiguous() for p in parts)
                y = self.latent[i].step(q, qr, latent, rope)
            # rows of free slots hold anything: kept out of the next layer's inputs
            x = x + torch.where(open_slots[:, None], y.reshape(MAX_SEQS, -1).to(BF16) @ w_out, 0)
        self.kv.end_step()
        return x

    def release(self, slot):
        self.kv.remove_sequence(slot)
        for layer in self.latent:
            layer.remove_sequence(slot)


def whole(weights, x, cos, sin):
    """The same model over a whole text at once, mixing in fp32."""
    for kind, w_in, w_out in weights.layers:
        n = x.shape[0]
        parts = Weights.split(kind, normed(x) @ w_in)
        if kind == "linear":
            q, k, v, decay = (p.float() for p in parts)
            state, rows = torch.zeros(HEADS, DIM, DIM, device=x.device), []
            for t in range(n):
                state = decay[t].exp()[:, None, None] * state + k[t][:, :, None] * v[t][:, None, :]
                rows.append((q[t][:, :, None] * state).sum(1) * DIM**-0.5)
            y = torch.stack(rows)
        elif kind == "kv":
            q, k, v = parts
            y = causal(rotate(q, cos, sin), rotate(k, cos, sin), v, DIM**-0.5)
        else:
            q, qr, latent, rope = parts
            y = causal(torch.cat((q, qr), -1), torch.cat((latent, rope), -1)[:, None], latent[:, None], (LATENT + ROPE) ** -0.5)
        x = x + y.reshape(n, -1).to(BF16) @ w_out
    return x


def main(steps=24):
    """Returns the largest relative error of a request's outputs against the whole-text run."""
    device = torch.device("cuda")
    torch.manual_seed(0)
    weights = Weights(device)
    server = Server(weights, device)
    inputs, outputs = {}, {}  # slot -> rows

    def admit(n):
        x = torch.randn(n, WIDTH, device=device).to(BF16)
        slot, y = server.admit(x)
        inputs[slot], outputs[slot] = [x], [y]

    def decode(count):
        for _ in range(count):
            x = torch.randn(MAX_SEQS, WIDTH, device=device).to(BF16)
            y = server.step(x)
            for s in inputs:
                inputs[s].append(x[s : s + 1])
                outputs[s].append(y[s : s + 1])

    def check(slot):
        want = whole(weights, torch.cat(inputs[slot]), server.cos, server.sin).float()
        got = torch.cat(outputs[slot]).float()
        error = float((got - want).norm() / want.norm())
        print(f"slot {slot}: {got.shape[0]} tokens, {len(outputs[slot]) - 1} of them decoded, relative error {error:.2e}")
        return error

    admit(150)
    admit(37)
    decode(steps)
    admit(65)  # joins while the others run
    decode(steps)
    errors = [check(0)]
    server.release(0)  # its slot and pages go to the next request
    del inputs[0], outputs[0]
    admit(20)
    decode(steps)
    errors += [check(s) for s in sorted(inputs)]
    server.kv.raise_if_failed()
    return max(errors)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=24)
    main(parser.parse_args().steps)
