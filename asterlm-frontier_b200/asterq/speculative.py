"""Verification of drafted tokens: which nodes of a draft the target's probabilities accept, and the next token.

``verify_drafts`` walks each sequence's chain or tree of drafted tokens by given random numbers so that what it keeps and
draws is distributed as the target's own sampling (speculative sampling; a rejected token's siblings are tried against what
is left of the target).  ``paged_kv.PagedKVBatch.accept`` then keeps the accepted rows of the caches.

It calls ``asterq_verify_drafts``; nothing waits for the GPU or reads from it, so calls can be recorded in a CUDA graph.
"""
from __future__ import annotations

import torch

from . import _lib, paged_kv
from .paged_kv import _call, _check_int, _check_no_gradient

_PARAMS = _lib.packer(_lib.VerifyParams)
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _probs(x: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    if x.dim() != 2 or x.shape != like.shape:
        raise ValueError(f"{name} must be {tuple(like.shape)}, got {tuple(x.shape)}")
    if x.dtype != like.dtype:
        raise TypeError(f"{name} is {x.dtype}, target_probs is {like.dtype}")
    if x.device != like.device:
        raise RuntimeError(f"{name} is on {x.device}, target_probs on {like.device}")
    _check_no_gradient(x, name)
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _uniforms(x: torch.Tensor, name: str, n: int, like: torch.Tensor) -> None:
    if x.dtype != torch.float32 or x.shape != (n,) or not x.is_contiguous() or x.device != like.device:
        raise ValueError(f"{name} must be a contiguous float32 tensor ({n},) on {like.device}")


def verify_drafts(
    target_probs: torch.Tensor,
    tokens: torch.Tensor,
    row_offsets: torch.Tensor,
    parents: torch.Tensor | None,
    accept_uniforms: torch.Tensor,
    sample_uniforms: torch.Tensor,
    *,
    draft_probs: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted nodes of each sequence's draft, their number, and the next token.

    Rows ``row_offsets[s]`` .. ``row_offsets[s + 1]`` are sequence s's nodes, at most 1024.  Node 0 is the root: the last
    token that is accepted already.  tokens int32 [rows]; parents int32 [rows], each below its node's own number (-1 for the
    root), None for chains.  target_probs [rows, vocab] (float32, bfloat16 or float16, any row stride): the target's
    probabilities behind each node, which sum to 1.  draft_probs, like them: those that a node's children were drawn from, in
    the order of their numbers; None for drafts that were not drawn (the best tokens), which then count as certain.
    accept_uniforms float32 [rows] and sample_uniforms float32 [n_seqs]: random numbers in [0, 1).

    At node ``cur`` with what is left of its target, r (mass m; r = target, m = 1 at first), a child with token x is accepted if
    ``u draft[cur][x] m < r(x)``.  If not, r = max(r - m draft[cur], 0) and m its sum (without draft_probs r(x) = 0 and m
    goes down by it), and the next child is tried; where nothing is left, r is the target again.  The next token is
    the first whose running sum of r is above ``sample_uniforms[s]`` times all of it.  Sums are in 64 bits.

    Returns kept int32 [rows] (a sequence's accepted nodes from its first row on, the root first, -1 behind them), n_kept int32
    [n_seqs] (the root counted) and next_token int32 [n_seqs].  status int32 [1]: set to 1 by a token outside the
    vocabulary (never accepted), a parent out of range (never reached), a distribution without a positive sum (next token
    -1), offsets out of order or too many nodes (nothing is kept, next token -1).  kept of rows of no sequence is not written.
    """
    quick = paged_kv._quick()
    if quick is not None:
        done = quick.verify(target_probs, tokens, row_offsets, parents, accept_uniforms, sample_uniforms, draft_probs, status)
        if done is not NotImplemented:
            return done
    if target_probs.dim() != 2 or row_offsets.dim() != 1 or row_offsets.shape[0] < 1:
        raise ValueError("target_probs must be [rows, vocab] and row_offsets [n_seqs + 1]")
    if target_probs.dtype not in _DTYPES:
        raise TypeError(f"target_probs is {target_probs.dtype}: float32, bfloat16 or float16")
    if not target_probs.is_cuda:
        raise RuntimeError("asterq verifies on the GPU; there is no CPU path")
    rows, vocab = target_probs.shape
    if vocab == 0:
        raise ValueError("an empty vocabulary")
    n_seqs = row_offsets.shape[0] - 1
    target_probs = _probs(target_probs, "target_probs", target_probs)
    if draft_probs is not None:
        draft_probs = _probs(draft_probs, "draft_probs", target_probs)
    _check_int(tokens, "tokens", (rows,), target_probs)
    _check_int(row_offsets, "row_offsets", (n_seqs + 1,), target_probs)
    if parents is not None:
        _check_int(parents, "parents", (rows,), target_probs)
    _uniforms(accept_uniforms, "accept_uniforms", rows, target_probs)
    _uniforms(sample_uniforms, "sample_uniforms", n_seqs, target_probs)
    if status is not None:
        _check_int(status, "status", (1,), target_probs)
    device = target_probs.device
    kept = torch.empty(rows, dtype=torch.int32, device=device)
    n_kept = torch.empty(n_seqs, dtype=torch.int32, device=device)
    next_token = torch.empty(n_seqs, dtype=torch.int32, device=device)
    if n_seqs:
        _call(_lib.load().asterq_verify_drafts,
              _PARAMS.pack(_DTYPES[target_probs.dtype], n_seqs, vocab, 0, rows, target_probs.stride(0),
                           0 if draft_probs is None else draft_probs.stride(0), target_probs.data_ptr(),
                           0 if draft_probs is None else draft_probs.data_ptr(), tokens.data_ptr(),
                           0 if parents is None else parents.data_ptr(), row_offsets.data_ptr(), accept_uniforms.data_ptr(),
                           sample_uniforms.data_ptr(), kept.data_ptr(), n_kept.data_ptr(), next_token.data_ptr(),
                           0 if status is None else status.data_ptr()),
              device, torch.cuda.current_stream(device).cuda_stream)
    return kept, n_kept, next_token
