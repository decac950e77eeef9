"""Paged grouped-query keys and values: the attention layers beside the latent ones.

A hybrid model serves ordinary attention layers by the same sequence slots as its latent layers.
Their keys and values live in page pools (``PagedKVPools``) with int32 page tables and lengths on
the GPU:

* ``append_kv``: a step's or a prompt chunk's new keys and values at the end of each sequence,
  rotated by position on the way, with the rotated queries beside them (``asterq_kv_append``), their heads
  normed first and their positions given where asked (``asterq_kv_append_normed``);
* ``paged_attention``: one new token a sequence over its pages, the work split evenly over all SMs
  and joined in the same launch (``asterq_paged_attention``);
* ``paged_prompt_attention``, ``paged_tree_attention``: many new tokens a sequence, causal among themselves or
  nodes of a tree of drafted tokens (``asterq_rows_attention``);
* ``keep_kv_rows``, ``copy_kv_pages``: accepted rows closed up, pages copied, in all layers of a
  ``PagedKVStack`` (``asterq_kv_keep``, ``asterq_kv_copy_pages``);
* ``PagedKVBatch``: the pools of a stack of layers with the page tables they share, for a server that
  admits, steps, forks and removes sequences.

There is no backward pass: inputs that require a gradient are refused outside of ``torch.no_grad()``.
But for ``PagedKVBatch.accept`` nothing here waits for the GPU or reads from it, so all of it can be recorded in a CUDA graph.  A first
call on a stream, or ``workspace``, gives that stream's calls their workspace; a captured ``paged_attention``
without either has one of its own, zeroed at every replay (5 MB).  A captured call keeps its workspace wherever
its graph is replayed: graphs that overlap each other, or other calls of the stream, need one each.  A captured
``paged_prompt_attention`` or ``paged_tree_attention`` has one of its graph's own memory unless one is given (40 MB, shared by a
graph's calls one after the other).
"""
from __future__ import annotations

import math
from collections.abc import Sequence

import numpy as np
import torch

from . import _lib
from .batch import _PagePool

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_APPEND = _lib.packer(_lib.KvAppendParams)
_ATTEND = _lib.packer(_lib.PagedAttentionParams)
_ROWS = _lib.packer(_lib.RowsAttentionParams)
_NORMED = _lib.packer(_lib.KvAppendNormedParams)
_KEEP = _lib.packer(_lib.KvKeepParams)
_COPY = _lib.packer(_lib.KvCopyParams)
ATTENTION_HEAD_DIMS = (64, 128, 256)
MAX_TREE_NODES = 128


_quick_module = 0  # not looked for yet


def _quick():
    global _quick_module
    if _quick_module == 0:
        _quick_module = _lib.quick_calls()
    return _quick_module


class PagedKVPools:
    """Page pools of one layer: ``k`` and ``v`` [n_pages, n_kv_heads, page_tokens, head_dim], contiguous,
    bfloat16 or float16 on the GPU."""

    __slots__ = ("k", "v")

    def __init__(self, k: torch.Tensor, v: torch.Tensor) -> None:
        self.k, self.v = k, v
        quick = _quick()
        if quick is not None and quick.check_pools(k, v) is True:
            return
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [n_pages, n_kv_heads, page_tokens, head_dim]")
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise TypeError(f"pools of {k.dtype} and {v.dtype}: both bfloat16 or both float16")
        if not (k.is_cuda and v.device == k.device):
            raise RuntimeError("asterq caches live on the GPU; there is no CPU path")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("the pools must be contiguous")

    @staticmethod
    def empty(n_pages: int, n_kv_heads: int, page_tokens: int, head_dim: int, *, dtype=torch.bfloat16,
              device="cuda") -> "PagedKVPools":
        shape = (n_pages, n_kv_heads, page_tokens, head_dim)
        return PagedKVPools(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


class PagedAttentionWorkspace:
    """Device memory in which the pieces of sequences that several SMs share are joined.  One serves any
    sequence of calls on one stream; calls that overlap on the GPU need one each."""

    # the most any geometry needs: rows of 16 x 256 for two pieces a CTA, and a counter a piece
    def __init__(self, device="cuda") -> None:
        device = torch.device(device)
        p = _lib.PagedAttentionParams()
        p.dtype = p.out_dtype = _lib.DTYPE_BF16
        p.n_heads, p.n_kv_heads, p.head_dim, p.page_tokens = 16, 1, 256, 16
        with torch.cuda.device(device):
            self.nbytes = int(_lib.load().asterq_paged_attention_workspace_bytes(_lib.ctypes.byref(p)))
            self.buffer = torch.zeros(self.nbytes, dtype=torch.uint8, device=device)


_workspaces: dict[tuple[int, int], PagedAttentionWorkspace] = {}


def _capturing(device: torch.device) -> bool:
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _workspace(device: torch.device, stream: int) -> PagedAttentionWorkspace:
    """The workspace that calls on this stream share when the caller brings none."""
    ws = _workspaces.get((device.index, stream))
    if ws is None:
        ws = PagedAttentionWorkspace(device)
        if _capturing(device):
            return ws  # of the graph's own memory and zeroed when the graph runs: not for any call but this one
        ws = _workspaces.setdefault((device.index, stream), ws)  # another host thread's may have come first
    if _quick() is not None:  # whose calls come here until it knows the workspace
        _quick().workspace(0, device.index, stream, ws.buffer.data_ptr(), ws.nbytes)
    return ws


def _check_no_gradient(x: torch.Tensor, name: str) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, and there is no backward pass: call under torch.no_grad(), or "
                           "detach it")


def _check_rows(x: torch.Tensor, name: str, like: torch.Tensor, heads: int | None, dim: int) -> torch.Tensor:
    """[rows, heads, dim] of the pools' type whose rows and heads the kernels can read in 16-byte loads; a
    copy where they cannot."""
    if x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {dim}], got {tuple(x.shape)}")
    if x.dtype != like.dtype:
        raise TypeError(f"{name} is {x.dtype}, the pools are {like.dtype}")
    if x.device != like.device:
        raise RuntimeError(f"{name} is on {x.device}, the pools are on {like.device}")
    _check_no_gradient(x, name)
    row, head, one = x.stride()
    if one != 1 or (row | head) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _check_int(x: torch.Tensor, name: str, shape: tuple, like: torch.Tensor) -> None:
    if x.dtype != torch.int32 or x.shape != shape or not x.is_contiguous() or x.device != like.device:
        raise ValueError(f"{name} must be a contiguous int32 tensor {shape} on {like.device}, got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")


def _call(fn, packed: bytes, device: torch.device, stream: int) -> None:
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            status = fn(packed, stream)
    else:
        status = fn(packed, stream)
    if status:
        _lib.check(status)


def append_kv(
    pools: PagedKVPools,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    row_offsets: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    q_norm: torch.Tensor | None = None,
    k_norm: torch.Tensor | None = None,
    norm_eps: float = 1e-6,
    positions: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write new keys and values behind each sequence's cached tokens; returns the rotated queries.

    Rows ``row_offsets[s]`` .. ``row_offsets[s + 1]`` of k and v [rows, n_kv_heads, head_dim] (any row and
    head stride, so slices of a fused projection work) are sequence s's new tokens, at positions
    ``lengths[s]`` and on.  page_table int32 [n_seqs, max_pages], lengths int32 [n_seqs] (negative: an
    empty slot, whose rows are left out), row_offsets int32 [n_seqs + 1].  ``lengths`` is not advanced.

    cos, sin: float32 [positions, rotary_dim / 2]; the first ``rotary_dim`` dims of each head of k and q
    turn in pairs (j, j + rotary_dim / 2), or (2j, 2j + 1) when ``interleaved``.  Without them k and q
    are copied as they are.  q [rows, n_heads, head_dim] comes back rotated as a contiguous tensor
    (``q_out``, not overlapping q, if given); rows left out leave it unwritten.  status int32 [1]: set to
    1 when a row had no page in the table or no row in cos / sin and was left out.

    q_norm, k_norm [head_dim], float32 or the pools' type: each head x of q or k becomes x / sqrt(mean(x^2) + ``norm_eps``)
    times the weight before it turns, in float32.  positions int32 [rows]: the rows of cos and sin, where a row's position
    is not its place behind the cached tokens (a drafted node's is ``lengths[s]`` and its depth).
    """
    quick = _quick()
    if quick is not None:
        done = quick.append(pools.k, pools.v, page_table, lengths, row_offsets, k, v, q, cos, sin, interleaved, q_out, status,
                            q_norm, k_norm, norm_eps, positions)
        if done is not NotImplemented:
            return done
    n_kv, page, dim = pools.k.shape[1:]
    if row_offsets.dim() != 1 or page_table.dim() != 2:
        raise ValueError("page_table must be [n_seqs, max_pages] and row_offsets [n_seqs + 1]")
    n_seqs, max_pages = page_table.shape
    k = _check_rows(k, "k", pools.k, n_kv, dim)
    v = _check_rows(v, "v", pools.k, n_kv, dim)
    rows = k.shape[0]
    if v.shape[0] != rows:
        raise ValueError(f"k has {rows} rows, v has {v.shape[0]}")
    _check_int(page_table, "page_table", (n_seqs, max_pages), pools.k)
    _check_int(lengths, "lengths", (n_seqs,), pools.k)
    _check_int(row_offsets, "row_offsets", (n_seqs + 1,), pools.k)
    if status is not None:
        _check_int(status, "status", (1,), pools.k)
    heads = q_ptr = q_row = q_head = 0
    out_ptr = None
    if q is not None:
        q = _check_rows(q, "q", pools.k, None, dim)
        if q.shape[0] != rows:
            raise ValueError(f"k has {rows} rows, q has {q.shape[0]}")
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.device != q.device or not q_out.is_contiguous():
            raise ValueError("q_out must be a contiguous tensor of q's shape and type")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        q_row, q_head, _ = q.stride()
    elif q_out is not None:
        raise ValueError("q_out without q")
    rotary = positions_n = 0
    cos_ptr = sin_ptr = None
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or sin.shape != cos.shape or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous [positions, rotary_dim / 2]")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != k.device or sin.device != k.device:
            raise TypeError("cos and sin must be float32 on the pools' device")
        positions_n, rotary = cos.shape[0], 2 * cos.shape[1]
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    k_row, k_head, _ = k.stride()
    v_row, v_head, _ = v.stride()
    device = pools.k.device
    if q_norm is not None or k_norm is not None or positions is not None:
        norm_dtype = _DTYPES[k.dtype]
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is None:
                continue
            if w.shape != (dim,) or not w.is_contiguous() or w.device != device:
                raise ValueError(f"{name} must be a contiguous tensor ({dim},) on {device}")
            if w.dtype != torch.float32 and w.dtype != k.dtype:
                raise TypeError(f"{name} is {w.dtype}: float32 or the pools' type")
            _check_no_gradient(w, name)
            norm_dtype = _lib.DTYPE_F32 if w.dtype == torch.float32 else norm_dtype
        if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
            raise TypeError("q_norm and k_norm must be of one type")
        if q_norm is not None and q is None:
            raise ValueError("q_norm without q")
        if not norm_eps >= 0:
            raise ValueError("norm_eps must not be negative")
        if positions is not None:
            _check_int(positions, "positions", (rows,), pools.k)
            if cos is None:
                raise ValueError("positions without cos and sin")
        _call(_lib.load().asterq_kv_append_normed,
              _NORMED.pack(_DTYPES[k.dtype], norm_dtype, n_seqs, heads, n_kv, dim, rotary, 1 if interleaved else 0, page,
                           max_pages, norm_eps, 0, rows, pools.k.shape[0], positions_n, q_row, q_head, k_row, k_head,
                           v_row, v_head, q_ptr or 0, k.data_ptr(), v.data_ptr(), _lib.ptr(q_norm) or 0,
                           _lib.ptr(k_norm) or 0, cos_ptr or 0, sin_ptr or 0, _lib.ptr(positions) or 0,
                           page_table.data_ptr(), lengths.data_ptr(), row_offsets.data_ptr(), out_ptr or 0,
                           pools.k.data_ptr(), pools.v.data_ptr(), 0 if status is None else status.data_ptr()),
              device, torch.cuda.current_stream(device).cuda_stream)
        return q_out
    _call(_lib.load().asterq_kv_append,
          _APPEND.pack(_DTYPES[k.dtype], n_seqs, heads, n_kv, dim, rotary, 1 if interleaved else 0, page, max_pages, 0,
                       rows, pools.k.shape[0], positions_n, q_row, q_head, k_row, k_head, v_row, v_head, q_ptr or 0,
                       k.data_ptr(), v.data_ptr(), cos_ptr or 0, sin_ptr or 0, page_table.data_ptr(),
                       lengths.data_ptr(), row_offsets.data_ptr(), out_ptr or 0, pools.k.data_ptr(),
                       pools.v.data_ptr(), 0 if status is None else status.data_ptr()),
          device, torch.cuda.current_stream(device).cuda_stream)
    return q_out


def paged_attention(
    pools: PagedKVPools,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    q: torch.Tensor,
    *,
    n_new: int = 0,
    softmax_scale: float | None = None,
    logit_softcap: float | None = None,
    window_size: int | None = None,
    sink_tokens: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    workspace: PagedAttentionWorkspace | None = None,
    status: torch.Tensor | None = None,
):
    """Attention of one new token a sequence over its pages: out [n_seqs, n_heads, head_dim], and with
    ``return_lse`` the scores' log-sum-exp, float32 [n_seqs, n_heads], beside it.

    q [n_seqs, n_heads, head_dim] (any row and head stride); query head h reads kv head
    ``h // (n_heads // n_kv_heads)``.  Sequence s has ``lengths[s] + n_new`` tokens: n_new = 1 when the
    step's token has been appended and ``lengths`` not advanced yet.  Slots with a negative length, or no
    tokens, get zeros and a log-sum-exp of -inf.  ``window_size`` keeps the first ``sink_tokens`` and the
    newest ``window_size - sink_tokens`` tokens (the trim rule of the latent cache).  Scores are
    ``softmax_scale`` (1 / sqrt(head_dim)) q . k, softcapped to ``logit_softcap`` if given.  ``out``: the
    queries' type, or float32 good to some 2^-17 of the values (weights enter as two 16-bit parts).  Infinities
    and NaN in visible values reach their dim as in the formula, in other places of the pages nothing.  A sequence longer than its row of the table ends with it.  status int32 [1]: set
    to 1 when a needed page id was outside the pool.
    """
    quick = _quick()
    if quick is not None and workspace is None and window_size != 0:
        done = quick.attend(pools.k, pools.v, page_table, lengths, q, n_new, window_size or 0, sink_tokens,
                            pools.k.shape[3] ** -0.5 if softmax_scale is None else softmax_scale, logit_softcap or 0.0,
                            out, return_lse, status)
        if done is not NotImplemented:
            return done
    if q.dim() != 3 or page_table.dim() != 2:
        raise ValueError("q must be [n_seqs, n_heads, head_dim] and page_table [n_seqs, max_pages]")
    n_pages, n_kv, page, dim = pools.k.shape
    q = _check_rows(q, "q", pools.k, None, dim)
    rows, heads, _ = q.shape
    if heads % n_kv:
        raise ValueError(f"{heads} query heads over {n_kv} kv heads")
    max_pages = page_table.shape[1]
    _check_int(page_table, "page_table", (rows, max_pages), pools.k)
    _check_int(lengths, "lengths", (rows,), pools.k)
    if status is not None:
        _check_int(status, "status", (1,), pools.k)
    if n_new < 0 or sink_tokens < 0:
        raise ValueError("n_new and sink_tokens must not be negative")
    if window_size is not None and window_size <= 0:
        raise ValueError("window_size must be positive")
    dtype = _DTYPES[q.dtype]
    out_dtype = dtype
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.device != q.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of q's shape")
        out_dtype = _lib.DTYPE_F32 if out.dtype == torch.float32 else _DTYPES.get(out.dtype, -1)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if return_lse else None
    device = q.device
    stream = torch.cuda.current_stream(device).cuda_stream
    ws = _workspace(device, stream) if workspace is None else workspace
    q_row, q_head, _ = q.stride()
    _call(_lib.load().asterq_paged_attention,
          _ATTEND.pack(dtype, out_dtype, rows, heads, n_kv, dim, page, max_pages, n_new, window_size or 0, sink_tokens,
                       1.0 / math.sqrt(dim) if softmax_scale is None else softmax_scale, logit_softcap or 0.0, 0,
                       n_pages, q_row, q_head, q.data_ptr(), pools.k.data_ptr(), pools.v.data_ptr(),
                       page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                       ws.buffer.data_ptr(), ws.nbytes, 0 if status is None else status.data_ptr()),
          device, stream)
    return (out, lse) if return_lse else out


class RowsAttentionWorkspace:
    """Device memory in which ``paged_prompt_attention`` and ``paged_tree_attention`` join the pieces of work that
    several SMs share (some 40 MB); its contents are of one call.  One serves any sequence of calls on one stream;
    calls that overlap on the GPU need one each."""

    def __init__(self, device="cuda") -> None:
        device = torch.device(device)
        p = _lib.RowsAttentionParams()
        p.dtype = p.out_dtype = _lib.DTYPE_BF16
        p.n_heads, p.n_kv_heads, p.page_tokens = 1, 1, 16
        with torch.cuda.device(device):
            self.nbytes = 0
            for p.head_dim in ATTENTION_HEAD_DIMS:
                self.nbytes = max(self.nbytes, int(_lib.load().asterq_rows_attention_workspace_bytes(_lib.ctypes.byref(p))))
            self.buffer = torch.empty(self.nbytes, dtype=torch.uint8, device=device)


_rows_workspaces: dict[tuple[int, int], RowsAttentionWorkspace] = {}


def _rows_workspace(device: torch.device, stream: int) -> RowsAttentionWorkspace:
    if _capturing(device):
        return RowsAttentionWorkspace(device)  # of the graph's own memory: graphs may run beside each other and other calls
    ws = _rows_workspaces.get((device.index, stream))
    if ws is None:
        # another host thread's may have come first
        ws = _rows_workspaces.setdefault((device.index, stream), RowsAttentionWorkspace(device))
    if _quick() is not None:  # whose calls come here until it knows the workspace
        _quick().workspace(2, device.index, stream, ws.buffer.data_ptr(), ws.nbytes)
    return ws


def _rows_attention(pools, page_table, lengths, row_offsets, parents, q, softmax_scale, logit_softcap, window_size,
                    sink_tokens, out, return_lse, workspace, status, active_seqs):
    quick = _quick()
    if quick is not None and workspace is None and window_size != 0:
        done = quick.rows(pools.k, pools.v, page_table, lengths, row_offsets, parents, q,
                          1.0 / math.sqrt(pools.k.shape[3]) if softmax_scale is None else softmax_scale, logit_softcap or 0.0,
                          window_size or 0, sink_tokens, out, return_lse, status, active_seqs or 0)
        if done is not NotImplemented:
            return done
    if q.dim() != 3 or page_table.dim() != 2 or row_offsets.dim() != 1:
        raise ValueError("q must be [rows, n_heads, head_dim], page_table [n_seqs, max_pages], row_offsets [n_seqs + 1]")
    n_pages, n_kv, page, dim = pools.k.shape
    q = _check_rows(q, "q", pools.k, None, dim)
    if min(q.stride()) <= 0 and q.numel():
        q = q.clone(memory_format=torch.contiguous_format)  # heads or rows that repeat
    rows, heads, _ = q.shape
    if heads == 0 or heads % n_kv:
        raise ValueError(f"{heads} query heads over {n_kv} kv heads")
    n_seqs, max_pages = page_table.shape
    _check_int(page_table, "page_table", (n_seqs, max_pages), pools.k)
    _check_int(lengths, "lengths", (n_seqs,), pools.k)
    _check_int(row_offsets, "row_offsets", (n_seqs + 1,), pools.k)
    if parents is not None:
        _check_int(parents, "parents", (rows,), pools.k)
    if status is not None:
        _check_int(status, "status", (1,), pools.k)
    if sink_tokens < 0:
        raise ValueError("sink_tokens must not be negative")
    if window_size is not None and window_size <= 0:
        raise ValueError("window_size must be positive")
    if active_seqs is not None and active_seqs < 0:
        raise ValueError("active_seqs must not be negative")
    dtype = _DTYPES[q.dtype]
    out_dtype = dtype
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.device != q.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of q's shape")
        _check_no_gradient(out, "out")
        out_dtype = _lib.DTYPE_F32 if out.dtype == torch.float32 else _DTYPES.get(out.dtype, -1)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if return_lse else None
    device = q.device
    stream = torch.cuda.current_stream(device).cuda_stream
    if rows and n_seqs:
        ws = _rows_workspace(device, stream) if workspace is None else workspace
        q_row, q_head, _ = q.stride()
        _call(_lib.load().asterq_rows_attention,
              _ROWS.pack(dtype, out_dtype, n_seqs, heads, n_kv, dim, page, max_pages, window_size or 0, sink_tokens,
                         1.0 / math.sqrt(dim) if softmax_scale is None else softmax_scale, logit_softcap or 0.0, rows,
                         n_pages, q_row, q_head, q.data_ptr(), pools.k.data_ptr(), pools.v.data_ptr(),
                         page_table.data_ptr(), lengths.data_ptr(), row_offsets.data_ptr(),
                         0 if parents is None else parents.data_ptr(), out.data_ptr(),
                         0 if lse is None else lse.data_ptr(), ws.buffer.data_ptr(), ws.nbytes,
                         0 if status is None else status.data_ptr(), active_seqs or 0, 0),
              device, stream)
    return (out, lse) if return_lse else out


def paged_prompt_attention(
    pools: PagedKVPools,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    row_offsets: torch.Tensor,
    q: torch.Tensor,
    *,
    softmax_scale: float | None = None,
    logit_softcap: float | None = None,
    window_size: int | None = None,
    sink_tokens: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    workspace: RowsAttentionWorkspace | None = None,
    status: torch.Tensor | None = None,
    active_seqs: int | None = None,
):
    """Attention of prompt chunks over their pages: out [rows, n_heads, head_dim], and with ``return_lse`` the scores'
    log-sum-exp, float32 [rows, n_heads], beside it.

    Rows ``row_offsets[s]`` .. ``row_offsets[s + 1]`` of q [rows, n_heads, head_dim] (any row and head stride) are
    sequence s's new tokens, whose keys and values ``append_kv`` has written and ``lengths`` does not count yet: token i
    has position ``lengths[s] + i`` and sees the positions up to its own.  With ``window_size`` it sees, of these, the
    first ``sink_tokens`` and the newest ``window_size - sink_tokens``.  Other arguments, types and values that are not
    finite as for ``paged_attention``, but weights enter their product rounded once to the pools' type (float16: to zero below
    2^-32 of the largest), so that outputs are good to that rounding of the values, also float32 ones.  Rows of empty slots get zeros and a log-sum-exp
    of -inf; rows of no sequence are not written.  status int32 [1]: set to 1 when a needed page id was outside the pool,
    a row's place behind the table (it gets zeros), or offsets are out of order (nothing is written then).

    ``active_seqs``: how many sequences have rows, where that is known.  It is for speed alone: the work is cut by
    the average of rows a sequence, and idle slots beside a long prompt make that small.  Outputs of different cuts differ by the
    rounding of float32 sums.
    """
    return _rows_attention(pools, page_table, lengths, row_offsets, None, q, softmax_scale, logit_softcap, window_size,
                           sink_tokens, out, return_lse, workspace, status, active_seqs)


def paged_tree_attention(
    pools: PagedKVPools,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    row_offsets: torch.Tensor,
    parents: torch.Tensor,
    q: torch.Tensor,
    *,
    softmax_scale: float | None = None,
    logit_softcap: float | None = None,
    window_size: int | None = None,
    sink_tokens: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    workspace: RowsAttentionWorkspace | None = None,
    status: torch.Tensor | None = None,
    active_seqs: int | None = None,
):
    """Attention of trees of drafted tokens over their pages, one tree a sequence of at most 128 nodes.

    parents int32 [rows]: the parent of each row among its sequence's rows (0: the first), before it, or -1 for a
    root.  A node sees the sequence's ``lengths[s]`` cached tokens, its ancestors and itself, and with a window of these
    the ones that the window of its position ``lengths[s] + depth`` shows.  Node i's key and value are at place
    ``lengths[s] + i`` of the pages (``append_kv`` with ``positions`` puts them there).  A parent out of range is taken as -1
    and sets ``status``; a tree of more nodes leaves the call undone with ``status`` 1.  Other arguments as for
    ``paged_prompt_attention``.
    """
    if parents is None:
        raise ValueError("parents must be int32 [rows]")
    return _rows_attention(pools, page_table, lengths, row_offsets, parents, q, softmax_scale, logit_softcap, window_size,
                           sink_tokens, out, return_lse, workspace, status, active_seqs)


class PagedKVStack:
    """The pools of a stack of layers that share page tables: one geometry, type and device, no pool twice.  It holds
    the pools' addresses for ``keep_kv_rows`` and ``copy_kv_pages``, which work on all layers at once."""

    __slots__ = ("layers", "like", "_k", "_v", "_k_address", "_v_address")

    def __init__(self, layers: Sequence[PagedKVPools]) -> None:
        self.layers = tuple(layers)
        if not self.layers:
            raise ValueError("a stack without layers")
        first = self.layers[0].k
        for pools in self.layers:
            if pools.k.shape != first.shape or pools.k.dtype != first.dtype or pools.k.device != first.device:
                raise ValueError(f"layers of {tuple(first.shape)} {first.dtype} on {first.device} and "
                                 f"{tuple(pools.k.shape)} {pools.k.dtype} on {pools.k.device}")
        address = [pools.k.data_ptr() for pools in self.layers] + [pools.v.data_ptr() for pools in self.layers]
        if first.numel() and len(set(address)) < len(address):
            raise ValueError("a pool is in the stack twice")
        n = len(self.layers)
        self._k = (_lib.ctypes.c_void_p * n)(*address[:n])
        self._v = (_lib.ctypes.c_void_p * n)(*address[n:])
        self._k_address, self._v_address = _lib.ctypes.addressof(self._k), _lib.ctypes.addressof(self._v)
        self.like = first


def keep_kv_rows(
    stack: PagedKVStack,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    row_offsets: torch.Tensor,
    kept: torch.Tensor,
    n_kept: torch.Tensor,
    *,
    status: torch.Tensor | None = None,
) -> None:
    """Close the accepted rows of drafts up behind the cached tokens, in all layers of a stack (one launch).

    kept int32 [rows] and n_kept int32 [n_seqs] as ``speculative.verify_drafts`` gives them: the keys and values at place
    ``lengths[s] + kept[row_offsets[s] + i]`` go to place ``lengths[s] + i``, for i < ``n_kept[s]``.  kept ascends within a
    sequence.  ``lengths`` is not advanced; empty slots are left out.  Sequences must not share a page that rows are moved
    in.  status int32 [1]: set to 1 when a sequence's kept does not ascend or leaves its rows, its offsets are out of order
    (the sequence is left as it is), or a place has no page (the row is left out).
    """
    quick = _quick()
    if quick is not None:
        done = quick.keep(stack.like, len(stack.layers), stack._k_address, stack._v_address, page_table, lengths, row_offsets,
                          kept, n_kept, status)
        if done is not NotImplemented:
            return
    if page_table.dim() != 2 or row_offsets.dim() != 1 or kept.dim() != 1:
        raise ValueError("page_table must be [n_seqs, max_pages], row_offsets [n_seqs + 1] and kept [rows]")
    n_seqs, max_pages = page_table.shape
    like = stack.like
    n_pages, n_kv, page, dim = like.shape
    _check_int(page_table, "page_table", (n_seqs, max_pages), like)
    _check_int(lengths, "lengths", (n_seqs,), like)
    _check_int(row_offsets, "row_offsets", (n_seqs + 1,), like)
    _check_int(kept, "kept", (kept.shape[0],), like)
    _check_int(n_kept, "n_kept", (n_seqs,), like)
    if status is not None:
        _check_int(status, "status", (1,), like)
    _call(_lib.load().asterq_kv_keep,
          _KEEP.pack(_DTYPES[like.dtype], len(stack.layers), n_seqs, n_kv, dim, page, max_pages, 0, kept.shape[0], n_pages,
                     stack._k_address, stack._v_address, page_table.data_ptr(),
                     lengths.data_ptr(), row_offsets.data_ptr(), kept.data_ptr(), n_kept.data_ptr(),
                     0 if status is None else status.data_ptr()),
          like.device, torch.cuda.current_stream(like.device).cuda_stream)


def copy_kv_pages(stack: PagedKVStack, pairs: torch.Tensor, *, status: torch.Tensor | None = None) -> None:
    """Copy pages in all layers of a stack (one launch): pairs int32 [n, 2], page ``pairs[i, 1]`` becomes a copy of page
    ``pairs[i, 0]``.  A pair with a negative entry is left out.  So is, with status int32 [1] set to 1, one with a page
    outside the pools, and every pair whose destination another pair names too or whose source another pair writes.
    Each pair is held against all others of the call for that, so thousands of pairs are better given in parts."""
    like = stack.like
    n_pages, n_kv, page, dim = like.shape
    if pairs.dim() != 2:
        raise ValueError("pairs must be [n, 2]")
    _check_int(pairs, "pairs", (pairs.shape[0], 2), like)
    if pairs.data_ptr() % 8:
        pairs = pairs.clone()
    if status is not None:
        _check_int(status, "status", (1,), like)
    _call(_lib.load().asterq_kv_copy_pages,
          _COPY.pack(_DTYPES[like.dtype], len(stack.layers), n_kv, dim, page, pairs.shape[0], n_pages,
                     stack._k_address, stack._v_address, pairs.data_ptr(),
                     0 if status is None else status.data_ptr()),
          like.device, torch.cuda.current_stream(like.device).cuda_stream)


class PagedKVBatch:
    """The paged keys and values of a stack of attention layers that share sequence slots.

    Slot s is row s of ``page_table`` and ``lengths``, which live on the GPU beside a host mirror that
    hands out pages ahead of need (sequences added or removed reach the GPU with the next step).  A decode step is ``begin_step`` once, then for each layer ``append``
    and ``attend`` with one row a slot (rows of idle slots are ignored, their outputs are zeros), then
    ``end_step`` (or ``abandon_step``, where it failed on the way).  A prompt chunk is ``begin_rows`` with the tokens each slot gets, ``append`` and
    ``attend_rows`` for each layer, ``end_step``.  A step of drafted tokens is ``begin_tree`` with the slots' trees,
    ``append`` and ``attend_rows`` for each layer, ``speculative.verify_drafts`` with the batch's ``row_offsets`` and ``parents``, and
    ``accept`` with what it kept.

    ``fork_sequence`` gives a slot that shares another's pages; a page that both hold is copied when one of them is about
    to write into it.  A slot holds its pages until it is removed or truncated, or ``release_behind_window`` gives up those that a
    window has passed.  ``compact_pages`` moves the pages in use to the front of the pools.
    """

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, *, max_seqs: int, max_tokens: int,
                 page_tokens: int = 64, pool_pages: int | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, interleaved: bool = False, window_size: int | None = None,
                 sink_tokens: int = 0, dtype=torch.bfloat16, device="cuda") -> None:
        if n_layers <= 0 or max_seqs <= 0 or max_tokens <= 0:
            raise ValueError("n_layers, max_seqs and max_tokens must be positive")
        if page_tokens <= 0 or page_tokens % 16:
            raise ValueError("page_tokens must be a positive multiple of 16")
        if head_dim not in ATTENTION_HEAD_DIMS:
            raise NotImplementedError(f"head_dim {head_dim}: the attention kernel reads {ATTENTION_HEAD_DIMS}")
        self.device = torch.device(device)
        self.page_tokens, self.max_tokens = page_tokens, max_tokens
        self.max_pages = -(-max_tokens // page_tokens)
        pool_pages = max_seqs * self.max_pages if pool_pages is None else pool_pages
        self.layers = [PagedKVPools.empty(pool_pages, n_kv_heads, page_tokens, head_dim, dtype=dtype, device=self.device)
                       for _ in range(n_layers)]
        self.cos, self.sin, self.interleaved = cos, sin, interleaved
        self.window_size, self.sink_tokens = window_size, sink_tokens
        self.stack = PagedKVStack(self.layers)
        self._free = _PagePool(pool_pages)
        self._users = np.zeros(pool_pages, np.int32)  # slots that hold each page
        self._held = [0] * max_seqs  # entries of each slot's row of the table
        self._length = np.full(max_seqs, -1, np.int32)
        self._table = np.full((max_seqs, self.max_pages), -1, np.int32)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.lengths = torch.full((max_seqs,), -1, **i32)
        self.page_table = torch.full((max_seqs, self.max_pages), -1, **i32)
        self._one_row = torch.arange(max_seqs + 1, **i32)  # a decode step's rows: row s is slot s
        self.row_offsets = self._one_row
        self._new = np.zeros(max_seqs, np.int32)
        self._active_rows = 0  # slots that have rows in the open step
        self._new_dev = torch.zeros(max_seqs, **i32)
        self._open = False
        self._tree = False
        self.parents = self.positions = None  # of an open step's drafted trees
        self._dirty = False
        self.status = torch.zeros(1, **i32)

    @property
    def max_seqs(self) -> int:
        return len(self._held)

    def length(self, slot: int) -> int:
        return int(self._length[slot])

    def active(self) -> np.ndarray:
        return np.nonzero(self._length >= 0)[0]

    def _upload(self) -> None:
        if self._dirty:
            # one copy each, staged through pinned memory that the allocator holds until it has run
            self.page_table.copy_(torch.from_numpy(self._table).pin_memory(), non_blocking=True)
            self.lengths.copy_(torch.from_numpy(self._length).pin_memory(), non_blocking=True)
            self._dirty = False

    def add_sequence(self, slot: int | None = None) -> int:
        """Open an empty sequence in a free slot (the given one, or the lowest)."""
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        if slot is None:
            free = np.nonzero(self._length < 0)[0]
            if not free.size:
                raise RuntimeError(f"all {self.max_seqs} sequence slots are in use")
            slot = int(free[0])
        elif not 0 <= slot < self.max_seqs or self._length[slot] >= 0:
            raise ValueError(f"slot {slot} is not free")
        self._length[slot] = 0
        self._dirty = True
        return slot

    def remove_sequence(self, slot: int) -> None:
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        if not 0 <= slot < self.max_seqs or self._length[slot] < 0:
            raise ValueError(f"slot {slot} holds no sequence")
        self._drop(slot, 0)
        self._length[slot] = -1

    def _drop(self, slot: int, first: int) -> None:
        """The slot's pages from entry ``first`` on are not held by it any more."""
        pages = self._table[slot, first : self._held[slot]]
        pages = pages[pages >= 0]
        self._users[pages] -= 1  # a slot holds a page once
        self._free.release(pages[self._users[pages] == 0].tolist())
        self._table[slot, first : self._held[slot]] = -1
        self._held[slot] = first
        self._dirty = True

    def fork_sequence(self, slot: int, into: int | None = None) -> int:
        """Open a sequence that has the tokens of ``slot``, in a free slot (the given one, or the lowest), by sharing its
        pages: nothing is copied until one of the two writes into a page that both hold."""
        if not 0 <= slot < self.max_seqs or self._length[slot] < 0:
            raise ValueError(f"slot {slot} holds no sequence")
        new = self.add_sequence(into)
        n = -(-int(self._length[slot]) // self.page_tokens)
        self._table[new, :n] = self._table[slot, :n]
        pages = self._table[new, :n]
        self._users[pages[pages >= 0]] += 1
        self._held[new] = n
        self._length[new] = self._length[slot]
        return new

    def truncate_sequence(self, slot: int, tokens: int) -> None:
        """Keep the first ``tokens`` tokens of a sequence; pages behind them are given up."""
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        if not 0 <= slot < self.max_seqs or self._length[slot] < 0:
            raise ValueError(f"slot {slot} holds no sequence")
        if not 0 <= tokens <= self._length[slot]:
            raise ValueError(f"slot {slot} has {self._length[slot]} tokens, not {tokens}")
        if self.window_size is not None and self._reach() > 1:  # else nothing of the window is among them
            first = max(0, tokens - self._reach() + 1)
            if (self._table[slot, first // self.page_tokens : -(-tokens // self.page_tokens)] < 0).any():
                raise ValueError(f"slot {slot}: a window behind {tokens} tokens needs pages that were given up")
        self._drop(slot, min(self._held[slot], -(-tokens // self.page_tokens)))
        self._length[slot] = tokens

    def _reach(self) -> int:
        return self.window_size - min(self.sink_tokens, self.window_size)

    def release_behind_window(self) -> int:
        """Give up the pages between the sink and what the window still shows; returns how many entries were."""
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        if self.window_size is None:
            return 0
        released = 0
        sink, page = min(self.sink_tokens, self.window_size), self.page_tokens
        for s in self.active():
            first = -(-sink // page)
            # tokens below it are passed; the next token's own page is not, also where a window shows nothing but the sink
            last = min(max(0, int(self._length[s]) - max(self._reach(), 1) + 1) // page, self._held[s])
            if last <= first:
                continue
            pages = self._table[s, first:last]
            pages = pages[pages >= 0]
            if pages.size:
                self._users[pages] -= 1
                self._free.release(pages[self._users[pages] == 0].tolist())
                self._table[s, first:last] = -1
                released += int(pages.size)
                self._dirty = True
        return released

    def compact_pages(self) -> int:
        """Move the pages in use to the front of the pools (one launch); returns their number."""
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        used = np.nonzero(self._users > 0)[0]
        n = int(used.size)
        source = used[used >= n]
        if source.size:
            target = np.nonzero(self._users[:n] == 0)[0]
            self._copy(np.stack((source, target), 1))
            to = np.arange(self._users.size, dtype=np.int32)
            to[source] = target
            self._table = np.where(self._table >= 0, to[self._table], -1).astype(np.int32)
            self._users[target] = self._users[source]
            self._users[source] = 0
            self._free.free = list(range(self._users.size - 1, n - 1, -1))
            self._dirty = True
        return n

    def _copy(self, pairs: np.ndarray) -> None:
        # no page is written by one pair and named by another, so they can go in parts
        pairs = torch.from_numpy(np.ascontiguousarray(pairs, np.int32)).pin_memory().to(self.device, non_blocking=True)
        for part in pairs.split(2048):
            copy_kv_pages(self.stack, part, status=self.status)

    def _begin(self, new: np.ndarray, one_row: bool) -> None:
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        want = np.where(new > 0, self._length + new, 0)
        if (want > self.max_tokens).any():
            raise ValueError(f"a sequence would pass {self.max_tokens} tokens")
        need = np.maximum(-(-want // self.page_tokens) - np.asarray(self._held), 0)
        # entries that a slot is about to write into: those that others hold too (the last of its holders keeps the page), and
        # those without a page
        shared, bare, users = [], [], {}
        for s in np.nonzero(new > 0)[0]:
            for at in range(int(self._length[s]) // self.page_tokens, min(self._held[s], -(-int(want[s]) // self.page_tokens))):
                page = int(self._table[s, at])
                if page < 0:
                    bare.append((int(s), at))
                    continue
                left = users.get(page, int(self._users[page]))
                if left > 1:
                    users[page] = left - 1
                    shared.append((int(s), at, page))
        wanted = int(need.sum()) + len(shared) + len(bare)
        pages = self._free.alloc(wanted) if wanted else []
        self._users[pages] = 1
        for s, at in bare:
            self._table[s, at] = pages.pop()
            self._dirty = True
        pairs = []
        for s, at, page in shared:
            self._users[page] -= 1
            self._table[s, at] = pages.pop()
            if at * self.page_tokens < self._length[s]:
                pairs.append((page, self._table[s, at]))
            self._dirty = True
        for s in np.nonzero(need > 0)[0]:
            at, n = self._held[s], int(need[s])
            self._table[s, at : at + n] = pages[:n]
            pages = pages[n:]
            self._held[s] = at + n
            self._dirty = True
        if pairs:
            self._copy(np.asarray(pairs, np.int32))
        self._upload()
        if one_row:
            self.row_offsets = self._one_row
        else:
            offsets = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
            self.row_offsets = torch.from_numpy(offsets).pin_memory().to(self.device, non_blocking=True)
        if not np.array_equal(new, self._new):
            self._new = new
            self._active_rows = int(np.count_nonzero(new))
            self._new_dev.copy_(torch.from_numpy(new).pin_memory(), non_blocking=True)
        self._open = True

    def begin_step(self) -> None:
        """Open a decode step: one new token for every sequence, row s for slot s."""
        self._begin((self._length >= 0).astype(np.int32), True)

    def begin_rows(self, slots: Sequence[int], tokens: Sequence[int]) -> None:
        """Open a prompt chunk: ``tokens[i]`` new tokens for slot ``slots[i]``; the rows of ``append`` are
        the slots' tokens in the order of the slots."""
        new = np.zeros(self.max_seqs, np.int32)
        for s, n in zip(slots, tokens, strict=True):
            if not 0 <= s < self.max_seqs or self._length[s] < 0 or n < 0 or new[s]:
                raise ValueError(f"slot {s}: {n} tokens")
            new[s] = n
        self._begin(new, False)

    def begin_tree(self, slots: Sequence[int], parents: Sequence[Sequence[int]]) -> None:
        """Open a step of drafted tokens: for slot ``slots[i]`` a tree whose node j's parent is ``parents[i][j]``, below j
        (-1 for node 0, the root: the token after the cached ones).  The rows are the slots' nodes in the order of the slots;
        ``parents`` and ``positions`` hold their parents and positions on the GPU."""
        new = np.zeros(self.max_seqs, np.int32)
        trees = {}
        for s, tree in zip(slots, parents, strict=True):
            if not 0 <= s < self.max_seqs or self._length[s] < 0 or s in trees or not 0 < len(tree) <= MAX_TREE_NODES:
                raise ValueError(f"slot {s}: a tree of {len(tree)} nodes (1 to {MAX_TREE_NODES})")
            if tree[0] != -1 or any(not 0 <= p < j for j, p in enumerate(tree) if j):
                raise ValueError(f"slot {s}: the first node is the root (-1), others have a parent before them")
            depth = []
            for p in tree:
                depth.append(0 if p < 0 else depth[p] + 1)
            trees[s] = (list(tree), depth)
            new[s] = len(tree)
        order = sorted(trees)
        flat = [p for s in order for p in trees[s][0]]
        at = [int(self._length[s]) + d for s in order for d in trees[s][1]]
        self._begin(new, False)
        both = torch.tensor([flat, at], dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)
        self.parents, self.positions = both[0], both[1]
        self._tree = True

    def append(self, layer: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, *,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               norm_eps: float = 1e-6) -> torch.Tensor | None:
        """The open step's keys and values into layer ``layer``'s pages; returns the rotated queries (of normed heads where
        weights are given)."""
        if not self._open:
            raise RuntimeError("no step is open: begin_step or begin_rows first")
        return append_kv(self.layers[layer], self.page_table, self.lengths, self.row_offsets, k, v, q=q, cos=self.cos,
                         sin=self.sin, interleaved=self.interleaved, q_norm=q_norm, k_norm=k_norm, norm_eps=norm_eps,
                         positions=self.positions if self._tree and self.cos is not None else None, status=self.status)

    def attend_rows(self, layer: int, q: torch.Tensor, **kw):
        """Attention of the open prompt chunk's or drafted trees' rotated queries over layer ``layer`` with their own tokens."""
        if not self._open or self.row_offsets is self._one_row:
            raise RuntimeError("no rows are open: begin_rows or begin_tree first")
        kw = dict(window_size=self.window_size, sink_tokens=self.sink_tokens, status=self.status,
                  active_seqs=self._active_rows, **kw)
        if self._tree:
            return paged_tree_attention(self.layers[layer], self.page_table, self.lengths, self.row_offsets, self.parents, q, **kw)
        return paged_prompt_attention(self.layers[layer], self.page_table, self.lengths, self.row_offsets, q, **kw)

    def accept(self, kept: torch.Tensor, n_kept: torch.Tensor) -> list[int]:
        """Close the open step of drafted tokens with what ``speculative.verify_drafts`` kept of it: the accepted rows are
        closed up behind the cached tokens in all layers and the sequences advance by them.  Returns the slots' numbers of
        accepted rows; waits for the GPU, since pages are handed out on the host."""
        if not self._open or self.row_offsets is self._one_row:
            raise RuntimeError("no drafted rows are open: begin_tree or begin_rows first")
        keep_kv_rows(self.stack, self.page_table, self.lengths, self.row_offsets, kept, n_kept, status=self.status)
        counts = n_kept.cpu().numpy()
        if (counts < 0).any() or (counts > self._new).any():
            raise ValueError("more rows kept than were drafted")
        self.lengths.add_(n_kept)
        self._length += counts
        self._close()
        return counts.tolist()

    def _close(self) -> None:
        self._open = self._tree = False
        self.parents = self.positions = None

    def attend(self, layer: int, q: torch.Tensor, **kw):
        """Attention of the open decode step's rotated queries over layer ``layer`` with its new token."""
        if not self._open or self.row_offsets is not self._one_row:
            raise RuntimeError("no decode step is open: begin_step first")
        return paged_attention(self.layers[layer], self.page_table, self.lengths, q, n_new=1,
                               window_size=self.window_size, sink_tokens=self.sink_tokens, status=self.status, **kw)

    def end_step(self) -> None:
        """Advance the sequences by the open step's tokens (one small launch; nothing is copied)."""
        if not self._open:
            raise RuntimeError("no step is open")
        if self._tree:
            raise RuntimeError("drafted tokens are open: accept or abandon_step")
        self.lengths.add_(self._new_dev)
        self._length += self._new
        self._close()

    def abandon_step(self) -> None:
        """Close the open step without advancing: the sequences stay as they were before it.  What it has appended is
        never read, and the next step's tokens go in its place; pages that it was handed stay with their slots."""
        if not self._open:
            raise RuntimeError("no step is open")
        self._close()

    def raise_if_failed(self) -> None:
        """Synchronize; raise if a row was left out or an attention did not finish."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError("asterq paged_kv: " + ("a row had no page or no position, or a page id was not valid"
                                                     if code == 1 else "a wait on the device ran out"))
