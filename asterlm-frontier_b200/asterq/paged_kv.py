"""Paged grouped-query keys and values: the attention layers beside the latent ones.

A hybrid model serves ordinary attention layers by the same sequence slots as its latent layers.
Their keys and values live in page pools (``PagedKVPools``) with int32 page tables and lengths on
the GPU:

* ``append_kv``: a step's or a prompt chunk's new keys and values at the end of each sequence,
  rotated by position on the way, with the rotated queries beside them (``asterq_kv_append``);
* ``paged_attention``: one new token a sequence over its pages, the work split evenly over all SMs
  and joined in the same launch (``asterq_paged_attention``);
* ``PagedKVBatch``: the pools of a stack of layers with the page tables they share, for a server that
  admits, steps and removes sequences.

There is no backward pass: inputs that require a gradient are refused outside of ``torch.no_grad()``.
Nothing here waits for the GPU or reads from it, so all of it can be recorded in a CUDA graph.  A first
call on a stream, or ``workspace``, gives that stream's calls their workspace; a captured ``paged_attention``
without either has one of its own, zeroed at every replay (5 MB).  A captured call keeps its workspace wherever
its graph is replayed: graphs that overlap each other, or other calls of the stream, need one each.
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
ATTENTION_HEAD_DIMS = (64, 128, 256)


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
        _workspaces[(device.index, stream)] = ws
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
    """
    quick = _quick()
    if quick is not None:
        done = quick.append(pools.k, pools.v, page_table, lengths, row_offsets, k, v, q, cos, sin, interleaved, q_out, status)
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
    rotary = positions = 0
    cos_ptr = sin_ptr = None
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or sin.shape != cos.shape or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous [positions, rotary_dim / 2]")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != k.device or sin.device != k.device:
            raise TypeError("cos and sin must be float32 on the pools' device")
        positions, rotary = cos.shape[0], 2 * cos.shape[1]
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    k_row, k_head, _ = k.stride()
    v_row, v_head, _ = v.stride()
    device = pools.k.device
    _call(_lib.load().asterq_kv_append,
          _APPEND.pack(_DTYPES[k.dtype], n_seqs, heads, n_kv, dim, rotary, 1 if interleaved else 0, page, max_pages, 0,
                       rows, pools.k.shape[0], positions, q_row, q_head, k_row, k_head, v_row, v_head, q_ptr or 0,
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


class PagedKVBatch:
    """The paged keys and values of a stack of attention layers that share sequence slots.

    Slot s is row s of ``page_table`` and ``lengths``, which live on the GPU beside a host mirror that
    hands out pages ahead of need (sequences added or removed reach the GPU with the next step).  A decode step is ``begin_step`` once, then for each layer ``append``
    and ``attend`` with one row a slot (rows of idle slots are ignored, their outputs are zeros), then
    ``end_step`` (or ``abandon_step``, where it failed on the way).  A prompt chunk is ``begin_rows`` with the tokens each slot gets, ``append`` for each
    layer, ``end_step``; the prompt's own attention is the caller's.  A slot holds its pages until it is
    removed, also those that a window has passed.
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
        self._free = _PagePool(pool_pages)
        self._held = [0] * max_seqs  # pages of each slot
        self._length = np.full(max_seqs, -1, np.int32)
        self._table = np.full((max_seqs, self.max_pages), -1, np.int32)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.lengths = torch.full((max_seqs,), -1, **i32)
        self.page_table = torch.full((max_seqs, self.max_pages), -1, **i32)
        self._one_row = torch.arange(max_seqs + 1, **i32)  # a decode step's rows: row s is slot s
        self.row_offsets = self._one_row
        self._new = np.zeros(max_seqs, np.int32)
        self._new_dev = torch.zeros(max_seqs, **i32)
        self._open = False
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
        n = self._held[slot]
        self._free.release(self._table[slot, :n].tolist())
        self._table[slot] = -1
        self._held[slot] = 0
        self._length[slot] = -1
        self._dirty = True

    def _begin(self, new: np.ndarray, one_row: bool) -> None:
        if self._open:
            raise RuntimeError("a step is open: end_step first")
        want = np.where(new > 0, self._length + new, 0)
        if (want > self.max_tokens).any():
            raise ValueError(f"a sequence would pass {self.max_tokens} tokens")
        need = -(-want // self.page_tokens) - np.asarray(self._held)
        short = np.nonzero(need > 0)[0]
        pages = self._free.alloc(int(need[short].sum())) if short.size else []
        for s in short:
            at, n = self._held[s], int(need[s])
            self._table[s, at : at + n] = pages[:n]
            pages = pages[n:]
            self._held[s] = at + n
            self._dirty = True
        self._upload()
        if one_row:
            self.row_offsets = self._one_row
        else:
            offsets = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
            self.row_offsets = torch.from_numpy(offsets).pin_memory().to(self.device, non_blocking=True)
        if not np.array_equal(new, self._new):
            self._new = new
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

    def append(self, layer: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor | None:
        """The open step's keys and values into layer ``layer``'s pages; returns the rotated queries."""
        if not self._open:
            raise RuntimeError("no step is open: begin_step or begin_rows first")
        return append_kv(self.layers[layer], self.page_table, self.lengths, self.row_offsets, k, v, q=q, cos=self.cos,
                         sin=self.sin, interleaved=self.interleaved, status=self.status)

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
        self.lengths.add_(self._new_dev)
        self._length += self._new
        self._open = False

    def abandon_step(self) -> None:
        """Close the open step without advancing: the sequences stay as they were before it.  What it has appended is
        never read, and the next step's tokens go in its place; pages that it was handed stay with their slots."""
        if not self._open:
            raise RuntimeError("no step is open")
        self._open = False

    def raise_if_failed(self) -> None:
        """Synchronize; raise if a row was left out or an attention did not finish."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError("asterq paged_kv: " + ("a row had no page or no position, or a page id was not valid"
                                                     if code == 1 else "a wait on the device ran out"))
