"""Linear attention with a decay for each head: recurrent layers beside the latent ones.

Such a layer keeps a fixed-size state instead of a cache.  Here a layer's states are a pool by sequence
slot, float32 [n_slots, n_heads, dk, dv], updated in place:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   out_t = scale q_t S_t

* ``linear_attention_prefill``: ragged prompt chunks, rows ``row_offsets[s]`` and on for sequence s;
* ``linear_attention_step``: one new token a sequence.

This is the plain recurrence.  The reference's KDA layers, whose states ``AsterCache.kda_states`` holds, update
theirs by a gated delta rule (a correction by what the state has for the key already): not served here.

There is no backward pass: inputs that require a gradient are refused outside of ``torch.no_grad()``.
Both call ``asterq_linear_attention``; nothing waits for the GPU or reads from it, so calls can be
recorded in a CUDA graph.  A first prompt call on a stream, or ``workspace``, gives that stream's prompts
their workspace; a captured prompt without either has one in the graph's memory.  Graphs that overlap each
other, or other prompts of the stream that they were captured on, need a ``workspace`` each.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .paged_kv import _call, _capturing, _check_int, _check_no_gradient, _quick

_PARAMS = _lib.packer(_lib.LinearParams)
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _rows(x: torch.Tensor, name: str, q: torch.Tensor, dim: int) -> torch.Tensor:
    if x.dim() != 3 or x.shape[0] != q.shape[0] or x.shape[1] != q.shape[1] or x.shape[2] != dim:
        raise ValueError(f"{name} must be [{q.shape[0]}, {q.shape[1]}, {dim}], got {tuple(x.shape)}")
    if x.dtype != q.dtype:
        raise TypeError(f"{name} is {x.dtype}, q is {q.dtype}")
    if x.device != q.device:
        raise RuntimeError(f"{name} is on {x.device}, q is on {q.device}")
    _check_no_gradient(x, name)
    row, head, one = x.stride()
    if one != 1 or (row | head) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


class LinearAttentionWorkspace:
    """Device memory for the states between the SMs that share a prompt; its contents are of one call.
    One serves any sequence of calls on one stream; calls that overlap on the GPU need one each."""

    def __init__(self, device="cuda") -> None:
        device = torch.device(device)
        p = _lib.LinearParams()  # the most any geometry needs
        p.dtype, p.n_seqs, p.n_heads, p.dk, p.dv, p.n_rows, p.row_offsets = _lib.DTYPE_BF16, 1, 1, 128, 128, 1 << 20, 1
        with torch.cuda.device(device):
            self.nbytes = int(_lib.load().asterq_linear_workspace_bytes(_lib.ctypes.byref(p)))
            self.buffer = torch.empty(self.nbytes, dtype=torch.uint8, device=device)


_workspaces: dict[tuple[int, int], LinearAttentionWorkspace] = {}


def _workspace(device: torch.device, stream: int) -> LinearAttentionWorkspace:
    """The workspace that calls on this stream share when the caller brings none."""
    ws = _workspaces.get((device.index, stream))
    if ws is None:
        ws = LinearAttentionWorkspace(device)
        if _capturing(device):
            return ws  # of the graph's own memory
        _workspaces[(device.index, stream)] = ws
    if _quick() is not None:  # whose calls come here until it knows the workspace
        _quick().workspace(1, device.index, stream, ws.buffer.data_ptr(), ws.nbytes)
    return ws


def _run(state, slots, lengths, row_offsets, q, k, v, log_decay, scale, out, workspace, status):
    quick = _quick()
    if quick is not None and workspace is None:
        done = quick.linear(state, slots, lengths, row_offsets, q, k, v, log_decay,
                            q.shape[-1] ** -0.5 if scale is None else scale, out, status)
        if done is not NotImplemented:
            return done
    if q.dim() != 3 or state.dim() != 4:
        raise ValueError("q must be [rows, n_heads, dk] and state [n_slots, n_heads, dk, dv]")
    if q.dtype not in _DTYPES:
        raise TypeError(f"q is {q.dtype}: float32, bfloat16 or float16")
    if not q.is_cuda:
        raise RuntimeError("asterq states live on the GPU; there is no CPU path")
    rows, heads, dk = q.shape
    n_slots, _, _, dv = state.shape
    if state.shape[1] != heads or state.shape[2] != dk:
        raise ValueError(f"state {tuple(state.shape)} is not of {heads} heads of {dk} key dims")
    if state.dtype != torch.float32 or not state.is_contiguous() or state.device != q.device:
        raise ValueError("state must be a contiguous float32 tensor on q's device")
    q = _rows(q, "q", q, dk)
    k = _rows(k, "k", q, dk)
    v = _rows(v, "v", q, dv)
    if log_decay.dtype != torch.float32 or log_decay.device != q.device or log_decay.stride(-1) != 1 or (
            log_decay.shape != (heads,) and log_decay.shape != (rows, heads)):
        raise ValueError(f"log_decay must be float32 [{heads}] or [{rows}, {heads}] on q's device, its heads contiguous")
    _check_no_gradient(log_decay, "log_decay")
    _check_no_gradient(state, "state")
    if slots.dim() != 1:
        raise ValueError("slots must be [n_seqs]")
    n_seqs = slots.shape[0]
    _check_int(slots, "slots", (n_seqs,), q)
    if lengths is not None:
        _check_int(lengths, "lengths", (n_seqs,), q)
    if row_offsets is not None:
        _check_int(row_offsets, "row_offsets", (n_seqs + 1,), q)
    elif n_seqs != rows:
        raise ValueError(f"{rows} rows for {n_seqs} slots: a step has one row a slot")
    if status is not None:
        _check_int(status, "status", (1,), q)
    if out is None:
        out = torch.empty((rows, heads, dv), dtype=q.dtype, device=q.device)
    elif out.shape != (rows, heads, dv) or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {(rows, heads, dv)}")
    device = q.device
    stream = torch.cuda.current_stream(device).cuda_stream
    ws_ptr = ws_bytes = 0
    if row_offsets is not None:
        ws = _workspace(device, stream) if workspace is None else workspace
        ws_ptr, ws_bytes = ws.buffer.data_ptr(), ws.nbytes
    q_row, q_head, _ = q.stride()
    k_row, k_head, _ = k.stride()
    v_row, v_head, _ = v.stride()
    _call(_lib.load().asterq_linear_attention,
          _PARAMS.pack(_DTYPES[q.dtype], n_seqs, heads, dk, dv, n_slots, 1.0 / math.sqrt(dk) if scale is None else scale,
                       0, rows, q_row, q_head, k_row, k_head, v_row, v_head,
                       log_decay.stride(0) if log_decay.dim() == 2 else 0, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                       log_decay.data_ptr(), state.data_ptr(), slots.data_ptr(),
                       0 if lengths is None else lengths.data_ptr(),
                       0 if row_offsets is None else row_offsets.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes,
                       0 if status is None else status.data_ptr()),
          device, stream)
    return out


def linear_attention_prefill(
    state: torch.Tensor,
    slots: torch.Tensor,
    lengths: torch.Tensor | None,
    row_offsets: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: LinearAttentionWorkspace | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Outputs [rows, n_heads, dv] of ragged prompt chunks; the slots' states move to the chunks' ends.

    state float32 [n_slots, n_heads, dk, dv]; slots int32 [n_seqs], each its own (negative: an empty slot,
    whose rows come back as zeros); lengths int32 [n_seqs], the tokens each sequence has behind it (0: it
    starts from a state of zeros, whatever its slot holds), None: all continue; row_offsets int32
    [n_seqs + 1].  q, k [rows, n_heads, dk] and v [rows, n_heads, dv] of one type, with any row and head
    stride.  log_decay float32 [n_heads] or [rows, n_heads], not above 0.  scale: 1 / sqrt(dk) unless
    given.  status int32 [1]: set to 1 when a slot or row offset was out of range, or offsets decreased.

    bf16 prompts run in chunks of 128 tokens on the tensor cores where ``out`` and ``state`` are 32-byte aligned,
    no stride is 0 and there are 24 rows a slot or more on average, other types and shorter prompts token by token:
    pass the slots that have rows, not idle ones beside them, and long prompts apart from single rows.

    What is not finite reaches what the recurrence takes it to, and nothing else: a value of v its column of the state
    and of the outputs from its row on; of k its row of the state and the outputs from its row on; of q its row's
    outputs; of a state its column's outputs.  An infinity may become NaN on the way.  Rows of no sequence are not
    written.
    """
    return _run(state, slots, lengths, row_offsets, q, k, v, log_decay, scale, out, workspace, status)


def linear_attention_step(
    state: torch.Tensor,
    slots: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    *,
    lengths: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """One new token a sequence: row i updates slot ``slots[i]`` and reads it; arguments as for
    ``linear_attention_prefill``."""
    return _run(state, slots, lengths, None, q, k, v, log_decay, scale, out, None, status)
