"""Many requests over one NVFP4 pool (include/qwz_b200.h, `qwz_batch_*`).

The reference serves one session (src/qwasar_runtime/engine.py:602-610); these
operators are new.  One step of any mix of decode rows, verify windows and
prompt chunks is

    batch.build_tables(...)          pages, block tables, slot map, row offsets
    per layer: batch.append(...)     the step's K/V rows into their slots
               batch.attend(...)     attention of all rows over their pages
    scoring.token_logprobs(...)      what the logits say of the drafted tokens

All lengths stay on the device, so a step can be captured into a CUDA graph.
As in `ops`: launches go to the current stream of the tensors' device, nothing
synchronises or allocates (except `attend_workspace`), a CPU tensor raises.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import PAGE, _contig, _cuda, _dtype_code, _p, _stream

_SCALES = (torch.uint8, torch.float8_e4m3fn)


def _int32(**tensors) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")


def _pool(k_cache, v_cache, k_scales, v_scales):
    """Checks the pool; returns (pages, kv_heads, head_dim)."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[1] != PAGE or shape[3] not in (32, 64, 128):
        raise ValueError(f"k_cache must be uint8 [P, 256, kv_heads, 32 | 64 | 128], got {tuple(shape)}")
    if v_cache.shape != shape or k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise ValueError("k_cache and v_cache must be uint8 of one shape")
    want = (shape[0], PAGE, shape[2], shape[3] // 8)
    if k_scales.shape != want or v_scales.shape != want:
        raise ValueError(f"scales must be [P, 256, kv_heads, head_dim / 16] = {want}")
    if k_scales.dtype not in _SCALES or v_scales.dtype not in _SCALES:
        raise ValueError("scales must be float8_e4m3fn")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scales.is_contiguous()
            and v_scales.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    return shape[0], shape[2], shape[3] * 2


def _rows(name: str, t, heads: int, dim: int) -> int:
    """Checks rows [T, heads, dim] with head and dim contiguous; returns the row stride."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise ValueError(f"{name} must be [rows, {heads}, {dim}], got {tuple(t.shape)}")
    row, head, one = t.stride()
    if (one != 1 and dim > 1) or (head != dim and heads > 1):
        raise ValueError(f"{name} must have head and dim contiguous")
    return row if t.shape[0] > 1 else max(row, heads * dim)


def build_tables(lengths, new_rows, held, ring, ring_state, block_table, cu_rows, kv_lens, held_out, ring_out,
                 slots, positions, request_of) -> None:
    """Page allocation, block tables, slot map and row offsets of one step.

    Request b holds `held[b]` pages and `lengths[b]` tokens and adds
    `new_rows[b]` rows (0: idle, negative: it ends and its pages are freed).
    `ring` [F] and `ring_state` (first, count) are the free page ids; pages are
    entered into `block_table` [R, W] in place.  Outputs: `cu_rows` [R + 1],
    `kv_lens` [R] (tokens after the step), `held_out` [R], `ring_out` [2], and
    for every row `slots` (page * 256 + offset, -1: none), `positions`,
    `request_of`; these may be longer than the step has rows (the rest gets
    -1, 0, -1).  To commit a step, use held_out, ring_out and the lengths
    that were kept (rejected rows need no undoing: their slots are written
    again) as the next step's inputs.  All tensors int32."""
    dev = _cuda(lengths, new_rows, held, ring, ring_state, block_table, cu_rows, kv_lens, held_out, ring_out,
                slots, positions, request_of)
    _int32(lengths=lengths, new_rows=new_rows, held=held, ring=ring, ring_state=ring_state, block_table=block_table,
           cu_rows=cu_rows, kv_lens=kv_lens, held_out=held_out, ring_out=ring_out, slots=slots, positions=positions,
           request_of=request_of)
    R, T = lengths.numel(), slots.numel()
    if new_rows.numel() != R or held.numel() != R or kv_lens.numel() != R or held_out.numel() != R:
        raise ValueError("lengths, new_rows, held, kv_lens and held_out must have one entry per request")
    if block_table.dim() != 2 or block_table.shape[0] != R:
        raise ValueError("block_table must be [requests, width]")
    if cu_rows.numel() != R + 1 or ring_state.numel() != 2 or ring_out.numel() != 2:
        raise ValueError("cu_rows has requests + 1 entries, ring_state and ring_out have 2")
    if positions.numel() != T or request_of.numel() != T:
        raise ValueError("slots, positions and request_of must have the same length")
    lib = _lib.load()
    _lib.check(lib.qwz_batch_tables(
        _p(lengths), _p(new_rows), _p(held), _p(ring), _p(ring_state), _p(block_table), _p(cu_rows), _p(kv_lens),
        _p(held_out), _p(ring_out), _p(slots), _p(positions), _p(request_of), R, block_table.shape[1], ring.numel(),
        T, _stream(dev)), "qwz_batch_tables")


def append(k, v, k_cache, v_cache, k_scales, v_scales, slots, k_held=None, v_held=None) -> None:
    """Quantise rows k, v [T, kv_heads, dim] (FP16/BF16, any row stride that is
    a multiple of 8) into slots [T] (int32, negative: not stored).  k_held and
    v_held (contiguous, same type) receive the values the cache holds for the
    rows, e.g. for attention within a prompt chunk on what later steps will read."""
    dev = _cuda(k, v, k_cache, v_cache, k_scales, v_scales, slots, k_held, v_held)
    P, heads, dim = _pool(k_cache, v_cache, k_scales, v_scales)
    ks, vs = _rows("k", k, heads, dim), _rows("v", v, heads, dim)
    T = k.shape[0]
    if v.shape[0] != T or v.dtype != k.dtype:
        raise ValueError("k and v must have the same rows and dtype")
    if slots.dtype != torch.int32 or slots.numel() != T or not slots.is_contiguous():
        raise ValueError("slots must be contiguous int32, one per row")
    for name, t in (("k_held", k_held), ("v_held", v_held)):
        if t is not None:
            if t.dtype != k.dtype or t.shape != k.shape:
                raise ValueError(f"{name} must have k's shape and dtype")
            _contig(name, t)
    lib = _lib.load()
    _lib.check(lib.qwz_batch_append(
        _p(k), _p(v), _p(k_cache), _p(v_cache), _p(k_scales), _p(v_scales), _p(slots), _p(k_held), _p(v_held), T, ks,
        vs, heads, dim, P, _dtype_code(k.dtype), _stream(dev)), "qwz_batch_append")


def attend_workspace(device, head_dim: int) -> torch.Tensor:
    """Workspace of `attend` for one call at a time (allocate before capture);
    its size does not depend on the requests."""
    n = _lib.load().qwz_batch_attend_workspace_bytes(head_dim)
    if n == 0:
        raise ValueError("head_dim must be 64, 128 or 256")
    return torch.empty(n, dtype=torch.uint8, device=device)


def attend(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace, max_rows: int,
           sm_scale: float | None = None) -> None:
    """Attention of the rows q [T, q_heads, dim] of all requests over their
    pages, into out (same shape and type; row strides any multiple of 8).
    Row s of a request's n rows sees its first kv - n + s + 1 tokens; a row
    that sees none is 0.  `max_rows` is a host bound of the rows a request
    has (1 for a decode step).  q_heads is 1 to 64 times kv_heads."""
    dev = _cuda(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace)
    P, heads, dim = _pool(k_cache, v_cache, k_scales, v_scales)
    if q.dim() != 3 or q.shape[1] % heads != 0:
        raise ValueError(f"q must be [rows, a multiple of {heads} heads, {dim}], got {tuple(q.shape)}")
    T, q_heads = q.shape[0], q.shape[1]
    qs, os = _rows("q", q, q_heads, dim), _rows("out", out, q_heads, dim)
    if out.dtype != q.dtype or out.shape[0] != T:
        raise ValueError("out must match q")
    _int32(block_table=block_table, cu_rows=cu_rows, kv_lens=kv_lens)
    R = kv_lens.numel()
    if block_table.dim() != 2 or block_table.shape[0] != R or cu_rows.numel() != R + 1:
        raise ValueError("block_table must be [requests, width], cu_rows [requests + 1], kv_lens [requests]")
    lib = _lib.load()
    _lib.check(lib.qwz_batch_attend(
        _p(q), _p(k_cache), _p(v_cache), _p(k_scales), _p(v_scales), _p(block_table), _p(cu_rows), _p(kv_lens),
        _p(out), _p(workspace), workspace.numel() * workspace.element_size(), T, R, max_rows, block_table.shape[1], P,
        q_heads, heads, dim, qs, os, dim ** -0.5 if sm_scale is None else float(sm_scale), _dtype_code(q.dtype),
        _stream(dev)), "qwz_batch_attend")
