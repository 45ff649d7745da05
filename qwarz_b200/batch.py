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
from .ops import PAGE, _contig, _dtype_code

_I32 = torch.int32
_U8 = torch.uint8
_SCALES = (torch.float8_e4m3fn, torch.uint8)
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone; a Stream object costs 2 us a call


def _device(first, rest) -> int:
    """Index of the one CUDA device that all tensors (None: absent) are on."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("qwarz_b200 operators run on CUDA tensors only (no CPU fallback)")
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on different devices: {first.device} vs {t.device}")
    return dev


def _launch(dev, name, *args) -> None:
    """Calls `name` on the current stream of device `dev`, which need not be the current device."""
    fn = getattr(_lib.load(), name)
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _lib.check(rc, name)


def _int32(names, tensors) -> None:
    for t in tensors:
        if t.dtype is not _I32 or not t.is_contiguous():
            raise ValueError(f"{', '.join(names)} must be contiguous int32 tensors")


def _pool(k_cache, v_cache, k_scales, v_scales):
    """Checks the pool; returns (pages, kv_heads, head_dim)."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[1] != PAGE or shape[3] not in (32, 64, 128):
        raise ValueError(f"k_cache must be uint8 [P, 256, kv_heads, 32 | 64 | 128], got {tuple(shape)}")
    pages, _, heads, half = shape
    if v_cache.shape != shape or k_cache.dtype is not _U8 or v_cache.dtype is not _U8:
        raise ValueError("k_cache and v_cache must be uint8 of one shape")
    want = (pages, PAGE, heads, half // 8)
    if k_scales.shape != want or v_scales.shape != want:
        raise ValueError(f"scales must be [P, 256, kv_heads, head_dim / 16] = {want}")
    if k_scales.dtype not in _SCALES or v_scales.dtype not in _SCALES:
        raise ValueError("scales must be float8_e4m3fn")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scales.is_contiguous()
            and v_scales.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    return pages, heads, half * 2


def _rows(name: str, t, heads: int, dim: int):
    """Checks rows [T, heads, dim] with head and dim contiguous; returns (T, row stride)."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{name} must be [rows, {heads}, {dim}], got {tuple(shape)}")
    row, head, one = t.stride()
    if one != 1 or (head != dim and heads > 1):
        raise ValueError(f"{name} must have head and dim contiguous")
    return shape[0], row if shape[0] > 1 else heads * dim


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
    again) as the next step's inputs.  A request that could not be served has
    kv_lens 0 and slots of -1, and keeps held_out = held; the device error word
    says why (include/qwz_b200.h).  All tensors int32."""
    dev = _device(lengths, (new_rows, held, ring, ring_state, block_table, cu_rows, kv_lens, held_out, ring_out,
                            slots, positions, request_of))
    _int32(("lengths", "new_rows", "held", "ring", "ring_state", "block_table", "cu_rows", "kv_lens", "held_out",
            "ring_out", "slots", "positions", "request_of"),
           (lengths, new_rows, held, ring, ring_state, block_table, cu_rows, kv_lens, held_out, ring_out, slots,
            positions, request_of))
    R, T = lengths.numel(), slots.numel()
    if new_rows.numel() != R or held.numel() != R or kv_lens.numel() != R or held_out.numel() != R:
        raise ValueError("lengths, new_rows, held, kv_lens and held_out must have one entry per request")
    width = block_table.shape[-1]
    if block_table.shape != (R, width):
        raise ValueError("block_table must be [requests, width]")
    if cu_rows.numel() != R + 1 or ring_state.numel() != 2 or ring_out.numel() != 2:
        raise ValueError("cu_rows has requests + 1 entries, ring_state and ring_out have 2")
    if positions.numel() != T or request_of.numel() != T:
        raise ValueError("slots, positions and request_of must have the same length")
    _launch(
        dev, "qwz_batch_tables",
        lengths.data_ptr(), new_rows.data_ptr(), held.data_ptr(), ring.data_ptr(), ring_state.data_ptr(),
        block_table.data_ptr(), cu_rows.data_ptr(), kv_lens.data_ptr(), held_out.data_ptr(), ring_out.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), request_of.data_ptr(), R, width, ring.numel(), T)


def append(k, v, k_cache, v_cache, k_scales, v_scales, slots, k_held=None, v_held=None) -> None:
    """Quantise rows k, v [T, kv_heads, dim] (FP16/BF16, any row stride that is
    a multiple of 8) into slots [T] (int32, negative: not stored).  k_held and
    v_held (contiguous, same type) receive the values the cache holds for the
    rows, e.g. for attention within a prompt chunk on what later steps will read."""
    dev = _device(k, (v, k_cache, v_cache, k_scales, v_scales, slots, k_held, v_held))
    P, heads, dim = _pool(k_cache, v_cache, k_scales, v_scales)
    T, k_stride = _rows("k", k, heads, dim)
    Tv, v_stride = _rows("v", v, heads, dim)
    dtype = k.dtype
    if Tv != T or v.dtype is not dtype:
        raise ValueError("k and v must have the same rows and dtype")
    if slots.dtype is not _I32 or slots.numel() != T or not slots.is_contiguous():
        raise ValueError("slots must be contiguous int32, one per row")
    held = [None, None]
    for i, t in enumerate((k_held, v_held)):
        if t is not None:
            if t.dtype is not dtype or t.shape != k.shape:
                raise ValueError("k_held and v_held must have k's shape and dtype")
            _contig("k_held and v_held", t)
            held[i] = t.data_ptr()
    _launch(
        dev, "qwz_batch_append",
        k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
        slots.data_ptr(), held[0], held[1], T, k_stride, v_stride, heads, dim, P, _dtype_code(dtype))


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
    that sees none is 0, one with a NaN or +inf score NaN.  `max_rows` is a
    host bound of the rows a request has (1 for a decode step).  q_heads is 1
    to 64 times kv_heads."""
    dev = _device(q, (k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace))
    P, heads, dim = _pool(k_cache, v_cache, k_scales, v_scales)
    q_heads = q.shape[1] if q.dim() == 3 else 0
    if q_heads == 0 or q_heads % heads != 0:
        raise ValueError(f"q must be [rows, a multiple of {heads} heads, {dim}], got {tuple(q.shape)}")
    T, q_stride = _rows("q", q, q_heads, dim)
    To, out_stride = _rows("out", out, q_heads, dim)
    dtype = q.dtype
    if out.dtype is not dtype or To != T:
        raise ValueError("out must match q")
    _int32(("block_table", "cu_rows", "kv_lens"), (block_table, cu_rows, kv_lens))
    R, width = kv_lens.numel(), block_table.shape[-1]
    if block_table.shape != (R, width) or cu_rows.numel() != R + 1:
        raise ValueError("block_table must be [requests, width], cu_rows [requests + 1], kv_lens [requests]")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _launch(
        dev, "qwz_batch_attend",
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
        block_table.data_ptr(), cu_rows.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), workspace.data_ptr(),
        workspace.nbytes, T, R, max_rows, width, P, q_heads, heads, dim, q_stride, out_stride,
        dim ** -0.5 if sm_scale is None else float(sm_scale), _dtype_code(dtype))
