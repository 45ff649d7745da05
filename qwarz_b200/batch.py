"""Many requests over one NVFP4 pool (include/qwz_b200.h, `qwz_batch_*`).

The reference serves one session (src/qwasar_runtime/engine.py:602-610); these
operators are new.  One step of any mix of decode rows, verify windows and
prompt chunks is

    batch.build_tables(...)          pages, block tables, slot map, row offsets
    per layer: batch.append(...)     the step's K/V rows into their slots
               batch.attend(...)     attention of all rows over their pages
    scoring.token_logprobs(...)      what the logits say of the drafted tokens

Where requests share a prompt prefix, and where Q and K are still to be rotated:

    batch.build_tables(...)
    batch.share_prefixes(...)        rows by prefix, positions behind it
    per layer: batch.append_rotated(...)  Q and K normed and rotated, K/V into their slots
               batch.attend_shared(...)   a prefix read once for all of its requests

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


def _attend_args(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace, max_rows,
                 sm_scale, plan=None):
    """Checks of `attend` and `attend_shared`; returns (device, the C arguments)."""
    dev = _device(q, (k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace, plan))
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
    shared = ()
    if plan is not None:
        _int32(("plan",), (plan,))
        if plan.numel() < 3 * R + 1 + T:
            raise ValueError(f"plan must have 3 * requests + 1 + rows = {3 * R + 1 + T} words (prefix_plan)")
        shared = (plan.data_ptr(),)
    return dev, (q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                 block_table.data_ptr(), cu_rows.data_ptr(), kv_lens.data_ptr(), *shared, out.data_ptr(),
                 workspace.data_ptr(), workspace.nbytes, T, R, max_rows, width, P, q_heads, heads, dim, q_stride,
                 out_stride, dim ** -0.5 if sm_scale is None else float(sm_scale), _dtype_code(dtype))


def attend(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace, max_rows: int,
           sm_scale: float | None = None) -> None:
    """Attention of the rows q [T, q_heads, dim] of all requests over their
    pages, into out (same shape and type; row strides any multiple of 8).
    Row s of a request's n rows sees its first kv - n + s + 1 tokens; a row
    that sees none is 0, one with a NaN or +inf score NaN.  `max_rows` is a
    host bound of the rows a request has (1 for a decode step).  q_heads is 1
    to 64 times kv_heads."""
    dev, args = _attend_args(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace,
                             max_rows, sm_scale)
    _launch(dev, "qwz_batch_attend", *args)


def prefix_plan(device, requests: int, rows: int) -> torch.Tensor:
    """The tensor that `share_prefixes` fills and `attend_shared` reads, for
    steps of that many requests and up to that many rows (allocate before capture)."""
    return torch.empty(3 * requests + 1 + rows, dtype=_I32, device=device)


def share_prefixes(prefix_of, kv_lens, cu_rows, positions, request_of, plan, positions_out) -> None:
    """Rows of a step by the shared prefix they read, once a step for all layers.

    A prefix is a request of the batch that holds its tokens, usually idle;
    `prefix_of[b]` [R] names the one whose tokens come before request b's own
    (-1: none).  What `build_tables` counts (lengths, rows, pages, positions) are
    a request's own.  `kv_lens`, `cu_rows`, `positions` [T] and `request_of` [T]
    are its outputs; `plan` (`prefix_plan`) receives the rows by prefix and
    `positions_out` [T] the positions from the prefix's start (may be
    `positions`).  A prefix that does not exist, is the request itself or has one
    itself counts as none (device error word).  So does one whose rows of this
    step were denied: drop its readers' rows with its own and run them again.  A
    prefix is ended after the last step that reads it.  All tensors int32, at most
    2^14 requests; the plan's layout is in include/qwz_b200.h."""
    dev = _device(prefix_of, (kv_lens, cu_rows, positions, request_of, plan, positions_out))
    _int32(("prefix_of", "kv_lens", "cu_rows", "positions", "request_of", "plan", "positions_out"),
           (prefix_of, kv_lens, cu_rows, positions, request_of, plan, positions_out))
    R, T = kv_lens.numel(), positions.numel()
    if prefix_of.numel() != R or cu_rows.numel() != R + 1:
        raise ValueError("prefix_of and kv_lens have one entry per request, cu_rows requests + 1")
    if request_of.numel() != T or positions_out.numel() != T:
        raise ValueError("positions, request_of and positions_out must have the same length")
    if plan.numel() < 3 * R + 1 + T:
        raise ValueError(f"plan must have 3 * requests + 1 + rows = {3 * R + 1 + T} words (prefix_plan)")
    _launch(
        dev, "qwz_batch_share_prefixes",
        prefix_of.data_ptr(), kv_lens.data_ptr(), cu_rows.data_ptr(), positions.data_ptr(), request_of.data_ptr(),
        plan.data_ptr(), positions_out.data_ptr(), R, T)


def _weight(name: str, t, dim: int) -> int:
    if t.dtype is not torch.float32 or t.dim() != 1 or t.numel() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 [{dim}]")
    return t.data_ptr()


def _held(t, k) -> int:
    if t.dtype is not k.dtype or t.shape != k.shape:
        raise ValueError("k_held and v_held must have k's shape and dtype")
    _contig("k_held and v_held", t)
    return t.data_ptr()


def append_rotated(q, k, v, q_out, k_cache, v_cache, k_scales, v_scales, slots, positions, inv_freq,
                   neighbours: bool = False, q_weight=None, k_weight=None, eps: float = 1e-6, k_held=None,
                   v_held=None) -> None:
    """`append` of rows whose Q and K are normed and rotated on the way.

    q [T, q_heads, dim], k and v [T, kv_heads, dim] (one of FP16/BF16, row
    strides multiples of 8, parts of a packed projection for instance); q_out
    receives the rotated q (it may be q).  `positions` [T] int32; `inv_freq`
    (FP32, a multiple of 8 long, at most dim / 2) is the angle of each pair of
    dims at position 1: pairs (i, i + len(inv_freq)), or (2i, 2i + 1) with
    `neighbours`; dims behind them are not rotated.  With `q_weight`,
    `k_weight` (FP32 [dim]) a head is first divided by the root of its mean
    square plus eps (taken as FP32) and multiplied by the weight.  K is quantised
    from the rotated values without a rounding in between.  slots (each
    non-negative one once), k_held and v_held: as in `append`."""
    dev = _device(q, (k, v, q_out, k_cache, v_cache, k_scales, v_scales, slots, positions, inv_freq, q_weight,
                      k_weight, k_held, v_held))
    P, heads, dim = _pool(k_cache, v_cache, k_scales, v_scales)
    T, q_heads, _ = shape = q.shape if q.dim() == 3 else (0, 0, 0)
    dtype = q.dtype
    if q_out.shape != shape or v.shape != k.shape or k.shape[0] != T \
            or q_out.dtype is not dtype or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k, v and q_out must have the same rows and dtype, q_out the shape of q, v that of k")
    q_stride, out_stride = _rows("q", q, q_heads, dim)[1], _rows("q_out", q_out, q_heads, dim)[1]
    k_stride, v_stride = _rows("k", k, heads, dim)[1], _rows("v", v, heads, dim)[1]
    _int32(("slots", "positions"), (slots, positions))
    if slots.numel() != T or positions.numel() != T:
        raise ValueError("slots and positions must have one entry per row")
    f32 = torch.float32
    if inv_freq.dtype is not f32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 vector")
    qw = kw = kh = vh = None
    if q_weight is not None:
        qw = _weight("q_weight", q_weight, dim)
    if k_weight is not None:
        kw = _weight("k_weight", k_weight, dim)
    if k_held is not None:
        kh = _held(k_held, k)
    if v_held is not None:
        vh = _held(v_held, k)
    _launch(
        dev, "qwz_batch_append_rotated",
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        k_scales.data_ptr(), v_scales.data_ptr(), slots.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), qw, kw,
        kh, vh, T, q_stride, k_stride, v_stride, out_stride, q_heads, heads, dim, inv_freq.numel(), bool(neighbours), eps,
        P, _dtype_code(dtype))


def shared_workspace(device, head_dim: int, rows: int, q_heads: int) -> torch.Tensor:
    """Workspace of `attend_shared` for steps of up to that many rows, for one
    call at a time (allocate before capture)."""
    n = _lib.load().qwz_batch_shared_workspace_bytes(head_dim, rows, q_heads)
    if n == 0:
        raise ValueError("head_dim must be 64, 128 or 256, rows >= 0, q_heads in 1..16384")
    return torch.empty(n, dtype=_U8, device=device)


def attend_shared(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, plan, out, workspace,
                  max_rows: int, sm_scale: float | None = None) -> None:
    """`attend` behind shared prefixes: a row sees every token of the prefix
    that its request reads and then its own as in `attend`.  The prefix's pages
    are read once for the rows of all its requests together.  `plan` is what
    `share_prefixes` wrote for the step, `workspace` a `shared_workspace`; out
    shares no storage with q.  It pays from about 1 M prefix tokens x KV heads
    that all rows read together (2 M at head dim 64); below, `attend` over tables
    that name the prefix's pages for every request takes fewer launches."""
    dev, args = _attend_args(q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows, kv_lens, out, workspace,
                             max_rows, sm_scale, plan)
    _launch(dev, "qwz_batch_attend_shared", *args)
