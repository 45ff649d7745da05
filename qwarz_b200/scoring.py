"""What a verify step takes from its logits (include/qwz_b200.h,
`qwz_token_logprobs`): log probabilities of given tokens, the entropy and the
top alternatives of every row, from one pass over the logits.

The reference compares argmax tokens only (engine/forward/mtp.py:36-50); this
is new.  As in `ops`: current stream, no synchronisation, no allocation (except
`workspace`), a CPU tensor raises.
"""
from __future__ import annotations

import torch

from . import _lib
from .batch import _device, _launch

_CODES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
MAX_TOP = 32


def workspace(device, rows: int, vocab: int, top: int) -> torch.Tensor:
    """Workspace of `token_logprobs` for logits of up to this size in any type
    (allocate before capture), for one call at a time."""
    lib = _lib.load()
    n = lib.qwz_token_logprobs_workspace_bytes(rows, vocab, top, _lib.DTYPE_F32)
    if n == 0 and rows > 0:
        raise ValueError(f"need vocab in 1..2^30 and top in 0..{MAX_TOP}")
    return torch.empty(n, dtype=torch.uint8, device=device)


def token_logprobs(logits, ids, logprob, entropy, top_logprobs, top_ids, workspace) -> None:
    """logits [T, V] (FP16/BF16/FP32, any row stride), ids [T] (int32/int64).
    Writes logprob [T] = log p(ids), entropy [T] (nats) and, for top_logprobs /
    top_ids [T, K] (FP32 / int32, K 0 to 32), the K most likely tokens, equal
    logits by lowest index.  ids < 0 gives 0; -inf logits are impossible tokens."""
    dev = _device(logits, (ids, logprob, entropy, top_logprobs, top_ids, workspace))
    code = _CODES.get(logits.dtype)
    if logits.dim() != 2 or code is None:
        raise ValueError("logits must be float16, bfloat16 or float32 [rows, vocab]")
    T, V = logits.shape
    stride, one = logits.stride()
    if one != 1 and V > 1:
        raise ValueError("logits must have contiguous rows")
    if ids.dtype not in (torch.int64, torch.int32) or ids.numel() != T:
        raise ValueError("ids must be int32 or int64, one per row")
    K = top_ids.shape[-1]
    if top_ids.shape != (T, K) or top_logprobs.shape != (T, K):
        raise ValueError("top_logprobs and top_ids must be [rows, K]")
    if logprob.numel() != T or entropy.numel() != T:
        raise ValueError("logprob and entropy must have one entry per row")
    f32 = torch.float32
    if logprob.dtype is not f32 or entropy.dtype is not f32 or top_logprobs.dtype is not f32 \
            or top_ids.dtype is not torch.int32:
        raise ValueError("logprob, entropy and top_logprobs must be float32, top_ids int32")
    if not (ids.is_contiguous() and logprob.is_contiguous() and entropy.is_contiguous()
            and top_logprobs.is_contiguous() and top_ids.is_contiguous() and workspace.is_contiguous()):
        raise ValueError("ids, the outputs and the workspace must be contiguous")
    _launch(
        dev, "qwz_token_logprobs",
        logits.data_ptr(), ids.data_ptr(), int(ids.dtype is torch.int64), logprob.data_ptr(), entropy.data_ptr(),
        top_logprobs.data_ptr(), top_ids.data_ptr(), workspace.data_ptr(), workspace.nbytes, T, V, K, stride, code)
