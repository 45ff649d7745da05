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
from .ops import _contig, _cuda, _p, _stream

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
    dev = _cuda(logits, ids, logprob, entropy, top_logprobs, top_ids, workspace)
    if logits.dim() != 2 or logits.dtype not in _CODES or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be float16, bfloat16 or float32 [rows, vocab] with contiguous rows")
    T, V = logits.shape
    if ids.dtype not in (torch.int32, torch.int64) or ids.numel() != T:
        raise ValueError("ids must be int32 or int64, one per row")
    if top_ids.dim() != 2 or top_ids.shape[0] != T or top_logprobs.shape != top_ids.shape:
        raise ValueError("top_logprobs and top_ids must be [rows, K]")
    if logprob.numel() != T or entropy.numel() != T:
        raise ValueError("logprob and entropy must have one entry per row")
    if logprob.dtype != torch.float32 or entropy.dtype != torch.float32 or top_logprobs.dtype != torch.float32 \
            or top_ids.dtype != torch.int32:
        raise ValueError("logprob, entropy and top_logprobs must be float32, top_ids int32")
    for name, t in (("ids", ids), ("logprob", logprob), ("entropy", entropy), ("top_logprobs", top_logprobs),
                    ("top_ids", top_ids), ("workspace", workspace)):
        _contig(name, t)
    lib = _lib.load()
    _lib.check(lib.qwz_token_logprobs(
        _p(logits), _p(ids), int(ids.dtype == torch.int64), _p(logprob), _p(entropy), _p(top_logprobs), _p(top_ids),
        _p(workspace), workspace.numel() * workspace.element_size(), T, V, top_ids.shape[1], logits.stride(0),
        _CODES[logits.dtype], _stream(dev)), "qwz_token_logprobs")
