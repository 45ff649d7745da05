"""Plain 64-bit forms of the operators for many requests and of the token log
probabilities — TEST INFRASTRUCTURE ONLY (see package doc)."""
from __future__ import annotations

import numpy as np
import torch

from . import nvfp4

PAGE = 256


def build_tables(lengths, new_rows, held, ring, ring_state, table, rows):
    """Request by request in Python integers; returns a dict of numpy arrays and
    the set of reasons why requests were denied."""
    table, ring = np.array(table, np.int64), np.array(ring, np.int64)
    before = ring.copy()
    R, W = table.shape
    F = len(ring)
    head, count = int(ring_state[0]), int(ring_state[1])
    taken = asked = freed = 0
    cu, kv, held_out, denied, why = [0], [], [], [], set()
    for b in range(R):
        n, have, used = max(int(new_rows[b]), 0), int(held[b]), int(lengths[b])
        no = False
        if new_rows[b] < 0:
            for j in range(have):
                ring[(head + count + freed) % F] = table[b, j]
                freed += 1
            kv.append(0)
            held_out.append(0)
        else:
            grow = 0
            if n and used + n > W * PAGE:
                no = True
                why.add("wide")
            elif n:
                grow = max(-(-(used + n) // PAGE) - have, 0)
                asked += grow
                if grow and asked > count:
                    no = True
                    why.add("empty")
            if not no:
                for j in range(grow):
                    table[b, have + j] = before[(head + asked - grow + j) % F]
                taken += grow
            kv.append(0 if no else used + n)
            held_out.append(have + (0 if no else grow))
        denied.append(no)
        cu.append(cu[-1] + n)
    slots, positions, request_of = np.full(rows, -1), np.zeros(rows, int), np.full(rows, -1)
    for b in range(R):
        for i in range(cu[b], min(cu[b + 1], rows)):
            p = int(lengths[b]) + i - cu[b]
            positions[i], request_of[i] = p, b
            if not denied[b]:
                slots[i] = table[b, p // PAGE] * PAGE + p % PAGE
    return {"block_table": table, "ring": ring, "cu_rows": np.array(cu), "kv_lens": np.array(kv),
            "held_out": np.array(held_out), "ring_out": np.array([(head + taken) % F, count - taken + freed]),
            "slots": slots, "positions": positions, "request_of": request_of}, why


def dequant(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """FP64 values of uint8 codes [..., D/2] and E4M3 bytes [..., D/16]."""
    lut = torch.tensor(nvfp4.E2M1_VALUE, dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = scales.view(torch.uint8).view(torch.float8_e4m3fn).double()
    return lut[c] * s.repeat_interleave(16, -1)


def attend(q, k_cache, v_cache, k_scales, v_scales, table, cu_rows, kv_lens, out, sm_scale):
    """FP64 attention, request by request; returns (out, the sum of p |v|) with
    rows outside every request taken from `out`.  Pages outside the pool count
    as absent."""
    ref, mag = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    P, H = k_cache.shape[0], k_cache.shape[2]
    G = q.shape[1] // H
    for b, kv in enumerate(kv_lens.tolist()):
        lo, hi = int(cu_rows[b]), int(cu_rows[b + 1])
        n, pages = hi - lo, -(-kv // PAGE)
        if n <= 0:
            continue
        if kv <= 0:
            ref[lo:hi] = 0
            continue
        ids = table[b, :pages].long()
        good = ((ids >= 0) & (ids < P)).repeat_interleave(PAGE)[:kv]
        ids = torch.where((ids >= 0) & (ids < P), ids, 0)
        k = dequant(k_cache[ids].flatten(0, 1)[:kv], k_scales[ids].flatten(0, 1)[:kv]).repeat_interleave(G, 1)
        v = dequant(v_cache[ids].flatten(0, 1)[:kv], v_scales[ids].flatten(0, 1)[:kv]).repeat_interleave(G, 1)
        j = torch.arange(kv, device=q.device)
        seen = (j[None] < kv - n + torch.arange(n, device=q.device)[:, None] + 1) & good[None]
        s = torch.einsum("nhd,thd->hnt", q[lo:hi].double(), k) * sm_scale
        s = s.masked_fill(~seen, -torch.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m.isinf(), 0.0, m))
        p = p / torch.where(m.isinf(), 1.0, p.sum(-1, keepdim=True))
        ref[lo:hi] = torch.einsum("hnt,thd->nhd", p, v)
        mag[lo:hi] = torch.einsum("hnt,thd->nhd", p, v.abs())
    return ref, mag


def token_logprobs(logits, ids, top):
    """FP64 log probabilities of ids, entropy, top log probabilities and their
    indices (equal values by lowest index, NaN last)."""
    x = logits.double()
    empty = (x == -torch.inf).all(-1)
    lp = torch.where(empty[:, None], -torch.inf, x.log_softmax(-1))
    p = lp.exp()
    entropy = torch.where(empty, 0.0, torch.where(p == 0, 0.0, -p * lp).sum(-1))
    key = torch.where(x.isnan(), -torch.inf, x)
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    # NaN after -inf
    rank_nan = torch.sort(x.gather(1, order).isnan().to(torch.int8), dim=-1, stable=True)[1]
    order = order.gather(1, rank_nan)[:, :top]
    given = torch.where(ids < 0, 0.0, lp.gather(1, ids.clamp(min=0)[:, None])[:, 0])
    return given, entropy, lp.gather(1, order), order
