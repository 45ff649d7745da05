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


def share_prefixes(prefix_of, kv_lens, cu_rows, positions, request_of):
    """(cu_shared, reads, alone, shared_rows, positions_out) request by request,
    and whether a prefix or a row range was not to be."""
    R, T = len(kv_lens), len(positions)
    bad, reads, alone = False, [], []
    for b, g in enumerate(prefix_of):
        fits = 0 <= g < R and g != b and prefix_of[g] < 0 and (kv_lens[g] > 0 or cu_rows[g + 1] <= cu_rows[g])
        bad |= g >= 0 and not fits
        reads.append(g if fits else -1)
    ranges = []
    for b in range(R):
        lo, hi = cu_rows[b], cu_rows[b + 1]
        fits = 0 <= lo <= hi <= T
        bad |= not fits
        ranges.append(range(lo, hi) if fits else range(0))
    cu, rows = [0], []
    for g in range(R):
        behind = [b for b in range(R) if reads[b] == g and len(ranges[b])]
        alone.append(behind[0] if len(behind) == 1 else -1)
        for b in behind:
            rows += ranges[b]
        cu.append(len(rows))
    rows += [-1] * (T - len(rows))
    out = [p + (max(kv_lens[reads[b]], 0) if b >= 0 and reads[b] >= 0 else 0) for p, b in zip(positions, request_of)]
    return (cu, reads, alone, rows, out), bad


def rotate(x, positions, inv_freq, neighbours, weight=None, eps=1e-6):
    """FP64 norm and rotation of rows [T, heads, D]; returns (y, |a| + |b| of every
    element's two terms)."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    h = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    i = torch.arange(h, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if neighbours else (i, i + h)
    y, mag = x.clone(), x.abs()
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    mag[..., lo] = mag[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    return y, mag


def quantise(y):
    """(packed E2M1 codes, E4M3 bytes) of FP64 rows [..., D], by distance to the
    grids, ties to the even code."""
    def nearest(v, grid):
        up = torch.searchsorted(grid, v).clamp(1, len(grid) - 1)
        lo, hi = v - grid[up - 1], grid[up] - v
        return torch.where((hi < lo) | ((hi == lo) & (up % 2 == 0)), up, up - 1)

    e4m3 = torch.arange(127, dtype=torch.uint8, device=y.device).view(torch.float8_e4m3fn).double()
    e2m1 = torch.tensor(nvfp4.E2M1_VALUE[:8], dtype=torch.float64, device=y.device)
    b = y.reshape(*y.shape[:-1], -1, 16)
    scale = nearest((b.abs().amax(-1) / 6).clamp(max=448), e4m3)
    s = e4m3[scale][..., None]
    q = torch.where(s > 0, b / torch.where(s > 0, s, 1.0), 0.0)
    m = nearest(q.abs().clamp(max=6), e2m1)
    code = (m + 8 * ((m > 0) & (q < 0))).view(y.shape).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.to(torch.uint8)


def attend_shared(q, k_cache, v_cache, k_scales, v_scales, table, cu_rows, kv_lens, reads, out, sm_scale):
    """`attend` where request b sees all tokens of request reads[b] (-1: none) first."""
    ref, mag = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    P, H = k_cache.shape[0], k_cache.shape[2]
    G = q.shape[1] // H

    def tokens(b):
        kv = max(int(kv_lens[b]), 0)
        ids = table[b, :-(-kv // PAGE)].long()
        good = ((ids >= 0) & (ids < P)).repeat_interleave(PAGE)[:kv]
        ids = torch.where((ids >= 0) & (ids < P), ids, 0)
        k, v = (dequant(c[ids].flatten(0, 1)[:kv], s[ids].flatten(0, 1)[:kv]).repeat_interleave(G, 1)
                for c, s in ((k_cache, k_scales), (v_cache, v_scales)))
        return k, v, good

    for b in range(len(kv_lens)):
        lo, hi = int(cu_rows[b]), int(cu_rows[b + 1])
        n = hi - lo
        if n <= 0:
            continue
        k, v, good = tokens(b)
        kv = k.shape[0]
        j = torch.arange(kv, device=q.device)
        seen = (j[None] < kv - n + torch.arange(n, device=q.device)[:, None] + 1) & good[None]
        if reads[b] >= 0:
            pk, pv, pgood = tokens(reads[b])
            k, v = torch.cat([pk, k]), torch.cat([pv, v])
            seen = torch.cat([pgood[None].expand(n, -1), seen], 1)
        if not k.shape[0]:
            ref[lo:hi] = 0
            continue
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
