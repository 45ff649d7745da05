"""Cases of the operators that let many requests share one NVFP4 pool, in the
order in which a speculative-verify step uses them:

  tables    block tables, slot maps and page allocation from request lengths
  append    new K/V rows quantised into the pages of their slots
  attend    attention of every request's rows over its pages (4-bit cache)
  logprobs  log probabilities of given tokens, entropy, top alternatives

`own` chooses between the plain form (elementary torch operations in 32 bits)
and the framework's operators.  Lengths follow from the case alone, values
from the seed.
"""
import math
import random

import torch

own = False

PAGE = 256
MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# (query heads, KV heads, head dim): the cache's own layout first, then generic ones
LAYOUTS = ((24, 4, 256), (32, 8, 128), (16, 2, 128), (24, 8, 128), (8, 8, 64), (14, 2, 64), (40, 8, 128), (16, 1, 256))


def listed():
    return [
        # one interactive user group: 8 requests each add one token (latency)
        {"name": "tables decode 8", "op": "tables", "requests": 8, "width": 256, "kv_lo": 100, "kv_hi": 60000,
         "rows": "decode", "ended": 0.0, "mix": 1},
        # a full server at a step boundary: decode rows, 7-row windows, prompt chunks, requests that end
        {"name": "tables mixed 2048", "op": "tables", "requests": 2048, "width": 128, "kv_lo": 1, "kv_hi": 30000,
         "rows": "mixed", "ended": 0.03, "mix": 2},
        # the 7-row windows of 32 requests: 224 new rows of one layer
        {"name": "append windows 32x7", "op": "append", "rows": 224, "kv_heads": 4, "dim": 256, "type": "bf16",
         "packed": True},
        # a prompt chunk budget of 16,384 rows, K and V inside the projection's packed rows
        {"name": "append prompts 16384", "op": "append", "rows": 16384, "kv_heads": 4, "dim": 256, "type": "f16",
         "packed": True},
        # a lone request's decode at 4,000 tokens (latency)
        {"name": "attend decode 1x4000", "op": "attend", "requests": 1, "kv_lo": 4000, "kv_hi": 4000, "rows": "decode",
         "heads": 24, "kv_heads": 4, "dim": 256, "type": "f16", "mix": 3},
        # a busy server's decode step, contexts from 256 to 32,768 tokens
        {"name": "attend decode 64", "op": "attend", "requests": 64, "kv_lo": 256, "kv_hi": 32768, "rows": "decode",
         "heads": 24, "kv_heads": 4, "dim": 256, "type": "bf16", "mix": 4},
        # many short chats on a 32/8/128 head layout
        {"name": "attend decode 256 d128", "op": "attend", "requests": 256, "kv_lo": 90, "kv_hi": 4096,
         "rows": "decode", "heads": 32, "kv_heads": 8, "dim": 128, "type": "f16", "mix": 5},
        # the 7-row verify windows of 16 requests at long contexts
        {"name": "attend verify 16x7", "op": "attend", "requests": 16, "kv_lo": 4096, "kv_hi": 32768, "rows": "window",
         "heads": 24, "kv_heads": 4, "dim": 256, "type": "bf16", "mix": 6},
        # a step that mixes prompt chunks, windows and decode rows
        {"name": "attend prompts 8", "op": "attend", "requests": 8, "kv_lo": 1500, "kv_hi": 8192, "rows": "prompts",
         "heads": 24, "kv_heads": 4, "dim": 256, "type": "bf16", "mix": 7},
        # one verify window's logits: 7 rows (latency)
        {"name": "logprobs window 7", "op": "logprobs", "rows": 7, "vocab": 131072, "pad": 0, "top": 8, "type": "bf16",
         "masked": 0.0},
        # the windows of 64 requests, logits in rows padded for the projection
        {"name": "logprobs 64x7", "op": "logprobs", "rows": 448, "vocab": 151000, "pad": 104, "top": 20, "type": "bf16",
         "masked": 0.0},
        # FP32 logits of an odd vocabulary, half of it masked off by a grammar
        {"name": "logprobs masked f32", "op": "logprobs", "rows": 33, "vocab": 50257, "pad": 0, "top": 5, "type": "f32",
         "masked": 0.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "append", "attend", "attend", "attend", "logprobs"))
    mix = rng.randrange(1 << 20)
    if op == "tables":
        width = _log(rng, 16, 256)
        return {"op": op, "requests": _log(rng, 1, 2048), "width": width, "kv_lo": 1,
                "kv_hi": _log(rng, 300, width * PAGE - 2600), "rows": rng.choice(("decode", "window", "mixed")),
                "ended": rng.choice((0.0, 0.1)), "mix": mix}
    if op == "append":
        _, kv_heads, dim = rng.choice(LAYOUTS)
        return {"op": op, "rows": _log(rng, 1, 16384), "kv_heads": kv_heads, "dim": dim,
                "type": rng.choice(("f16", "bf16")), "packed": rng.random() < 0.5}
    if op == "logprobs":
        vocab = _log(rng, 100, 160000)
        return {"op": op, "rows": min(_log(rng, 1, 448), 60_000_000 // vocab), "vocab": vocab,
                "pad": rng.choice((0, 0, 1, 64)), "top": rng.choice((0, 1, 5, 20, 32)),
                "type": rng.choice(("f16", "bf16", "f32")), "masked": rng.choice((0.0, 0.3))}
    heads, kv_heads, dim = rng.choice(LAYOUTS)
    rows = rng.choice(("decode", "decode", "window", "mixed", "prompts"))
    kv_hi = _log(rng, 2, 32768) if rows != "prompts" else _log(rng, 500, 8192)
    # padded tokens x KV width at most what "attend decode 64" has (half of it:
    # the plain form pads every request to the longest)
    most = max(1, min(256, 64 * 32768 * 1024 // (2 * kv_hi * kv_heads * dim)))
    if rows in ("prompts", "mixed"):
        most = max(1, min(most, 8 * 8192 * 24 // (kv_hi * heads)))
    return {"op": op, "requests": _log(rng, 1, most), "kv_lo": 1 + kv_hi // rng.choice((1, 3, 20, 100)), "kv_hi": kv_hi,
            "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": rng.choice(("f16", "bf16")),
            "mix": mix}


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """(tokens after the step, rows of the step) of every request."""
    rng = random.Random(case["mix"])
    kv, new = [], []
    for i in range(case["requests"]):
        lo, hi = min(case["kv_lo"], case["kv_hi"]), case["kv_hi"]
        n = _log(rng, lo, hi) if hi > lo else hi
        mode = case["rows"]
        if mode == "mixed":
            mode = rng.choice(("decode", "decode", "window", "chunk", "idle"))
        elif mode == "prompts":
            mode = ("chunk", "chunk", "prompt", "decode", "chunk", "window", "prompt", "chunk")[i % 8]
        r = {"decode": 1, "window": 7, "chunk": _log(rng, 9, 2048), "prompt": n, "idle": 0}[mode]
        kv.append(n)
        new.append(min(r, n, 2048))
    return kv, new


def _pages(n):
    return (n + PAGE - 1) // PAGE


# ------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantise(x):
    """FP32 [..., D] -> (E2M1 codes [..., D] as whole numbers, E4M3 scales [..., D/16]);
    amax / 6 rounded to E4M3, x / scale rounded to nearest even and saturated at 6."""
    b = x.view(*x.shape[:-1], -1, 16)
    scale = (b.abs().amax(-1) / 6).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float().unsqueeze(-1)
    y = torch.where(s > 0, b / s, torch.zeros_like(b))
    a = y.abs()
    m = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where((m > 0) & (y < 0), m + 8, m)
    return code.to(torch.uint8).view(x.shape), scale


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(code, scale):
    """The FP32 values that codes and scales stand for."""
    lut = torch.tensor(MAGS + tuple(-m for m in MAGS), device=code.device)
    v = lut[code.long()]
    return (v.view(*v.shape[:-1], -1, 16) * scale.float().unsqueeze(-1)).view(v.shape)


def _pool(pages, kv_heads, dim, g):
    """A pool filled with quantised rows: unit normal with a few strong channels."""
    codes = torch.empty(pages, PAGE, kv_heads, dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, PAGE, kv_heads, dim // 16, dtype=torch.float8_e4m3fn, device="cuda")
    gain = torch.exp(0.3 * torch.randn(kv_heads, dim, generator=g, device="cuda"))
    step = max(1, (1 << 26) // (PAGE * kv_heads * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        code, scale = _quantise(torch.randn(n, PAGE, kv_heads, dim, generator=g, device="cuda") * gain)
        codes[at:at + n] = _pack(code)
        scales[at:at + n] = scale
    return codes, scales


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"tables": _prepare_tables, "append": _prepare_append, "attend": _prepare_attend,
            "logprobs": _prepare_logprobs}[case["op"]](case, seed)


def _prepare_tables(case, seed):
    g = _generator(seed)
    kv, new = _lengths(case)
    rng = random.Random(seed)
    held = [_pages(n - r) + (rng.random() < 0.2) for n, r in zip(kv, new)]
    held = [min(h, case["width"]) for h in held]
    ends = [rng.random() < case["ended"] for _ in kv]
    total = sum(held)
    pool = 2 * sum(_pages(n) for n in kv) + len(kv) + 16
    free = pool - total
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["requests"], case["width"]), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(case["width"], device="cuda")
    h = _int(held)
    table[at[None] < h[:, None]] = ids[:total]
    ring = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    head = rng.randrange(pool)
    ring[(head + torch.arange(free, device="cuda")) % pool] = ids[total:]
    rows = sum(new)
    B = case["requests"]
    return {
        "op": "tables",
        "lengths": _int([n - r for n, r in zip(kv, new)]),
        "new": _int([-1 if e else r for r, e in zip(new, ends)]),
        "held": h, "ring": ring, "ring_state": _int([head, free]), "table": table,
        "cu_rows": torch.empty(B + 1, dtype=torch.int32, device="cuda"),
        "kv_lens": torch.empty(B, dtype=torch.int32, device="cuda"),
        "held_out": torch.empty(B, dtype=torch.int32, device="cuda"),
        "ring_out": torch.empty(2, dtype=torch.int32, device="cuda"),
        "slots": torch.empty(rows, dtype=torch.int32, device="cuda"),
        "positions": torch.empty(rows, dtype=torch.int32, device="cuda"),
        "requests": torch.empty(rows, dtype=torch.int32, device="cuda"),
    }


def _prepare_append(case, seed):
    g = _generator(seed)
    T, H, D = case["rows"], case["kv_heads"], case["dim"]
    dt = TYPES[case["type"]]
    gain = torch.exp(0.3 * torch.randn(H, D, generator=g, device="cuda"))
    if case["packed"]:  # K and V are slices of wider rows (query heads ahead of them)
        rows = torch.randn(T, 3 * H, D, generator=g, device="cuda")
        rows[:, H:2 * H] *= gain
        rows = rows.to(dt)
        k, v = rows[:, H:2 * H], rows[:, 2 * H:]
    else:
        k = (torch.randn(T, H, D, generator=g, device="cuda") * gain).to(dt)
        v = torch.randn(T, H, D, generator=g, device="cuda").to(dt)
    pages = _pages(T) + 3
    slots = torch.randperm(pages, generator=g, device="cuda")[:_pages(T)]
    slots = (slots[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:T].to(torch.int32)
    shape = (pages, PAGE, H)
    return {"op": "append", "k": k, "v": v, "slots": slots,
            "k_cache": torch.zeros(*shape, D // 2, dtype=torch.uint8, device="cuda"),
            "v_cache": torch.zeros(*shape, D // 2, dtype=torch.uint8, device="cuda"),
            "k_scales": torch.zeros(*shape, D // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            "v_scales": torch.zeros(*shape, D // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            "k_held": torch.empty(T, H, D, dtype=dt, device="cuda"),
            "v_held": torch.empty(T, H, D, dtype=dt, device="cuda")}


def _prepare_attend(case, seed):
    g = _generator(seed)
    kv, new = _lengths(case)
    Hq, H, D = case["heads"], case["kv_heads"], case["dim"]
    dt = TYPES[case["type"]]
    width = _pages(max(kv))
    total = sum(_pages(n) for n in kv)
    k_cache, k_scales = _pool(total + 1, H, D, g)
    v_cache, v_scales = _pool(total + 1, H, D, g)
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda")[None] < _int([_pages(n) for n in kv])[:, None]
    table[used] = torch.randperm(total + 1, generator=g, device="cuda")[:total].to(torch.int32)
    cu = [0]
    for r in new:
        cu.append(cu[-1] + r)
    T = max(cu[-1], 1)
    # the rows of a packed projection: queries ahead of the K and V heads
    packed = torch.randn(T, Hq + 2 * H, D, generator=g, device="cuda") * 1.5
    return {"op": "attend", "q": packed.to(dt)[:, :Hq], "k_cache": k_cache, "v_cache": v_cache,
            "k_scales": k_scales, "v_scales": v_scales, "table": table, "cu_rows": _int(cu), "kv_lens": _int(kv),
            "out": torch.zeros(T, Hq, D, dtype=dt, device="cuda"), "max_rows": max(max(new), 1),
            "max_kv": max(kv), "rows": cu[-1]}


def _prepare_logprobs(case, seed):
    g = _generator(seed)
    T, V, K = case["rows"], case["vocab"], case["top"]
    x = torch.randn(T, V + case["pad"], generator=g, device="cuda") * 2.5
    # a handful of likely tokens a row, as a trained model gives
    hot = torch.randint(0, V, (T, 6), generator=g, device="cuda")
    x.scatter_add_(1, hot, torch.rand(T, 6, generator=g, device="cuda") * 16)
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < 0.7, hot[:, 0],
                      torch.randint(0, V, (T,), generator=g, device="cuda"))
    if case["masked"]:
        off = torch.rand(V + case["pad"], generator=g, device="cuda") < case["masked"]
        x.masked_fill_(off[None], -math.inf)
        ids = torch.where(off[ids], x[:, :V].argmax(1), ids)
    return {"op": "logprobs", "logits": x.to(TYPES[case["type"]])[:, :V], "ids": ids, "top": K,
            "logprob": torch.empty(T, device="cuda"), "entropy": torch.empty(T, device="cuda"),
            "top_logprobs": torch.empty(T, K, device="cuda"),
            "top_ids": torch.empty(T, K, dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------- passes
def run(state):
    return {"tables": _run_tables, "append": _run_append, "attend": _run_attend,
            "logprobs": _run_logprobs}[state["op"]](state)


def _run_tables(s):
    if own:
        from qwarz_b200 import batch

        batch.build_tables(s["lengths"], s["new"], s["held"], s["ring"], s["ring_state"], s["table"], s["cu_rows"],
                           s["kv_lens"], s["held_out"], s["ring_out"], s["slots"], s["positions"], s["requests"])
        return {k: s[k] for k in ("table", "ring", "cu_rows", "kv_lens", "held_out", "ring_out", "slots", "positions",
                                  "requests")}
    length, held, table, ring = s["lengths"].long(), s["held"].long(), s["table"].long(), s["ring"].long()
    B, W = table.shape
    F = ring.numel()
    head, count = s["ring_state"].long()
    ends = s["new"] < 0
    new = s["new"].long().clamp(min=0)
    fits = length + new <= W * PAGE
    grow = torch.where((new > 0) & fits, ((length + new + PAGE - 1) // PAGE - held).clamp(min=0), 0)
    upto = grow.cumsum(0)
    denied = (new > 0) & (~fits | ((grow > 0) & (upto > count)))
    first = upto - grow
    grow = torch.where(denied, 0, grow)
    # the granted pages enter the table
    j = torch.arange(W, device=table.device)[None]
    fresh = (j >= held[:, None]) & (j < (held + grow)[:, None])
    table = torch.where(fresh, ring[(head + first[:, None] + j - held[:, None]) % F], table)
    # the pages of requests that end go back behind the free ones
    freed = torch.where(ends, held, 0)
    back = freed.cumsum(0) - freed
    gone = j < freed[:, None]
    ring = ring.scatter(0, ((head + count + back[:, None] + j) % F)[gone], table[gone])
    taken = grow.sum()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    r = torch.arange(s["slots"].numel(), device=table.device)
    req = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    pad = req >= B
    req = req.clamp(max=B - 1)
    pos = length[req] + r - cu[req]
    page = table[req, (pos // PAGE).clamp(max=W - 1)]
    slot = torch.where(pad | denied[req], -1, page * PAGE + pos % PAGE)
    i32 = torch.int32
    return {"table": table.to(i32), "ring": ring.to(i32), "cu_rows": cu.to(i32),
            "kv_lens": torch.where(ends | denied, 0, length + new).to(i32),
            "held_out": torch.where(ends, 0, held + grow).to(i32),
            "ring_out": torch.stack([(head + taken) % F, count - taken + freed.sum()]).to(i32),
            "slots": slot.to(i32), "positions": torch.where(pad, 0, pos).to(i32),
            "requests": torch.where(pad, -1, req).to(i32)}


def _run_append(s):
    names = ("k_held", "v_held", "k_cache", "v_cache", "k_scales", "v_scales")
    if own:
        from qwarz_b200 import batch

        batch.append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["slots"],
                     k_held=s["k_held"], v_held=s["v_held"])
        got = {n: s[n] for n in names}
    else:
        at = s["slots"].long()
        x = torch.stack([s["k"], s["v"]]).float()
        code, scale = _quantise(x)
        held, packed = _values(code, scale).to(s["k"].dtype), _pack(code)
        s["k_cache"].flatten(0, 1)[at] = packed[0]
        s["v_cache"].flatten(0, 1)[at] = packed[1]
        s["k_scales"].view(torch.uint8).flatten(0, 1)[at] = scale[0].view(torch.uint8)
        s["v_scales"].view(torch.uint8).flatten(0, 1)[at] = scale[1].view(torch.uint8)
        got = {n: s[n] for n in names[2:]} | {"k_held": held[0], "v_held": held[1]}
    return got | {n: got[n].view(torch.uint8) for n in names[4:]}


def _run_attend(s):
    if own:
        from qwarz_b200 import batch

        if "workspace" not in s:  # kept by a user for all layers and steps
            s["workspace"] = batch.attend_workspace(s["q"].device, s["k_cache"].shape[-1] * 2)
        batch.attend(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"], s["cu_rows"],
                     s["kv_lens"], s["out"], s["workspace"], max_rows=s["max_rows"])
        return s["out"]
    q = s["q"].float()
    T, Hq, D = q.shape
    H = s["k_cache"].shape[2]
    G, N, S = Hq // H, s["max_rows"], _pages(s["max_kv"]) * PAGE
    cu, kv = s["cu_rows"].long(), s["kv_lens"].long()
    new = cu[1:] - cu[:-1]
    B = kv.numel()
    dev = q.device
    n = torch.arange(N, device=dev)
    rows = (cu[:-1, None] + n).clamp(max=T - 1)
    qp = q[rows].view(B, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * N, D)
    pages = s["table"].long().clamp(min=0)

    def dense(cache, scales):
        byte = cache[pages]
        code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
        return _values(code, scales.view(torch.uint8)[pages].view(torch.float8_e4m3fn)).flatten(1, 2).transpose(1, 2)

    sc = (qp @ dense(s["k_cache"], s["k_scales"]).transpose(2, 3)) * D ** -0.5
    limit = (kv - new)[:, None] + n + 1
    seen = torch.arange(S, device=dev) < limit[:, :, None]
    sc = sc.view(B, H, G, N, S).masked_fill_(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(B, H, G * N, S) @ dense(s["v_cache"], s["v_scales"])
    o = torch.where(total > 0, o.view(B, H, G, N, D) / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)
    out = torch.zeros(T, Hq, D, dtype=s["out"].dtype, device=dev)
    mine = n < new[:, None]
    out[rows[mine]] = o[mine].to(out.dtype)
    return out


def _run_logprobs(s):
    if own:
        from qwarz_b200 import scoring

        if "workspace" not in s:  # kept by a user for every step
            s["workspace"] = scoring.workspace(s["logits"].device, *s["logits"].shape, s["top"])
        scoring.token_logprobs(s["logits"], s["ids"], s["logprob"], s["entropy"], s["top_logprobs"], s["top_ids"],
                               s["workspace"])
        return {k: s[k] for k in ("logprob", "entropy", "top_logprobs", "top_ids")}
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    mean = torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True) / total
    value, at = torch.sort(x, dim=-1, descending=True, stable=True)  # equal values keep their order: lowest index first
    return {"logprob": (x.gather(1, s["ids"][:, None]) - lse)[:, 0], "entropy": (torch.log(total) - mean)[:, 0],
            "top_logprobs": value[:, :s["top"]] - lse, "top_ids": at[:, :s["top"]].to(torch.int32)}


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "tables":
        kv, new = _lengths(case)
        B = case["requests"]
        grown = sum(_pages(n) - _pages(n - r) for n, r in zip(kv, new))
        return {"bytes": 4 * (3 * B + 2) + 4 * (3 * B + 3) + 8 * grown + 12 * sum(new), "flops": 0}
    if case["op"] == "append":
        n = case["rows"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": n * 2 + n // 2 + n // 16 + n * 2 + 4 * case["rows"], "flops": 6 * n}
    if case["op"] == "attend":
        kv, new = _lengths(case)
        Hq, H, D = case["heads"], case["kv_heads"], case["dim"]
        read = sum(n for n, r in zip(kv, new) if r)
        pairs = sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(kv, new))
        return {"bytes": read * H * 2 * (D // 2 + D // 16) + sum(new) * Hq * D * 4 + 4 * sum(_pages(n) for n in kv),
                "flops": 4 * D * Hq * pairs}
    T, V = case["rows"], case["vocab"]
    return {"bytes": T * V * (4 if case["type"] == "f32" else 2) + T * (16 + 8 * case["top"]), "flops": 6 * T * V}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    return None


def _grid64(y):
    """Nearest of the E2M1 magnitudes, ties to the even code, by distance."""
    grid = torch.tensor(MAGS, dtype=torch.float64, device=y.device)
    d = (y.abs().unsqueeze(-1) - grid).abs()
    # of two equally near magnitudes the one with the even code wins
    d = d + torch.tensor([0, 1] * 4, dtype=torch.float64, device=y.device) * 1e-9
    return grid[d.argmin(-1)] * torch.sign(y)


def _exact_append(s):
    out = {n: None for n in ("k_cache", "v_cache", "k_scales", "v_scales")}
    byte = torch.arange(127, dtype=torch.uint8, device="cuda")
    e4m3 = byte.view(torch.float8_e4m3fn).double()  # 0 .. 448, ascending
    mid = (e4m3[1:] + e4m3[:-1]) / 2
    for name in ("k", "v"):
        parts = []
        for x in s[name].split(1024):
            b = x.double().reshape(*x.shape[:-1], -1, 16)
            want = b.abs().amax(-1) / 6
            up = torch.bucketize(want, mid, right=False)  # a tie stays below ...
            tie = (up < mid.numel()) & (mid[up.clamp(max=mid.numel() - 1)] == want) & (up % 2 == 1)
            sc = e4m3[(up + tie).clamp(max=126)].unsqueeze(-1)  # ... unless the code above is even
            y = torch.where(sc > 0, b / torch.where(sc > 0, sc, 1.0), 0.0).clamp(-6, 6)
            parts.append((_grid64(y) * sc).reshape(x.shape))
        out[name + "_held"] = torch.cat(parts)
    return out


def _exact_attend(s):
    q, cu, kv = s["q"].double(), s["cu_rows"].tolist(), s["kv_lens"].tolist()
    T, Hq, D = q.shape
    H = s["k_cache"].shape[2]
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)

    def rows(cache, scales, pages, n, h):
        c = cache[pages, :, h].flatten(0, 1)[:n]
        c = torch.stack((c % 16, c // 16), -1).flatten(1).double()
        sign, mag = torch.where(c >= 8, -1.0, 1.0).double(), c % 8
        mag = torch.where(mag < 2, mag / 2, (1 + (mag % 2) / 2) * 2.0 ** ((mag // 2) - 1))
        return sign * mag * scales[pages, :, h].flatten(0, 1)[:n].double().repeat_interleave(16, 1)

    for b, n in enumerate(kv):
        r = cu[b + 1] - cu[b]
        if not r:
            continue
        pages = s["table"][b, :_pages(n)].long()
        causal = torch.arange(n, device=q.device)[None] <= torch.arange(n - r, n, device=q.device)[:, None]
        for h in range(H):
            k = rows(s["k_cache"], s["k_scales"], pages, n, h)
            v = rows(s["v_cache"], s["v_scales"], pages, n, h)
            mine = q[cu[b]:cu[b + 1], h * (Hq // H):(h + 1) * (Hq // H)].transpose(0, 1)
            w = (mine @ k.T / math.sqrt(D)).masked_fill(~causal, -math.inf).softmax(-1)
            out[cu[b]:cu[b + 1], h * (Hq // H):(h + 1) * (Hq // H)] = (w @ v).transpose(0, 1)
    return out


def _exact_logprobs(s):
    K = s["top"]
    parts = []
    for x, i in zip(s["logits"].split(64), s["ids"].split(64)):
        lp = x.double().log_softmax(-1)
        p = lp.exp()
        parts.append((lp.gather(1, i[:, None])[:, 0], torch.special.entr(p).sum(-1), lp.topk(K, -1).values))
    a, b, c = (torch.cat(p) for p in zip(*parts))
    return {"logprob": a, "entropy": b, "top_logprobs": c, "top_ids": None}
