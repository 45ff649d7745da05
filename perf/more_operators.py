"""Cases of the operators with which requests that share a prompt prefix are
served from one NVFP4 pool, in the order in which a step uses them:

  share   the step's rows sorted by the prefix they read, positions behind it
  rotate  Q and K normed and rotated by position, K and V quantised into their slots
  attend  attention of every row over its prefix, read once for all, and its own pages

A prefix is a request of the batch that holds tokens and adds none.  `own`
chooses between the plain form (elementary torch operations) and the
framework's operators.  Lengths follow from the case alone, values from the seed.
"""
import math
import random

import torch

own = False

PAGE = 256
MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, KV heads, head dim): the cache's own layout first, then generic ones
LAYOUTS = ((24, 4, 256), (32, 8, 128), (16, 2, 128), (8, 8, 64), (14, 2, 64), (40, 8, 128), (16, 1, 256))


def listed():
    return [
        # a decode step of 64 chats behind two system prompts (latency)
        {"name": "share decode 64", "op": "share", "readers": 64, "prefixes": 2, "prefix_lo": 1000, "prefix_hi": 8000,
         "kv_lo": 1, "kv_hi": 4000, "rows": "decode", "free": 0.1, "mix": 1},
        # a full server: decode rows, windows and prompt chunks behind 24 prompts
        {"name": "share mixed 2048", "op": "share", "readers": 2048, "prefixes": 24, "prefix_lo": 300,
         "prefix_hi": 30000, "kv_lo": 1, "kv_hi": 8000, "rows": "mixed", "free": 0.2, "mix": 2},
        # a decode step of 16 requests, a quarter of the head dims rotated, Q and K normed (latency)
        {"name": "rotate decode 16", "op": "rotate", "rows": 16, "heads": 24, "kv_heads": 4, "dim": 256, "rotary": 64,
         "pairs": "half", "norm": True, "type": "bf16", "far": 65536},
        # the 7-row windows of 64 requests, whole heads rotated
        {"name": "rotate windows 64x7", "op": "rotate", "rows": 448, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "pairs": "half", "norm": False, "type": "f16", "far": 131072},
        # an odd prompt budget of a small model, neighbouring dims paired
        {"name": "rotate prompts 5001 d64", "op": "rotate", "rows": 5001, "heads": 14, "kv_heads": 2, "dim": 64,
         "rotary": 32, "pairs": "neighbours", "norm": False, "type": "f16", "far": 8192},
        # a prompt chunk budget of 16,384 rows at far positions
        {"name": "rotate prompts 16384", "op": "rotate", "rows": 16384, "heads": 24, "kv_heads": 4, "dim": 256,
         "rotary": 64, "pairs": "half", "norm": True, "type": "bf16", "far": 262144},
        # four chats behind a short system prompt (latency)
        {"name": "attend decode 4 behind 2000", "op": "attend", "readers": 4, "prefixes": 1, "prefix_lo": 2000,
         "prefix_hi": 2000, "kv_lo": 20, "kv_hi": 500, "rows": "decode", "free": 0.0, "heads": 24, "kv_heads": 4,
         "dim": 256, "type": "f16", "mix": 3},
        # 64 chats over one long document
        {"name": "attend decode 64 behind 32768", "op": "attend", "readers": 64, "prefixes": 1, "prefix_lo": 32768,
         "prefix_hi": 32768, "kv_lo": 20, "kv_hi": 2000, "rows": "decode", "free": 0.0, "heads": 24, "kv_heads": 4,
         "dim": 256, "type": "bf16", "mix": 4},
        # many chats behind a handful of prompts, some without one, on a 32/8/128 head layout
        {"name": "attend decode 256 d128", "op": "attend", "readers": 256, "prefixes": 6, "prefix_lo": 1000,
         "prefix_hi": 16384, "kv_lo": 10, "kv_hi": 1500, "rows": "decode", "free": 0.1, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f16", "mix": 5},
        # the 7-row verify windows of 24 requests over two documents
        {"name": "attend windows 24x7", "op": "attend", "readers": 24, "prefixes": 2, "prefix_lo": 8192,
         "prefix_hi": 32768, "kv_lo": 100, "kv_hi": 4000, "rows": "window", "free": 0.0, "heads": 24, "kv_heads": 4,
         "dim": 256, "type": "bf16", "mix": 6},
        # questions of a few hundred rows, windows and decode rows behind two prompts
        {"name": "attend questions 12", "op": "attend", "readers": 12, "prefixes": 2, "prefix_lo": 5000,
         "prefix_hi": 16384, "kv_lo": 60, "kv_hi": 900, "rows": "questions", "free": 0.1, "heads": 24, "kv_heads": 4,
         "dim": 256, "type": "bf16", "mix": 7},
        # every request behind a prompt of its own: nothing to share at this moment
        {"name": "attend decode 48 apart", "op": "attend", "readers": 48, "prefixes": 48, "prefix_lo": 500,
         "prefix_hi": 6000, "kv_lo": 10, "kv_hi": 1000, "rows": "decode", "free": 0.0, "heads": 14, "kv_heads": 2,
         "dim": 64, "type": "f16", "mix": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("share", "rotate", "rotate", "attend", "attend", "attend"))
    mix = rng.randrange(1 << 20)
    if op == "share":
        hi = _log(rng, 2, 30000)
        return {"op": op, "readers": _log(rng, 1, 2048), "prefixes": _log(rng, 1, 64), "prefix_lo": 1 + hi // 10,
                "prefix_hi": hi, "kv_lo": 1, "kv_hi": _log(rng, 2, 8000),
                "rows": rng.choice(("decode", "window", "mixed")), "free": rng.choice((0.0, 0.3)), "mix": mix}
    heads, kv_heads, dim = rng.choice(LAYOUTS)
    if op == "rotate":
        return {"op": op, "rows": min(_log(rng, 1, 16384), 100_000_000 // ((heads + 2 * kv_heads) * dim)),
                "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([r for r in (16, 32, 48, 64, 96, 128, 256) if r <= dim]),
                "pairs": rng.choice(("half", "neighbours")), "norm": rng.random() < 0.5,
                "type": rng.choice(("f16", "bf16")), "far": _log(rng, 100, 1_000_000)}
    rows = rng.choice(("decode", "decode", "window", "questions"))
    readers = _log(rng, 1, 256 if rows == "decode" else 32)
    prefixes = min(readers, rng.choice((1, 1, 2, 5, readers)))
    # readers x longest prefix x query width at most what "attend decode 64 behind 32768" has
    wide = readers * {"decode": 1, "window": 7, "questions": 128}[rows] * heads * dim
    hi = _log(rng, 2, max(4, min(32768, 64 * 32768 * 24 * 256 // wide, 65536 * 1024 // (prefixes * kv_heads * dim))))
    return {"op": op, "readers": readers, "prefixes": prefixes, "prefix_lo": 1 + hi // rng.choice((1, 4, 30)),
            "prefix_hi": hi, "kv_lo": 1, "kv_hi": _log(rng, 2, 2000), "rows": rows, "free": rng.choice((0.0, 0.2)),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": rng.choice(("f16", "bf16")), "mix": mix}


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """Tokens after the step, rows of the step and the prefix (-1: none) of every
    request; the prefixes come first."""
    rng = random.Random(case["mix"])
    kv, new, prefix = [], [], []
    P = case["prefixes"]
    for _ in range(P):
        lo, hi = min(case["prefix_lo"], case["prefix_hi"]), case["prefix_hi"]
        kv.append(_log(rng, lo, hi) if hi > lo else hi)
        new.append(0)
        prefix.append(-1)
    for i in range(case["readers"]):
        lo, hi = min(case["kv_lo"], case["kv_hi"]), case["kv_hi"]
        n = _log(rng, lo, hi) if hi > lo else hi
        mode = case["rows"]
        if mode == "mixed":
            mode = rng.choice(("decode", "decode", "window", "chunk", "idle"))
        elif mode == "questions":
            mode = ("chunk", "question", "decode", "question", "window", "chunk")[i % 6]
        r = {"decode": 1, "window": 7, "chunk": _log(rng, 9, 256), "question": n, "idle": 0}[mode]
        kv.append(n)
        new.append(min(r, n, 256))
        # as many prefixes as requests: one each; otherwise the first ones are the popular ones
        mine = i if P == case["readers"] else min(int(P * rng.random() ** 1.5), P - 1)
        prefix.append(-1 if rng.random() < case["free"] else mine)
    return kv, new, prefix


def _pages(n):
    return (n + PAGE - 1) // PAGE


# ------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(values):
    at = [0]
    for v in values:
        at.append(at[-1] + v)
    return at


def _quantise(x):
    """[..., D] -> (E2M1 codes [..., D], E4M3 scales [..., D/16]) as whole numbers:
    amax / 6 rounded to E4M3, x / scale to E2M1, both to nearest, ties to even."""
    b = x.view(*x.shape[:-1], -1, 16)
    grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).to(x.dtype)
    want = (b.abs().amax(-1) / 6).clamp(max=448.0)
    lo = (torch.searchsorted(grid, want, right=True) - 1).clamp(0, 125)  # grid[lo] <= want
    mid = (grid[lo] + grid[lo + 1]) / 2
    scale = lo + ((want > mid) | ((want == mid) & (lo % 2 == 1)))
    s = grid[scale].unsqueeze(-1)
    y = torch.where(s > 0, b / torch.where(s > 0, s, 1.0), 0.0)
    a = y.abs()
    m = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where((m > 0) & (y < 0), m + 8, m)
    return code.to(torch.uint8).view(x.shape), scale.to(torch.uint8)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(code, scale):
    """The FP32 values that codes and E4M3 scale bytes stand for."""
    lut = torch.tensor(MAGS + tuple(-m for m in MAGS), device=code.device)
    v = lut[code.long()]
    s = scale.view(torch.float8_e4m3fn).float()
    return (v.view(*v.shape[:-1], -1, 16) * s.unsqueeze(-1)).view(v.shape)


def _pool(pages, kv_heads, dim, g):
    """A pool filled with quantised rows: unit normal with a few strong channels."""
    codes = torch.empty(pages, PAGE, kv_heads, dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, PAGE, kv_heads, dim // 16, dtype=torch.uint8, device="cuda")
    gain = torch.exp(0.3 * torch.randn(kv_heads, dim, generator=g, device="cuda"))
    step = max(1, (1 << 25) // (PAGE * kv_heads * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        code, scale = _quantise(torch.randn(n, PAGE, kv_heads, dim, generator=g, device="cuda") * gain)
        codes[at:at + n] = _pack(code)
        scales[at:at + n] = scale
    return codes, scales.view(torch.float8_e4m3fn)


def prepare(case, seed):
    return {"share": _prepare_share, "rotate": _prepare_rotate, "attend": _prepare_attend}[case["op"]](case, seed)


def _prepare_share(case, seed):
    g = _generator(seed)
    kv, new, prefix = _lengths(case)
    # the same requests in an order of the seed's
    order = torch.randperm(len(kv), generator=g, device="cuda")
    place = torch.empty_like(order)
    place[order] = torch.arange(len(kv), device="cuda")
    kv, new, prefix = _int(kv)[order], _int(new)[order], _int(prefix)[order]
    prefix = torch.where(prefix >= 0, place[prefix.clamp(min=0).long()], -1).to(torch.int32)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)
    T = int(cu[-1])
    req = torch.repeat_interleave(torch.arange(len(kv), device="cuda"), new.long())
    pos = (kv - new)[req] + torch.arange(T, device="cuda") - cu[req]
    return {"op": "share", "prefix_of": prefix, "kv_lens": kv, "cu_rows": cu, "positions": pos.to(torch.int32),
            "request_of": req.to(torch.int32), "positions_out": torch.empty(T, dtype=torch.int32, device="cuda"),
            "plan": torch.empty(3 * len(kv) + 1 + T, dtype=torch.int32, device="cuda")}


def _prepare_rotate(case, seed):
    g = _generator(seed)
    T, Hq, H, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    dt = TYPES[case["type"]]
    # Q, K and V are parts of the projection's packed rows; K has strong channels
    x = torch.randn(T, Hq + 2 * H, D, generator=g, device="cuda")
    x[:, Hq:Hq + H] *= torch.exp(0.3 * torch.randn(H, D, generator=g, device="cuda"))
    x = (x * 1.5).to(dt)
    pages = _pages(T) + 3
    slots = torch.randperm(pages, generator=g, device="cuda")[:_pages(T)]
    slots = (slots[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:T].to(torch.int32)
    base = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda"))
    half = case["rotary"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    weight = lambda: torch.exp(0.2 * torch.randn(D, generator=g, device="cuda")) if case["norm"] else None  # noqa: E731
    shape = (pages, PAGE, H)
    return {"op": "rotate", "q": x[:, :Hq], "k": x[:, Hq:Hq + H], "v": x[:, Hq + H:], "slots": slots,
            # a prompt's rows, or rows of requests far apart
            "positions": ((base + torch.arange(T, device="cuda") * (1 if T > 1000 else 977)) % case["far"]).to(torch.int32),
            "inv_freq": freq.float(), "neighbours": case["pairs"] == "neighbours", "q_weight": weight(),
            "k_weight": weight(), "q_out": torch.empty(T, Hq, D, dtype=dt, device="cuda"),
            "k_cache": torch.zeros(*shape, D // 2, dtype=torch.uint8, device="cuda"),
            "v_cache": torch.zeros(*shape, D // 2, dtype=torch.uint8, device="cuda"),
            "k_scales": torch.zeros(*shape, D // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            "v_scales": torch.zeros(*shape, D // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            "k_held": torch.empty(T, H, D, dtype=dt, device="cuda"),
            "v_held": torch.empty(T, H, D, dtype=dt, device="cuda")}


def _prepare_attend(case, seed):
    g = _generator(seed)
    kv, new, prefix = _lengths(case)
    Hq, H, D, P = case["heads"], case["kv_heads"], case["dim"], case["prefixes"]
    dt = TYPES[case["type"]]
    width = _pages(max(kv))
    total = sum(_pages(n) for n in kv)
    k_cache, k_scales = _pool(total + 1, H, D, g)
    v_cache, v_scales = _pool(total + 1, H, D, g)
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda")[None] < _int([_pages(n) for n in kv])[:, None]
    table[used] = torch.randperm(total + 1, generator=g, device="cuda")[:total].to(torch.int32)
    cu = _sums(new)
    T = cu[-1]
    packed = torch.randn(T, Hq + 2 * H, D, generator=g, device="cuda") * 1.5
    # the step's plan, as the share operator makes it (once for all layers)
    behind = [[b for b in range(len(kv)) if prefix[b] == p and new[b]] for p in range(len(kv))]
    rows = [[r for b in bs for r in range(cu[b], cu[b + 1])] for bs in behind]
    plan = _sums([len(r) for r in rows]) + prefix + [bs[0] if len(bs) == 1 else -1 for bs in behind]
    listed_rows = [r for rs in rows for r in rs]
    plan += listed_rows + [-1] * (T - len(listed_rows))
    return {"op": "attend", "q": packed.to(dt)[:, :Hq], "k_cache": k_cache, "v_cache": v_cache,
            "k_scales": k_scales, "v_scales": v_scales, "table": table, "cu_rows": _int(cu), "kv_lens": _int(kv),
            "prefix_of": _int(prefix), "plan": _int(plan), "prefixes": P, "max_rows": max(max(new), 1),
            "max_kv": max(kv[P:]), "max_prefix": max(kv[:P]), "max_shared": max(max(len(r) for r in rows), 1),
            "out": torch.zeros(T, Hq, D, dtype=dt, device="cuda")}


# ------------------------------------------------------------------- passes
def run(state):
    return {"share": _run_share, "rotate": _run_rotate, "attend": _run_attend}[state["op"]](state)


def _run_share(s):
    R, T = s["kv_lens"].numel(), s["positions"].numel()
    if own:
        from qwarz_b200 import batch

        batch.share_prefixes(s["prefix_of"], s["kv_lens"], s["cu_rows"], s["positions"], s["request_of"], s["plan"],
                             s["positions_out"])
        cu, prefix, alone, rows = s["plan"].split([R + 1, R, R, T])
        return {"cu_shared": cu, "prefix": prefix, "alone": alone, "rows": rows, "positions": s["positions_out"]}
    prefix, kv, cu, req = (s[n].long() for n in ("prefix_of", "kv_lens", "cu_rows", "request_of"))
    # a prefix has none itself
    prefix = torch.where((prefix >= 0) & (prefix[prefix.clamp(min=0)] < 0), prefix, -1)
    new = cu[1:] - cu[:-1]
    at = prefix.clamp(min=0)
    behind = torch.where(prefix >= 0, new, 0)
    count = torch.zeros(R, dtype=torch.long, device=kv.device)
    cu_shared = torch.cat([count.new_zeros(1), count.scatter_add(0, at, behind).cumsum(0)])
    some = (behind > 0).long()
    alone = torch.where(count.scatter_add(0, at, some) == 1,
                        count.scatter_add(0, at, some * torch.arange(R, device=kv.device)), -1)
    mine = prefix[req]
    order = torch.sort(torch.where(mine >= 0, mine, R), stable=True).indices
    rows = torch.where(torch.arange(T, device=kv.device) < cu_shared[-1], order, -1)
    positions = s["positions"].long() + torch.where(mine >= 0, kv[mine.clamp(min=0)], 0)
    i32 = torch.int32
    return {"cu_shared": cu_shared.to(i32), "prefix": prefix.to(i32), "alone": alone.to(i32), "rows": rows.to(i32),
            "positions": positions.to(i32)}


def _rotated(x, weight, cos, sin, neighbours, eps=1e-6):
    """x [T, heads, D] normed (where there is a weight) and its first dims rotated, in x's own precision."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype)
    h = cos.shape[-1]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if neighbours else (x[..., :h], x[..., h:2 * h])
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * h:]], -1)


def _run_rotate(s):
    names = ("q_out", "k_held", "v_held", "k_cache", "v_cache", "k_scales", "v_scales")
    if own:
        from qwarz_b200 import batch

        batch.append_rotated(s["q"], s["k"], s["v"], s["q_out"], s["k_cache"], s["v_cache"], s["k_scales"],
                             s["v_scales"], s["slots"], s["positions"], s["inv_freq"], neighbours=s["neighbours"],
                             q_weight=s["q_weight"], k_weight=s["k_weight"], k_held=s["k_held"], v_held=s["v_held"])
        got = {n: s[n] for n in names}
    else:
        at, dt = s["slots"].long(), s["q"].dtype
        # far positions have angles that 32 bits do not hold, and K lies next to rounding borders: 64 bits
        angle = s["positions"].double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos(), angle.sin()
        q = _rotated(s["q"].float(), s["q_weight"], cos, sin, s["neighbours"])
        got = {"q_out": q.to(dt)}
        for n, x in (("k", _rotated(s["k"].double(), s["k_weight"], cos, sin, s["neighbours"])), ("v", s["v"].float())):
            code, scale = _quantise(x)
            got[n + "_held"] = _values(code, scale).to(dt)
            s[n + "_cache"].flatten(0, 1)[at] = _pack(code)
            s[n + "_scales"].view(torch.uint8).flatten(0, 1)[at] = scale
        got |= {n: s[n] for n in names[3:]}
    return got | {n: got[n].view(torch.uint8) for n in names[5:]}


def _run_attend(s):
    if own:
        from qwarz_b200 import batch

        T, Hq, D = s["q"].shape
        if "workspace" not in s:  # kept by a user for all layers and steps
            s["workspace"] = batch.shared_workspace(s["q"].device, D, T, Hq)
        batch.attend_shared(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"],
                            s["cu_rows"], s["kv_lens"], s["plan"], s["out"], s["workspace"], max_rows=s["max_rows"])
        return s["out"]
    q = s["q"].float()
    T, Hq, D = q.shape
    H = s["k_cache"].shape[2]
    G, P, R = Hq // H, s["prefixes"], s["kv_lens"].numel()
    cu, kv, dev = s["cu_rows"].long(), s["kv_lens"].long(), q.device
    cu_shared, prefix, _, by_prefix = s["plan"].long().split([R + 1, R, R, T])
    new = cu[1:] - cu[:-1]

    def part(rows, there, requests, limit, most):
        """(max, sum, unnormalised output) of the rows [B, N] of the given requests, which see `limit` [B, N] tokens."""
        B, N = rows.shape
        S = _pages(most) * PAGE
        pages = s["table"][requests, :_pages(most)].long().clamp(min=0)

        def dense(cache, scales):
            byte = cache[pages]
            code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
            return _values(code, scales.view(torch.uint8)[pages]).flatten(1, 2).transpose(1, 2)

        qp = q[rows.clamp(0, T - 1)].view(B, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * N, D)
        sc = ((qp @ dense(s["k_cache"], s["k_scales"]).transpose(2, 3)) * D ** -0.5).view(B, H, G, N, S)
        sc.masked_fill_(~(torch.arange(S, device=dev) < limit[:, :, None])[:, None, None], -math.inf)
        top = sc.amax(-1)
        p = sc.sub_(torch.where(top == -math.inf, 0.0, top).unsqueeze(-1)).exp_()
        o = (p.view(B, H, G * N, S) @ dense(s["v_cache"], s["v_scales"])).view(B, H, G, N, D)
        at = rows[there]
        full = [torch.full((T, H, G), -math.inf, device=dev), torch.zeros(T, H, G, device=dev),
                torch.zeros(T, H, G, D, device=dev)]
        for f, x in zip(full, (top, p.sum(-1), o)):
            f[at] = x.movedim(3, 1)[there]
        return full

    n = torch.arange(s["max_shared"], device=dev)
    there = n < (cu_shared[1:] - cu_shared[:-1])[:P, None]
    shared = by_prefix[(cu_shared[:P, None] + n).clamp(max=T - 1)]
    m0, l0, o0 = part(shared, there, torch.arange(P, device=dev), torch.where(there, kv[:P, None], 0), s["max_prefix"])
    n = torch.arange(s["max_rows"], device=dev)
    m1, l1, o1 = part(cu[P:-1, None] + n, n < new[P:, None], torch.arange(P, R, device=dev),
                      (kv - new)[P:, None] + n + 1, s["max_kv"])
    m = torch.maximum(m0, m1)
    w0, w1 = (torch.where(x == -math.inf, 0.0, torch.exp(x - m)) for x in (m0, m1))
    total = w0 * l0 + w1 * l1
    o = (w0.unsqueeze(-1) * o0 + w1.unsqueeze(-1) * o1) / total.unsqueeze(-1)
    return torch.where(total.unsqueeze(-1) > 0, o, 0.0).reshape(T, Hq, D).to(s["out"].dtype)


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "share":
        kv, new, _ = _lengths(case)
        return {"bytes": 4 * (6 * len(kv) + 2 + 4 * sum(new)), "flops": 0}
    Hq, H, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        n = case["rows"] * H * D * 2
        return {"bytes": 4 * case["rows"] * Hq * D + 4 * n + n // 2 + n // 16 + 8 * case["rows"],
                "flops": case["rows"] * (6 * (Hq + H) * D + 12 * H * D)}
    kv, new, prefix = _lengths(case)
    read = sum(n for n, r in zip(kv, new) if r) + sum(kv[p] for p in {p for p, r in zip(prefix, new) if r} - {-1})
    pairs = sum(r * (n - r) + r * (r + 1) // 2 + (r * kv[p] if p >= 0 else 0) for n, r, p in zip(kv, new, prefix))
    return {"bytes": read * H * 2 * (D // 2 + D // 16) + sum(new) * Hq * D * 4 + 4 * sum(_pages(n) for n in kv),
            "flops": 4 * D * Hq * pairs}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "share":
        return None
    s = prepare(case, seed)
    return _exact_rotate(s) if case["op"] == "rotate" else _exact_attend(s)


def _exact_turn(x, weight, positions, freq, neighbours):
    """Rows x [T, heads, D] as complex numbers times e^(i angle)."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * weight.double()
    h = freq.numel()
    angle = torch.outer(positions.double(), freq.double()).unsqueeze(1)
    i = torch.arange(h, device=x.device)
    re, im = (2 * i, 2 * i + 1) if neighbours else (i, i + h)
    z = torch.complex(x[..., re], x[..., im]) * torch.polar(torch.ones_like(angle), angle)
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_held(x):
    """What an NVFP4 cache holds for the 64-bit rows x."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    e4m3 = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    mid = (e4m3[1:] + e4m3[:-1]) / 2
    want = b.abs().amax(-1) / 6
    up = torch.bucketize(want, mid)  # a tie stays below ...
    tie = (up < mid.numel()) & (mid[up.clamp(max=mid.numel() - 1)] == want) & (up % 2 == 1)
    s = e4m3[(up + tie).clamp(max=126)].unsqueeze(-1)  # ... unless the code above is even
    y = torch.where(s > 0, b / torch.where(s > 0, s, 1.0), 0.0).clamp(-6, 6)
    grid = torch.tensor(MAGS, dtype=torch.float64, device=x.device)
    d = (y.abs().unsqueeze(-1) - grid).abs() + torch.tensor([0, 1] * 4, device=x.device) * 1e-12
    return (grid[d.argmin(-1)] * torch.sign(y) * s).reshape(x.shape)


def _exact_rotate(s):
    got = {n: None for n in ("k_cache", "v_cache", "k_scales", "v_scales")}
    parts = []
    for at in torch.arange(s["positions"].numel(), device="cuda").split(1024):
        q, k = (_exact_turn(s[n][at], s[n + "_weight"], s["positions"][at], s["inv_freq"], s["neighbours"])
                for n in ("q", "k"))
        parts.append((q, _exact_held(k), _exact_held(s["v"][at].double())))
    return got | dict(zip(("q_out", "k_held", "v_held"), (torch.cat(p) for p in zip(*parts))))


def _exact_attend(s):
    q, cu, kv, prefix = s["q"].double(), s["cu_rows"].tolist(), s["kv_lens"].tolist(), s["prefix_of"].tolist()
    T, Hq, D = q.shape
    H = s["k_cache"].shape[2]
    G = Hq // H
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)

    def tokens(cache, scales, b, h):
        pages = s["table"][b, :_pages(kv[b])].long()
        c = cache[pages, :, h].flatten(0, 1)[:kv[b]]
        c = torch.stack((c % 16, c // 16), -1).flatten(1).double()
        sign, mag = torch.where(c >= 8, -1.0, 1.0).double(), c % 8
        mag = torch.where(mag < 2, mag / 2, (1 + (mag % 2) / 2) * 2.0 ** ((mag // 2) - 1))
        return sign * mag * scales[pages, :, h].flatten(0, 1)[:kv[b]].double().repeat_interleave(16, 1)

    for h in range(H):
        first = {p: [tokens(s[n + "_cache"], s[n + "_scales"], p, h) for n in ("k", "v")] for p in set(prefix) - {-1}}
        for b, n in enumerate(kv):
            r = cu[b + 1] - cu[b]
            if not r:
                continue
            k, v = (tokens(s[x + "_cache"], s[x + "_scales"], b, h) for x in ("k", "v"))
            before = 0
            if prefix[b] >= 0:
                before = kv[prefix[b]]
                k, v = torch.cat([first[prefix[b]][0], k]), torch.cat([first[prefix[b]][1], v])
            last = before + n - r + torch.arange(r, device=q.device)
            seen = torch.arange(before + n, device=q.device)[None] <= last[:, None]
            mine = q[cu[b]:cu[b + 1], h * G:(h + 1) * G].transpose(0, 1)
            w = (mine @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf).softmax(-1)
            out[cu[b]:cu[b + 1], h * G:(h + 1) * G] = (w @ v).transpose(0, 1)
    return out
