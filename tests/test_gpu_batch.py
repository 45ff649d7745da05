"""The operators that serve many requests from one NVFP4 pool (qwarz_b200.batch)
against plain 64-bit forms (oracle/batch.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import batch as obatch
from oracle import nvfp4
from qwarz_b200 import _lib, batch, ops

pytestmark = pytest.mark.gpu
PAGE = 256


@pytest.fixture(autouse=True)
def clean_errors(cuda):
    _lib.device_error(clear=True)
    yield
    assert _lib.device_error(clear=True) == 0  # a test that expects a bit clears it itself


def i32(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------- tables
def run_tables(lengths, new_rows, held, pool, width, rows, head=0, seed=0, count=None):
    g = np.random.default_rng(seed)
    ids = g.permutation(pool)
    total = int(np.sum(held))
    table = np.full((len(lengths), width), -1)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    count = pool - total if count is None else count
    ring = np.full(pool, -1)
    ring[(head + np.arange(count)) % pool] = ids[total:total + count]
    want, why = obatch.build_tables(lengths, new_rows, held, ring, (head, count), table, rows)
    R = len(lengths)
    got = {"block_table": i32(table), "ring": i32(ring), "cu_rows": i32([-7] * (R + 1)), "kv_lens": i32([-7] * R),
           "held_out": i32([-7] * R), "ring_out": i32([-7, -7]), "slots": i32([-7] * rows),
           "positions": i32([-7] * rows), "request_of": i32([-7] * rows)}
    for _ in range(2):  # the same state gives the same step again
        batch.build_tables(i32(lengths), i32(new_rows), i32(held), got["ring"], i32([head, count]), got["block_table"],
                           got["cu_rows"], got["kv_lens"], got["held_out"], got["ring_out"], got["slots"],
                           got["positions"], got["request_of"])
        for name, t in got.items():
            assert np.array_equal(t.cpu().numpy(), want[name]), name
    return want, why


@pytest.mark.parametrize("lengths,new_rows,held,extra", [
    ([0], [1], [0], 0),                                   # the first token of a request
    ([255], [1], [1], 0), ([256], [1], [1], 0),           # to and past a page's end
    ([0, 5, 700], [0, 0, 0], [0, 1, 3], 0),               # nothing to do
    ([0, 300, 511, 512, 1], [600, 7, 1, 1, 513], [0, 2, 2, 2, 1], 3),  # windows and chunks, rows past the end
    ([100, 900, 40, 0], [-1, 8, -1, 300], [2, 4, 1, 0], 5),  # requests that end, held pages beyond the length
])
def test_tables_small(lengths, new_rows, held, extra):
    rows = sum(max(n, 0) for n in new_rows) + extra
    _, why = run_tables(lengths, new_rows, held, 24, 8, rows, head=20)
    assert not why


def test_tables_denied():
    # 3 free pages: request 1 does not get its 2, nor does any later one that needs some; one without need goes on
    want, why = run_tables([0, 0, 0, 10], [512, 512, 1, 1], [0, 0, 0, 1], 10, 4, 1026, count=3)
    assert why == {"empty"} and want["kv_lens"].tolist() == [512, 0, 0, 11]
    assert _lib.device_error(clear=True) == 16
    # a request longer than its table row
    want, why = run_tables([1000, 3], [100, 1], [4, 1], 12, 4, 101)
    assert why == {"wide"} and want["kv_lens"].tolist() == [0, 4]
    assert _lib.device_error(clear=True) == 1


@pytest.mark.parametrize("R", [1, 33, 1024, 1500])
def test_tables_many(R):
    g = np.random.default_rng(R)
    lengths = g.integers(0, 3000, R)
    new_rows = g.choice([0, 1, 1, 7, 300, -1], R)
    held = -(-lengths // PAGE) + g.integers(0, 2, R)
    rows = int(np.maximum(new_rows, 0).sum()) + 11
    pool = int(held.sum() + R * 3 + 8)
    _, why = run_tables(lengths, new_rows, held, pool, 16, rows, head=pool - 5, seed=R)
    assert not why


@pytest.mark.parametrize("head,count", [(16, 3), (-1, 3), (2, 17), (2, -1)])
def test_tables_bad_ring_state(head, count):
    """A ring state that cannot be: no page moves, no request keeps rows of the
    step (all slots -1, kv_lens 0 where there are rows), and the state that
    comes out is the one that went in."""
    lengths, new_rows, held, width, rows = [10, 300, 0, 700, 5, 900], [3, -1, 600, 1, 0, 200], [1, 2, 0, 3, 1, 4], 4, 810
    table = np.arange(24).reshape(6, 4)
    ring = np.arange(16) + 30
    out = {"cu_rows": i32([-7] * 7), "kv_lens": i32([-7] * 6), "held_out": i32([-7] * 6), "ring_out": i32([-7, -7]),
           "slots": i32([-7] * rows), "positions": i32([-7] * rows), "request_of": i32([-7] * rows)}
    table_d, ring_d = i32(table), i32(ring)
    batch.build_tables(i32(lengths), i32(new_rows), i32(held), ring_d, i32([head, count]), table_d, *out.values())
    assert _lib.device_error(clear=True) == 2 | 1  # the state, and the last request, which does not fit its table row
    got = {k: t.tolist() for k, t in out.items()}
    assert got["cu_rows"] == [0, 3, 3, 603, 604, 604, 804]
    assert got["kv_lens"] == [0, 0, 0, 0, 5, 0]
    assert got["held_out"] == held and got["ring_out"] == [head, count]
    assert np.array_equal(table_d.cpu().numpy(), table) and np.array_equal(ring_d.cpu().numpy(), ring)
    assert got["slots"] == [-1] * rows
    assert got["request_of"] == [0] * 3 + [2] * 600 + [3] + [5] * 200 + [-1] * 6
    assert got["positions"] == [10, 11, 12] + list(range(600)) + [700] + list(range(900, 1100)) + [0] * 6


@pytest.mark.parametrize("wide", [1, 2, 3, 700])
def test_tables_rows_past_32_bits(wide):
    """Requests whose rows do not fit their tables, and whose sum does not fit 32
    bits: they are denied, the others get their pages in order, row offsets stop
    at the largest int32."""
    big = 2 ** 31 - 1
    lengths, new_rows = [0] + [0] * wide + [2048, 255, 0], [2] + [big] * wide + [3, 2, 300]
    held, pool, width, rows = [0] + [0] * wide + [8, 1, 0], 24, 8, 9
    table, ring = np.full((len(held), width), -1), np.arange(pool) + 50
    table[-3], table[-2, 0] = np.arange(8), 8
    want, why = obatch.build_tables(lengths, new_rows, held, ring, (20, 10), table, rows)
    assert why == {"wide"} and want["ring_out"].tolist() == [0, 6]
    want["cu_rows"] = np.minimum(want["cu_rows"], big)
    R = len(held)
    out = {"block_table": i32(table), "ring": i32(ring), "cu_rows": i32([-7] * (R + 1)), "kv_lens": i32([-7] * R),
           "held_out": i32([-7] * R), "ring_out": i32([-7, -7]), "slots": i32([-7] * rows),
           "positions": i32([-7] * rows), "request_of": i32([-7] * rows)}
    names = list(out)
    batch.build_tables(i32(lengths), i32(new_rows), i32(held), out["ring"], i32([20, 10]), out["block_table"],
                       *[out[n] for n in names[2:]])
    assert _lib.device_error(clear=True) == 1 | 4  # a table row too short, more rows than the slot map has
    for name, t in out.items():
        assert np.array_equal(t.cpu().numpy(), want[name]), name


def test_tables_pages_past_32_bits():
    """Denied requests may ask for more pages together than 32 bits count."""
    R, width = 520, 1 << 22
    lengths = [0] + [2 ** 30 - 1] * (R - 2) + [5]
    new_rows, held = [1] + [1] * (R - 2) + [1], [0] * (R - 1) + [1]
    table = torch.empty(R, width, dtype=torch.int32, device="cuda")
    table[R - 1, 0] = 3
    ring = i32([7, 8, 9, -1])
    out = [i32([-7] * (R + 1)), i32([-7] * R), i32([-7] * R), i32([-7, -7])] + [i32([-7] * R) for _ in range(3)]
    batch.build_tables(i32(lengths), i32(new_rows), i32(held), ring, i32([0, 3]), table, *out)
    assert _lib.device_error(clear=True) == 16
    assert out[0].tolist() == list(range(R + 1)) and out[3].tolist() == [1, 2]
    assert out[1].tolist() == [1] + [0] * (R - 2) + [6] and out[2].tolist() == [1] + [0] * (R - 2) + [1]
    assert out[4].tolist() == [7 * PAGE] + [-1] * (R - 2) + [3 * PAGE + 5]
    assert out[5].tolist() == [0] + [2 ** 30 - 1] * (R - 2) + [5]


def test_tables_ring_without_room():
    """Pages that find no place behind the free ones stay with the request that
    ends, and so do those of any that ends after it: no page is lost, and the
    count is of pages that are in the ring."""
    table = i32([[1, 2, -1], [3, -1, -1], [4, 5, -1], [6, -1, -1], [-1, -1, -1]])
    ring = i32([40, 41, -1, -1, 42])  # 42, 40, 41 are free
    out = {"cu_rows": i32([-7] * 6), "kv_lens": i32([-7] * 5), "held_out": i32([-7] * 5), "ring_out": i32([-7, -7]),
           "slots": i32([-7] * 3), "positions": i32([-7] * 3), "request_of": i32([-7] * 3)}
    for _ in range(2):
        batch.build_tables(i32([300, 10, 400, 20, 0]), i32([3, -1, -1, -1, -1]), i32([2, 1, 2, 1, 0]), ring,
                           i32([4, 3]), table, *out.values())
        assert _lib.device_error(clear=True) == 16
        got = {k: t.tolist() for k, t in out.items()}
        assert ring.tolist() == [40, 41, 3, -1, 42]  # one of two places taken: request 2 needs two, request 3 comes after it
        assert got["held_out"] == [2, 0, 2, 1, 0] and got["ring_out"] == [4, 4]
        assert got["kv_lens"] == [303, 0, 0, 0, 0] and got["cu_rows"] == [0, 3, 3, 3, 3, 3]
    # ended again once there is room
    ring2 = i32([40, 41, 3, -1, -1, -1, -1, 42])
    batch.build_tables(i32([303, 0, 0, 0, 0]), i32([300, 0, -1, -1, 0]), i32([2, 0, 2, 1, 0]), ring2, i32([7, 4]), table,
                       out["cu_rows"], out["kv_lens"], out["held_out"], out["ring_out"],
                       *[i32([0] * 300) for _ in range(3)])
    assert ring2.tolist() == [40, 41, 3, 4, 5, 6, -1, 42]
    assert out["held_out"].tolist() == [3, 0, 0, 0, 0] and out["ring_out"].tolist() == [0, 6]


# ------------------------------------------------------------------- append
def without_nan(x):
    """The device writers' rule for NaN, which the oracle's numpy maximum does not
    have: NaN does not count for a block's maximum and is stored as +6 times the
    scale (a block of nothing else as 0)."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    top = np.abs(np.where(np.isnan(b), 0.0, b)).max(-1, keepdims=True)
    return np.where(np.isnan(b), top, b).reshape(x.shape).astype(np.float32)


@pytest.mark.parametrize("heads,dim", [(4, 256), (8, 128), (1, 64), (3, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
def test_append_bytes(heads, dim, dtype, packed):
    T, pages = 77, 3
    g = torch.Generator().manual_seed(heads * dim)
    x = torch.randn(T, 4 * heads, dim, generator=g) * torch.exp(2 * torch.randn(T, 4 * heads, 1, generator=g))
    x[3, :, :16] = 0.0
    x[4, :, 0] = torch.inf
    x[5, :, 1] = -torch.inf
    x[6, :, 2] = torch.nan
    x[7] = torch.nan
    x[8] *= 1e-30
    x[9] = 60000.0
    x[10, :, :16] = torch.tensor([6.0, 0.25, -0.25, 0.75, -0.75, 1.25, 1.75, 2.5, -2.5, 3.5, 5.0, -5.0, 1e-3, -1e-3, 4.5, 2.25])
    x = x.to(dtype)
    k, v = (x[:, heads:2 * heads], x[:, 3 * heads:]) if packed else (x[:, :heads].contiguous(), x[:, heads:2 * heads].contiguous())
    slots = torch.randperm(pages * PAGE, generator=g)[:T].to(torch.int32)
    slots[20] = -1
    shapes = {"k_cache": dim // 2, "v_cache": dim // 2, "k_scales": dim // 16, "v_scales": dim // 16}
    pool = {n: torch.full((pages, PAGE, heads, w), 0xAB, dtype=torch.uint8, device="cuda") for n, w in shapes.items()}
    xd = x.cuda()
    kd, vd = ((xd[:, heads:2 * heads], xd[:, 3 * heads:]) if packed
              else (xd[:, :heads].contiguous(), xd[:, heads:2 * heads].contiguous()))
    held = [torch.empty(T, heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    batch.append(kd, vd, *pool.values(), slots.cuda(), k_held=held[0], v_held=held[1])
    for rows, cn, sn, h in ((k, "k_cache", "k_scales", held[0]), (v, "v_cache", "v_scales", held[1])):
        codes, scales = nvfp4.quantize_rows(without_nan(rows.float().numpy()))
        want_c, want_s = (np.full(tuple(pool[n].shape), 0xAB, np.uint8).reshape(pages * PAGE, heads, -1) for n in (cn, sn))
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                want_c[s], want_s[s] = codes[i], scales[i]
        assert np.array_equal(pool[cn].cpu().numpy().reshape(want_c.shape), want_c)
        assert np.array_equal(pool[sn].cpu().numpy().reshape(want_s.shape), want_s)
        values = obatch.dequant(torch.from_numpy(codes), torch.from_numpy(scales))
        assert torch.equal(h.double().cpu(), values)  # exact in the input's type, the unstored row too


def test_append_matches_the_single_sequence_writer():
    T, P = 300, 4
    k = torch.randn(T, 4, 256, device="cuda").half()
    v = torch.randn(T, 4, 256, device="cuda").half()
    v[5, 0, 3], v[5, 1, 2], v[5, 2, 7], v[6, 0, :40] = torch.nan, torch.inf, -torch.inf, torch.nan
    table = i32([[2, 0, 3]])
    one = [torch.zeros(P, PAGE, 4, w, dtype=torch.uint8, device="cuda") for w in (128, 128, 16, 16)]
    many = [t.clone() for t in one]
    ops.nvfp4_append(k, v, *one, table, i32([100]))
    pos = torch.arange(100, 100 + T, device="cuda")
    slots = (table[0, pos // PAGE] * PAGE + pos % PAGE).to(torch.int32)
    batch.append(k, v, *many, slots)
    assert all(torch.equal(a, b) for a, b in zip(one, many))


def test_append_slot_outside_the_pool():
    pool = [torch.zeros(2, PAGE, 1, w, dtype=torch.uint8, device="cuda") for w in (32, 32, 4, 4)]
    k = torch.ones(3, 1, 64, device="cuda").half()
    batch.append(k, k, *pool, i32([0, 2 * PAGE, 0x7fffffff]))
    assert _lib.device_error(clear=True) == 4
    assert int((pool[0] != 0).sum()) == 32


# ------------------------------------------------------------------- attend
def make_pool(pages, heads, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = [torch.randint(0, 256, (pages, PAGE, heads, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
             for _ in range(2)]
    scales = [(0.1 + torch.rand(pages, PAGE, heads, dim // 16, generator=g, device="cuda")).to(torch.float8_e4m3fn)
              for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def make_tables(kv_lens, width, pages, seed):
    ids = np.random.default_rng(seed).permutation(pages)
    table, at = np.full((len(kv_lens), width), -1), 0
    for b, kv in enumerate(kv_lens):
        n = -(-max(kv, 0) // PAGE)
        table[b, :n] = ids[at:at + n]
        at += n
    return i32(table)


def check(out, ref, mag, dtype):
    """P is rounded to FP16 once (2^-11 of each weight), scores and sums are FP32
    (well below 3e-5 of a weight), and the output is rounded to its type."""
    eps = 2.0 ** -10 if dtype == torch.float16 else 2.0 ** -7
    ulp = torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=2.0 ** -14)))) * eps
    tol = (2.0 ** -11 + 3e-5) * mag + ulp + 1e-7
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert bool((err <= tol).all()), float((err / tol).max())


def run_attend(rows, kv_lens, heads, kv_heads, dim, dtype, seed=0, spare=0, gap=0, table=None, pool=None, q_scale=1.0):
    width = max(1, max(-(-max(kv, 0) // PAGE) for kv in kv_lens))
    pages = sum(-(-max(kv, 0) // PAGE) for kv in kv_lens) + 2
    pool = pool or make_pool(pages, kv_heads, dim, seed)
    table = make_tables(kv_lens, width, pages, seed) if table is None else table
    cu = np.concatenate([[0], np.cumsum(rows)])
    T = int(cu[-1]) + spare
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (torch.randn(T, heads + gap, dim, generator=g, device="cuda") * q_scale).to(dtype)[:, :heads]
    out = torch.full((T, heads + gap, dim), 7.0, dtype=dtype, device="cuda")[:, :heads]
    ws = batch.attend_workspace("cuda", dim)
    args = (q, *pool, table, i32(cu), i32(kv_lens))
    want, mag = obatch.attend(*args, out, dim ** -0.5)
    batch.attend(*args, out, ws, max_rows=max(max(rows), 1))
    check(out, want, mag, dtype)
    again = out.clone()
    batch.attend(*args, out, ws, max_rows=max(max(rows), 1) + 3)
    assert torch.equal(out, again)  # no result depends on timing
    return args, out, ws


LENGTHS = [1, 2, 15, 31, 33, 64, 127, 128, 129, 255, 256, 257, 600, 1025]


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (8, 8, 64), (14, 2, 64), (7, 1, 128), (16, 1, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_decode(heads, kv_heads, dim, dtype):
    run_attend([1] * len(LENGTHS), LENGTHS, heads, kv_heads, dim, dtype, seed=dim)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (8, 8, 64), (14, 2, 64), (16, 1, 256), (64, 1, 64)])
@pytest.mark.parametrize("n", [2, 7, 8, 9, 30])
def test_attend_windows(heads, kv_heads, dim, n):
    kv = [k for k in LENGTHS if k >= n]
    run_attend([n] * len(kv), kv, heads, kv_heads, dim, torch.bfloat16, seed=n)


@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 1, 256), (24, 2, 128), (32, 2, 64), (51, 3, 64)])
def test_attend_wide_groups(heads, kv_heads, dim):
    """9 to 17 heads a KV head: decode rows beside windows and requests without tokens."""
    run_attend([1, 1, 0, 2, 1, 5, 1, 1], [700, 1, 9, 300, 0, 513, 256, 2049], heads, kv_heads, dim, torch.float16,
               seed=heads, gap=kv_heads)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (14, 2, 64)])
def test_attend_mixed_step(heads, kv_heads, dim):
    """Decode rows, windows, prompt chunks, whole prompts and idle requests in one
    call; rows past the step's end and a strided q and out."""
    run_attend([1, 0, 7, 200, 300, 0, 1, 129, 2], [5, 40, 300, 1000, 300, 0, 2000, 130, 257], heads, kv_heads, dim,
               torch.float16, spare=5, gap=kv_heads)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128)])
def test_attend_rows_that_see_nothing(heads, kv_heads, dim):
    """More rows than tokens (the first rows see none) and a request without
    tokens: those rows are 0."""
    _, out, _ = run_attend([1, 9, 1, 40, 3], [0, 4, 3, 17, 1], heads, kv_heads, dim, torch.float16)
    assert int(out[0].count_nonzero()) == 0 and int(out[1:6].count_nonzero()) == 0
    assert int(out[11:34].count_nonzero()) == 0 and int(out[51:53].count_nonzero()) == 0


@pytest.mark.parametrize("rows,kv", [([1], [30000]), ([7], [30000]), ([1] * 700, [90] * 700), ([5] * 90, [300] * 90),
                                     ([1, 1, 1], [40000, 1, 513])])
def test_attend_work_split(rows, kv):
    """One long request over all CTAs; many short items a CTA."""
    run_attend(rows, kv, 24, 4, 256, torch.float16)


def test_attend_large_scores():
    """Scores of hundreds: the reference maximum moves often."""
    run_attend([1, 7, 40], [3000, 2000, 1000], 24, 4, 256, torch.float16, q_scale=60.0)


@pytest.mark.parametrize("rows", [[1, 1], [9, 9]])
def test_attend_page_order_and_stale_bytes(rows):
    """Another physical order of the same pages gives the same bits, and what
    lies in the pool past a request's end (NaN scales too) does not matter."""
    kv, dim = [700, 300], 256
    pool = make_pool(8, 4, dim, 3)
    ids = np.arange(5)
    table = np.full((2, 3), -1)
    table[0], table[1, :2] = ids[:3], ids[3:5]
    args, out, ws = run_attend(rows, kv, 24, 4, dim, torch.float16, pool=pool, table=i32(table))
    order = torch.tensor([6, 2, 7, 0, 5])
    other = [t.clone() for t in pool]
    for t, u in zip(pool, other):
        u.view(torch.uint8).fill_(0x7F)  # NaN as a scale
        u[order] = t[:5]
    moved = np.full((2, 3), -1)
    moved[0], moved[1, :2] = order[:3], order[3:5]
    for t in other:
        flat = t.view(torch.uint8)
        flat[order[2], 700 - 512:] = 0x7F
        flat[order[4], 300 - 256:] = 0x7F
    out2 = torch.empty_like(out)
    batch.attend(args[0], *other, i32(moved), args[6], args[7], out2, ws, max_rows=max(rows))
    assert torch.equal(out, out2)


@pytest.mark.parametrize("rows", [[1, 1, 1], [10, 10, 10]])
def test_attend_bad_pages_and_ranges(rows):
    """Table entries outside the pool count as absent tokens; lengths beyond the
    table are cut; both set their bits and nothing else happens."""
    kv = [600, 600, 600]
    pool = make_pool(9, 4, 256, 5)
    table = i32([[0, -1, 2], [3, 4, 999], [-5, 9, 77]])
    run_attend(rows, kv, 24, 4, 256, torch.float16, pool=pool, table=table)
    assert _lib.device_error(clear=True) == 2
    q = torch.randn(2, 24, 256, device="cuda").half()
    out = torch.full_like(q, 7.0)
    ws = batch.attend_workspace("cuda", 256)
    good = i32([[0, 1], [2, 3]])
    batch.attend(q, *pool, good, i32([0, 1, 2]), i32([512, 5000]), out, ws, max_rows=1)
    assert _lib.device_error(clear=True) == 1
    want = torch.empty_like(out)
    batch.attend(q, *pool, good, i32([0, 1, 2]), i32([512, 512]), want, ws, max_rows=1)
    assert torch.equal(out, want)
    out.fill_(7.0)
    batch.attend(q, *pool, good, i32([0, 1, 9]), i32([512, 512]), out, ws, max_rows=8)  # rows that do not exist
    assert _lib.device_error(clear=True) == 1
    # (without request 1 the work is split elsewhere: the last bit may differ)
    assert float((out[0].float() - want[0].float()).abs().max()) <= 2.0 ** -10 * float(want[0].float().abs().max())
    assert bool((out[1] == 7.0).all())


def test_attend_offsets_past_32_bits():
    """A pool of more than 4 GB of codes a tensor; the pages used lie at its end."""
    pages = 34000  # x 128 KB
    shapes = ((128, torch.uint8), (128, torch.uint8), (16, torch.uint8), (16, torch.uint8))
    big = [torch.zeros(pages, PAGE, 4, w, dtype=d, device="cuda") for w, d in shapes]
    small = make_pool(6, 4, 256, 9)
    at = torch.tensor([33999, 33990, 20000, 33000, 32768, 16384])
    for b, s in zip(big, small):
        b[at] = s.view(torch.uint8)
    for rows in ([1, 1], [8, 8]):
        args, out, ws = run_attend(rows, [700, 500], 24, 4, 256, torch.float16, pool=small,
                                   table=i32([[0, 1, 2], [3, 4, -1]]))
        out2 = torch.empty_like(out)
        batch.attend(args[0], *big, i32([[33999, 33990, 20000], [33000, 32768, -1]]), args[6], args[7], out2, ws,
                     max_rows=max(rows))
        assert torch.equal(out, out2)
    k = torch.randn(2, 4, 256, device="cuda").half()
    batch.append(k, k, *big, i32([33998 * PAGE + 255, 16385 * PAGE]))
    want, _ = nvfp4.quantize_rows(k.float().cpu().numpy())
    assert np.array_equal(big[0][33998, 255].cpu().numpy(), want[0])
    assert np.array_equal(big[1][16385, 0].cpu().numpy(), want[1])


def test_attend_matches_the_single_sequence_kernels():
    pool = make_pool(20, 4, 256, 11)
    table = i32([list(range(18))])
    for n, pre in ((1, 4000), (7, 4000), (40, 2000)):
        q = torch.randn(n, 24, 256, device="cuda").half()
        out, one = torch.empty_like(q), torch.empty_like(q)
        batch.attend(q, *pool, table, i32([0, n]), i32([pre + n]), out, batch.attend_workspace("cuda", 256), max_rows=n)
        if n > 8:
            ops.nvfp4_prefill(q, *pool, table, i32([pre]), one)
        else:
            po, pml = ops.split_workspace("cuda", n, 16)
            ops.attn_split(q, pool[0], pool[1], table, i32([pre]), po, pml, pool[2], pool[3], 16)
            ops.attn_combine(po, pml, one, 16)
        scale = float(one.abs().max())
        assert float((out.float() - one.float()).abs().max()) <= 2.0 ** -10 * 2 * scale  # two roundings of P


def test_step_in_a_graph_and_on_a_stream():
    """tables + append + attend captured once; lengths change between replays; all
    of it on a stream of its own."""
    R, W, rows, dim = 3, 4, 16, 128
    state = {"lengths": i32([0, 0, 0]), "new": i32([1, 1, 1]), "held": i32([0, 0, 0]),
             "ring": i32(list(range(12))), "ring_state": i32([0, 12]), "table": i32(np.full((R, W), -1)),
             "cu": i32([0] * 4), "kv": i32([0] * 3), "held_out": i32([0] * 3), "ring_out": i32([0, 0])}
    maps = [i32([0] * rows) for _ in range(3)]
    pool = [torch.zeros(12, PAGE, 2, w, dtype=torch.uint8, device="cuda") for w in (64, 64, 8, 8)]
    q = torch.zeros(rows, 6, dim, device="cuda").half()
    k, v = (torch.zeros(rows, 2, dim, device="cuda").half() for _ in range(2))
    out, ws = torch.zeros_like(q), batch.attend_workspace("cuda", dim)

    def step():
        batch.build_tables(state["lengths"], state["new"], state["held"], state["ring"], state["ring_state"],
                           state["table"], state["cu"], state["kv"], state["held_out"], state["ring_out"], *maps)
        batch.append(k, v, *pool, maps[0])
        batch.attend(q, *pool, state["table"], state["cu"], state["kv"], out, ws, max_rows=8)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for t in (state["held"], state["lengths"]):
            t.zero_()
        g = torch.Generator(device="cuda").manual_seed(0)
        for new in ([5, 1, 0], [1, 7, 3], [1, 8, 1], [2, 0, 7]):
            n = sum(new)
            state["new"].copy_(i32(new))
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            graph.replay()
            want, mag = obatch.attend(q, *pool, state["table"], state["cu"], state["kv"], out, dim ** -0.5)
            check(out[:n], want[:n], mag[:n], torch.float16)
            state["held"].copy_(state["held_out"])
            state["ring_state"].copy_(state["ring_out"])
            state["lengths"].copy_(state["kv"])
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert state["lengths"].tolist() == [9, 16, 11]


def test_example_serves_requests():
    """examples/batched_verify.py: pages are neither lost nor held twice, requests
    end, drafts are accepted."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "batched_verify.py"
    spec = importlib.util.spec_from_file_location("batched_verify", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.serve(requests=6, steps=25, seed=1, say=lambda *_: None)
    assert got["free"] + got["held"] == got["pages"]
    assert got["lengths"] == got["done"] and got["finished"] > 0 and 0 < got["accepted"] <= got["drafted"]


@pytest.mark.parametrize("rows,kv", [([1, 1], [700, 40]), ([1], [30000]), ([9, 9], [700, 300]), ([7], [30000])])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attend_nan_query(rows, kv, value):
    """A query element that is not finite makes its row and head NaN and nothing
    else, whether one CTA has the item (the short ones) or many share it."""
    args, out, ws = run_attend(rows, kv, 24, 4, 256, torch.float16)
    want, mag = obatch.attend(*args, out, 256 ** -0.5)
    q = args[0].clone()
    q[-1, 5, 100] = value
    got = torch.empty_like(out)
    batch.attend(q, *args[1:], got, ws, max_rows=max(rows))
    assert bool(got[-1, 5].isnan().all())
    got[-1, 5] = out[-1, 5]
    check(got, want, mag, torch.float16)


def test_step_without_rows():
    """Every request is idle or ends: pages go back, no row is attended, written
    or scored."""
    from qwarz_b200 import scoring

    pool = make_pool(6, 4, 256, 0)
    before = [t.clone() for t in pool]
    ring, table = i32([5, -1, -1, -1, -1, -1]), i32([[0, 1], [2, -1], [3, 4]])
    cu, kv, held_out, ring_out, maps = i32([-7] * 4), i32([-7] * 3), i32([-7] * 3), i32([-7] * 2), [i32([]) for _ in range(3)]
    batch.build_tables(i32([300, 20, 500]), i32([-1, 0, -1]), i32([2, 1, 2]), ring, i32([0, 1]), table, cu, kv, held_out,
                       ring_out, *maps)
    rows = torch.empty(0, 32, 256, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(0, 24, 256, dtype=torch.bfloat16, device="cuda")
    batch.append(rows[:, 24:28], rows[:, 28:], *pool, maps[0])
    batch.attend(rows[:, :24], *pool, table, cu, kv, out, batch.attend_workspace("cuda", 256), max_rows=1)
    scoring.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"),
                           torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), torch.empty(0, 2, device="cuda"),
                           torch.empty(0, 2, dtype=torch.int32, device="cuda"), scoring.workspace("cuda", 0, 100, 2))
    assert ring.tolist() == [5, 0, 1, 3, 4, -1] and ring_out.tolist() == [0, 5] and cu.tolist() == [0] * 4
    assert kv.tolist() == [0, 20, 0] and held_out.tolist() == [0, 1, 0]
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, before))


def test_example_serves_one_request():
    """A server of one slot has steps without rows, when its request ends."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "batched_verify.py"
    spec = importlib.util.spec_from_file_location("batched_verify", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.serve(requests=1, steps=8, seed=13, say=lambda *_: None)
    assert got["free"] + got["held"] == got["pages"] and got["finished"] > 0 and got["lengths"] == got["done"]


def test_one_row_of_any_stride():
    """One row whose view has a stride that rows could not have."""
    def view(x):
        return torch.empty(2 * 1001 * x.shape[1], dtype=x.dtype, device="cuda").as_strided(
            x.shape, (1001, x.shape[2], 1)).copy_(x)

    pool = make_pool(2, 2, 64, 8)
    ws, table, cu, kv = batch.attend_workspace("cuda", 64), i32([[1, 0]]), i32([0, 1]), i32([300])
    q = torch.randn(1, 6, 64, device="cuda").half()
    want, out = torch.empty_like(q), view(torch.zeros_like(q))
    batch.attend(q, *pool, table, cu, kv, want, ws, max_rows=1)
    batch.attend(view(q), *pool, table, cu, kv, out, ws, max_rows=1)
    assert torch.equal(out, want)
    k = torch.randn(1, 2, 64, device="cuda").half()
    other = [t.clone() for t in pool]
    batch.append(k, k, *pool, i32([7]))
    batch.append(view(k), view(k), *other, i32([7]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, other))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (64, 8, 64)])
@pytest.mark.parametrize("rows,kv", [([7], [30001]), ([12, 7, 3, 40], [9000, 20001, 3000, 12345])])
def test_attend_long_windows_below_dim_256(heads, kv_heads, dim, rows, kv):
    """A dozen tiles and more a CTA: every buffer, barrier and parity of the
    many-row kernel's two-buffer form comes round several times, with changes of
    item between."""
    run_attend(rows, kv, heads, kv_heads, dim, torch.float16, seed=dim)
