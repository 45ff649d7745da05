"""The operators for requests that share prefixes (qwarz_b200.batch: share_prefixes,
append_rotated, attend_shared) against plain 64-bit forms (oracle/batch.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import batch as obatch
from qwarz_b200 import _lib, batch
from tests.test_gpu_batch import check, i32, make_pool, make_tables

pytestmark = pytest.mark.gpu
PAGE = 256


@pytest.fixture(autouse=True)
def clean_errors(cuda):
    _lib.device_error(clear=True)
    yield
    assert _lib.device_error(clear=True) == 0  # a test that expects a bit clears it itself


# -------------------------------------------------------------------- share
def run_share(prefix_of, kv_lens, cu_rows, extra=0, bad=False, in_place=False, requests=None):
    R = len(kv_lens)
    T = max(0, max(cu_rows)) + extra if requests is None else len(requests)
    if requests is None:
        requests = np.repeat(np.arange(R), np.diff(cu_rows)).tolist() + [-1] * extra
    positions = np.random.default_rng(T).integers(0, 9000, T).tolist()
    want, why = obatch.share_prefixes(prefix_of, kv_lens, cu_rows, positions, requests)
    assert why == bad
    plan = torch.full((3 * R + 1 + T + 3,), -7, dtype=torch.int32, device="cuda")
    pos = i32(positions)
    out = pos if in_place else torch.full_like(pos, -7)
    batch.share_prefixes(i32(prefix_of), i32(kv_lens), i32(cu_rows), pos, i32(requests), plan, out)
    got = [x.tolist() for x in plan.split([R + 1, R, R, T, 3])]
    assert got[4] == [-7] * 3
    for name, a, b in zip(("cu_shared", "reads", "alone", "shared_rows"), got, want):
        assert a == b, name
    assert out.tolist() == want[4]
    return plan


@pytest.mark.parametrize("prefix_of,new,extra", [
    ([-1], [1], 0), ([-1, 0], [0, 1], 0), ([-1, 0], [0, 0], 3), ([1, -1, 1], [2, 0, 3], 1),
    ([3, -1, 3, -1, 1, 1, -1, 3], [1, 0, 7, 2, 0, 4, 1, 300], 5),   # a prefix that has rows itself, an idle reader
    ([2, 2, -1], [0, 5, 0], 0),                                     # alone beside an idle one
])
@pytest.mark.parametrize("in_place", [False, True])
def test_share_small(prefix_of, new, extra, in_place):
    run_share(prefix_of, [100 * i for i in range(len(new))], np.cumsum([0] + new).tolist(), extra, in_place=in_place)


@pytest.mark.parametrize("R", [1, 31, 33, 1025, 3000])
def test_share_many(R):
    g = np.random.default_rng(R)
    prefix = g.integers(-1, R, R)
    prefix[g.random(R) < 0.5] = -1
    prefix = np.where((prefix >= 0) & (prefix[prefix] < 0) & (prefix != np.arange(R)), prefix, -1)
    prefix = np.where((prefix >= 0) & (prefix[prefix] >= 0), -1, prefix)
    new = g.choice([0, 1, 1, 7, 40], R)
    run_share(prefix.tolist(), g.integers(0, 5000, R).tolist(), np.cumsum([0] + new.tolist()).tolist(), 2)


def test_share_most_requests():
    """2^14 requests behind three prefixes, the most a call takes."""
    R = 1 << 14
    g = np.random.default_rng(0)
    prefix = g.integers(0, 3, R)
    prefix[:3] = -1
    new = g.choice([0, 1, 2], R)
    new[:3] = 0
    cu = np.cumsum(np.concatenate([[0], new]))
    T = int(cu[-1])
    req = np.repeat(np.arange(R), new)
    plan = batch.prefix_plan("cuda", R, T)
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    batch.share_prefixes(i32(prefix), i32(np.arange(R)), i32(cu), pos, i32(req), plan, pos)
    rows = plan[3 * R + 1:].cpu().numpy()
    assert (rows == np.argsort(prefix[req], kind="stable")).all()
    assert (pos.cpu().numpy() == prefix[req]).all()
    assert plan[:4].tolist() == np.cumsum([0] + [int((prefix[req] == i).sum()) for i in range(3)]).tolist()


@pytest.mark.parametrize("prefix_of", [[5, -1], [1, 0], [0, -1], [-1, 0, 1]])
def test_share_prefixes_that_cannot_be(prefix_of):
    """One that does not exist, one that reads back, oneself, a prefix of a prefix."""
    n = len(prefix_of)
    run_share(prefix_of, [9] * n, list(range(n + 1)), bad=True)
    assert _lib.device_error(clear=True) == 1


@pytest.mark.parametrize("cu_rows", [[0, 4, 2, 6], [-3, 2, 3, 6], [0, 2, 4, 900], [0, 6, 0, 6]])
def test_share_row_ranges_that_cannot_be(cu_rows):
    """Nothing is written outside the plan; the other requests' rows are listed."""
    R, T = 3, 6
    plan = torch.full((3 * R + 1 + T + 8,), -7, dtype=torch.int32, device="cuda")
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    batch.share_prefixes(i32([2, 2, -1]), i32([1, 1, 50]), i32(cu_rows), pos, i32([0, 0, 1, 1, 7, -4]), plan, pos)
    assert _lib.device_error(clear=True) == 1
    assert plan[-8:].tolist() == [-7] * 8
    fits = [list(range(lo, hi)) if 0 <= lo <= hi <= T else [] for lo, hi in zip(cu_rows, cu_rows[1:])][:2]
    assert plan[3 * R + 1:-8].tolist()[:len(fits[0]) + len(fits[1])] == fits[0] + fits[1]
    assert pos.tolist() == [50, 50, 50, 50, 0, 0]


# ------------------------------------------------------------------- rotate
def make_rows(T, heads, kv_heads, dim, dtype, seed):
    """q, k, v as parts of packed rows (with a few columns more)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, heads + 2 * kv_heads + 1, dim, generator=g, device="cuda")
    x[:, heads:heads + kv_heads] *= torch.exp(torch.randn(kv_heads, dim, generator=g, device="cuda"))
    x = x.to(dtype)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:heads + 2 * kv_heads], x


def make_slots(T, pages, seed):
    return i32(np.random.default_rng(seed).permutation(pages * PAGE)[:T])


def freqs_of(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


def weight_of(dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.exp(0.3 * torch.randn(dim, generator=g, device="cuda"))


def close(got, y, mag, dtype):
    """y in 32 bits: products, sum, cosine, sine (5 roundings of 2^-24 of |a| + |b|),
    and with a norm the sum of squares (13 additions on a path, half their effect), the
    root and two products (13 more); then one rounding to the type, which is off by
    half a step (2^-25 at least in FP16's subnormals)."""
    off = mag * 18 * 2.0 ** -24
    tol = off + (y.abs() + off) * (torch.finfo(dtype).eps / 2) + 2.0 ** -25
    assert bool(((got.double() - y).abs() <= tol).all()), float(((got.double() - y).abs() / tol).max())


@pytest.mark.parametrize("T", [1, 3, 300])
@pytest.mark.parametrize("heads,kv_heads,dim,freqs", [(24, 4, 256, 32), (24, 4, 256, 128), (32, 8, 128, 64), (16, 2, 128, 24),
                                                      (14, 2, 64, 8), (5, 5, 64, 32), (3, 1, 64, 16), (7, 1, 128, 0)])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("norm,dtype", [(False, torch.float16), (True, torch.bfloat16), (True, torch.float16)])
def test_rotated(T, heads, kv_heads, dim, freqs, neighbours, norm, dtype):
    q, k, v, _ = make_rows(T, heads, kv_heads, dim, dtype, seed=T + dim)
    P = T // PAGE + 2
    slots = make_slots(T, P, T)
    slots[T // 2] = -1 if T > 1 else slots[0]
    positions = i32(np.random.default_rng(T).integers(0, 1 << 22, T))
    inv = freqs_of(freqs)
    qw, kw = (weight_of(dim, 1), weight_of(dim, 2)) if norm else (None, None)
    widths = (dim // 2, dim // 2, dim // 16, dim // 16)
    pool = [torch.full((P, PAGE, kv_heads, w), 0xA5, dtype=torch.uint8, device="cuda") for w in widths]
    held = [torch.empty(T, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    q_out = torch.full((T, heads + 2, dim), 7.0, dtype=dtype, device="cuda")
    batch.append_rotated(q, k, v, q_out[:, 1:-1], *pool, slots, positions, inv, neighbours, qw, kw, 1e-5, *held)
    y, mag = obatch.rotate(q, positions, inv, neighbours, qw, 1e-5)
    close(q_out[:, 1:-1], y, mag, dtype)
    assert bool((q_out[:, 0] == 7).all()) and bool((q_out[:, -1] == 7).all())
    y, _ = obatch.rotate(k, positions, inv, neighbours, kw, 1e-5)
    for rows, c, s, h in ((y, pool[0], pool[2], held[0]), (v.double(), pool[1], pool[3], held[1])):
        codes, scales = obatch.quantise(rows)
        assert torch.equal(h.double(), obatch.dequant(codes, scales))
        want_c, want_s = torch.full_like(c, 0xA5), torch.full_like(s, 0xA5)
        some = slots >= 0
        want_c.flatten(0, 1)[slots[some].long()] = codes[some]
        want_s.flatten(0, 1)[slots[some].long()] = scales[some]
        assert torch.equal(c, want_c) and torch.equal(s, want_s)


@pytest.mark.parametrize("heads,kv_heads,dim,freqs", [(24, 4, 256, 32), (32, 8, 128, 64), (14, 2, 64, 8), (40, 3, 128, 24)])
@pytest.mark.parametrize("norm,dtype,neighbours", [(True, torch.bfloat16, False), (False, torch.float16, True)])
def test_rotated_long_steps(heads, kv_heads, dim, freqs, norm, dtype, neighbours):
    """More rows than are taken one by one (1,101 = 275 x 4 + 1)."""
    test_rotated(1101, heads, kv_heads, dim, freqs, neighbours, norm, dtype)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (14, 2, 64)])
def test_rotated_rows_do_not_depend_on_the_step(heads, kv_heads, dim):
    """The first rows of a step of 1,400 have the bytes that they have in steps of 725, 700 and 1."""
    T, P = 1400, 6
    q, k, v, _ = make_rows(T, heads, kv_heads, dim, torch.bfloat16, 9)
    slots, positions, inv, w = make_slots(T, P, 9), i32(np.arange(T) * 37), freqs_of(dim // 8), weight_of(dim, 3)
    got = []
    for n in (T, 725, 700, 1):
        pool = [torch.zeros(P * PAGE, kv_heads, x, dtype=torch.uint8, device="cuda").view(P, PAGE, kv_heads, x)
                for x in (dim // 2, dim // 2, dim // 16, dim // 16)]
        out = torch.empty(n, heads, dim, dtype=torch.bfloat16, device="cuda")
        batch.append_rotated(q[:n], k[:n], v[:n], out, *pool, slots[:n], positions[:n], inv, False, w, w)
        got.append([out] + [x.flatten(0, 1)[slots[:n].long()] for x in pool])
    for other in got[1:]:
        assert all(torch.equal(a[:len(b)], b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotated_in_place(neighbours):
    """q rotated in the packed rows it lies in; K and V beside it stay as they were."""
    T = 290
    q, k, v, x = make_rows(T, 24, 4, 256, torch.bfloat16, 5)
    before = x.clone()
    pool = [[torch.zeros(3, PAGE, 4, w, dtype=torch.uint8, device="cuda") for w in (128, 128, 16, 16)] for _ in range(2)]
    slots, positions, inv = make_slots(T, 3, 1), i32(np.arange(T) + 7), freqs_of(32)
    out = torch.empty(T, 24, 256, dtype=torch.bfloat16, device="cuda")
    batch.append_rotated(q, k, v, out, *pool[0], slots, positions, inv, neighbours)
    assert torch.equal(x, before)
    batch.append_rotated(q, k, v, q, *pool[1], slots, positions, inv, neighbours)
    assert torch.equal(q, out) and torch.equal(x[:, 24:], before[:, 24:])
    assert all(torch.equal(a, b) for a, b in zip(*pool))


def test_rotated_without_rotation_is_append():
    """No frequencies, or position 0: the bytes of `append`, for NaN and infinite rows too."""
    T = 40
    q, k, v, _ = make_rows(T, 8, 4, 128, torch.float16, 6)
    k[3, 1, 5], k[4, 0, 64], v[5, 2, 7], k[6] = torch.nan, torch.inf, -torch.inf, 0.0
    slots = make_slots(T, 1, 2)
    pool = [[torch.zeros(1, PAGE, 4, w, dtype=torch.uint8, device="cuda") for w in (64, 64, 8, 8)] for _ in range(2)]
    batch.append(k, v, *pool[0], slots)
    out = torch.empty_like(q.contiguous())
    batch.append_rotated(q, k, v, out, *pool[1], slots, i32([1000] * T), freqs_of(0))
    assert torch.equal(out, q) and all(torch.equal(a, b) for a, b in zip(*pool))
    for t in pool[1]:
        t.zero_()
    finite = torch.ones(T, dtype=torch.bool, device="cuda")
    finite[3:5] = False  # 0 x NaN and 0 x infinity reach the other dim of a pair
    batch.append_rotated(q, k, v, out, *pool[1], slots, i32([0] * T), freqs_of(64))
    assert torch.equal(out, q)
    at = slots[finite].long()
    assert all(torch.equal(a.flatten(0, 1)[at], b.flatten(0, 1)[at]) for a, b in zip(*pool))


def test_rotated_far_positions():
    """Angles of positions up to 2^30 - 1 keep their digits."""
    positions = [0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 30 - 1, 777777777]
    T = len(positions)
    q, k, v, _ = make_rows(T, 6, 1, 256, torch.float16, 7)
    pool = [torch.zeros(1, PAGE, 1, w, dtype=torch.uint8, device="cuda") for w in (128, 128, 16, 16)]
    out, held = torch.empty(T, 6, 256, dtype=torch.float16, device="cuda"), torch.empty(T, 1, 256, dtype=torch.float16,
                                                                                       device="cuda")
    inv = freqs_of(128)
    batch.append_rotated(q, k, v, out, *pool, make_slots(T, 1, 3), i32(positions), inv, k_held=held)
    y, mag = obatch.rotate(q, i32(positions), inv, False)
    close(out, y, mag, torch.float16)
    y, _ = obatch.rotate(k, i32(positions), inv, False)
    assert torch.equal(held.double(), obatch.dequant(*obatch.quantise(y)))


@pytest.mark.parametrize("norm,eps", [(True, 0.0), (True, 1e-6), (False, 1e-6)])
def test_rotated_smallest_and_largest_k(norm, eps):
    """K rows whose squares 32 bits do not hold, and rows of zeros."""
    T = 8
    q, k, v, _ = make_rows(T, 4, 2, 128, torch.bfloat16, 8)
    k.mul_(torch.tensor([1.0, 2.0 ** -90, 2.0 ** -60, 2.0 ** -20, 2.0 ** 30, 2.0 ** 63, 2.0 ** 80, 2.0 ** -126],
                        device="cuda").bfloat16()[:, None, None])
    pool = [torch.zeros(1, PAGE, 2, w, dtype=torch.uint8, device="cuda") for w in (64, 64, 8, 8)]
    held = torch.empty(T, 2, 128, dtype=torch.bfloat16, device="cuda")
    kw, positions, inv = weight_of(128, 3) if norm else None, i32(range(5, 5 + T)), freqs_of(32)
    batch.append_rotated(q, k, v, torch.empty_like(q.contiguous()), *pool, make_slots(T, 1, 4), positions, inv,
                         k_weight=kw, eps=eps, k_held=held)
    y, _ = obatch.rotate(k, positions, inv, False, kw, eps)
    assert torch.equal(held.double(), obatch.dequant(*obatch.quantise(y)))
    k.zero_()
    batch.append_rotated(q, k, v, torch.empty_like(q.contiguous()), *pool, make_slots(T, 1, 4), positions, inv,
                         k_weight=kw, eps=1e-6, k_held=held)
    assert int(held.count_nonzero()) == 0


def test_rotated_slot_outside_the_pool():
    x = torch.ones(3, 1, 64, device="cuda").half()
    pool = [torch.zeros(2, PAGE, 1, w, dtype=torch.uint8, device="cuda") for w in (32, 32, 4, 4)]
    batch.append_rotated(x, x.clone(), x.clone(), torch.empty_like(x), *pool, i32([0, 2 * PAGE, 0x7fffffff]), i32([0, 0, 0]),
                         freqs_of(8))
    assert _lib.device_error(clear=True) == 4
    assert int((pool[0] != 0).sum()) == 32


# ------------------------------------------------------------------- attend
def make_plan(prefix_of, kv_lens, cu, T):
    R = len(kv_lens)
    plan = batch.prefix_plan("cuda", R, T)
    req = np.repeat(np.arange(R), np.diff(cu)).tolist()
    req = i32(req + [-1] * (T - len(req)))
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    batch.share_prefixes(i32(prefix_of), i32(kv_lens), i32(cu), pos, req, plan, pos)
    return plan


def run_shared(prefix_of, rows, kv_lens, heads, kv_heads, dim, dtype, seed=0, spare=0, gap=0, table=None, pool=None,
               q_scale=1.0):
    width = max(1, max(-(-max(kv, 0) // PAGE) for kv in kv_lens))
    pages = sum(-(-max(kv, 0) // PAGE) for kv in kv_lens) + 2
    pool = pool or make_pool(pages, kv_heads, dim, seed)
    table = make_tables(kv_lens, width, pages, seed) if table is None else table
    cu = np.concatenate([[0], np.cumsum(rows)])
    T = int(cu[-1]) + spare
    plan = make_plan(prefix_of, kv_lens, cu, T)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (torch.randn(T, heads + gap, dim, generator=g, device="cuda") * q_scale).to(dtype)[:, :heads]
    out = torch.full((T, heads + gap, dim), 7.0, dtype=dtype, device="cuda")[:, :heads]
    ws = batch.shared_workspace("cuda", dim, T, heads)
    ws.fill_(0xFF)  # nothing of the workspace is read before it is written
    head = (q, *pool, table, i32(cu), i32(kv_lens))
    want, mag = obatch.attend_shared(*head, prefix_of, out, dim ** -0.5)
    batch.attend_shared(*head, plan, out, ws, max_rows=max(max(rows), 1))
    check(out, want, mag, dtype)
    again = out.clone()
    batch.attend_shared(*head, plan, out, ws, max_rows=max(max(rows), 1) + 3)
    assert torch.equal(out, again)  # no result depends on timing
    return head, plan, out, ws


LAYOUTS = [(24, 4, 256), (32, 8, 128), (8, 8, 64), (14, 2, 64), (7, 1, 128), (16, 1, 256), (40, 1, 64)]
# prefixes of 0 to 1025 tokens (requests 0 to 9), read by one request, by several, by none
PREFIXES = [0, 1, 127, 128, 129, 255, 256, 257, 600, 1025]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("n", [1, 2, 7])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_behind_prefixes(heads, kv_heads, dim, n, dtype):
    own = [n, n + 1, 31, 64, 129, 256, 257, 300, 513, 40, 9, 700, 33, 8, 100, 77]
    reads = [0, 1, 1, 2, 3, 3, 3, 4, 4, 5, 6, 7, 8, 8, 8, -1]
    run_shared([-1] * 10 + reads, [0] * 10 + [n] * 16, PREFIXES + own, heads, kv_heads, dim, dtype, seed=dim + n)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (14, 2, 64)])
def test_attend_shared_mixed_step(heads, kv_heads, dim):
    """Decode rows, windows, chunks and idle requests in any order behind two
    prefixes, one of which takes rows itself; rows past the step's end, strided q
    and out."""
    prefix = [3, -1, 6, -1, 3, 6, -1, 3, -1, 6, 3, 3]
    rows = [1, 5, 200, 0, 7, 0, 130, 1, 0, 1, 300, 2]
    kv = [10, 300, 333, 2000, 40, 64, 700, 1, 20, 257, 300, 514]
    _, _, out, _ = run_shared(prefix, rows, kv, heads, kv_heads, dim, torch.float16, spare=5, gap=kv_heads)
    assert bool((out[-5:] == 7).all())


@pytest.mark.parametrize("readers", [2, 5, 21, 22, 64, 200])
@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (8, 8, 64)])
def test_attend_one_prefix(readers, heads, kv_heads, dim):
    """From a few columns of one item of 128 to several full ones."""
    kv = [3000] + [1 + 37 * i % 400 for i in range(readers)]
    run_shared([-1] + [0] * readers, [0] + [1] * readers, kv, heads, kv_heads, dim, torch.bfloat16, seed=readers)


@pytest.mark.parametrize("prefix,own", [(40000, 1), (1, 40000), (30000, 5000)])
@pytest.mark.parametrize("readers", [1, 3])
def test_attend_shared_work_split(prefix, own, readers):
    """A long prefix or a long request over all CTAs."""
    run_shared([-1] + [0] * readers, [0] + [1] * readers, [prefix] + [own] * readers, 24, 4, 256, torch.float16)


def test_attend_shared_many_prefixes():
    """Hundreds of requests, each behind its own prefix or sharing it with one other."""
    P = 150
    kv = [1 + 13 * i % 500 for i in range(P)] + [1 + 7 * i % 300 for i in range(P + 50)]
    run_shared([-1] * P + list(range(P)) + list(range(50)), [0] * P + [1] * (P + 50), kv, 24, 4, 256, torch.float16)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (8, 8, 64)])
def test_attend_shared_rows_that_see_nothing(heads, kv_heads, dim):
    """No own tokens: the prefix alone; an empty prefix too: 0; more rows than own tokens."""
    prefix, rows, kv = [-1, -1, 0, 1, -1, 0, 1, 1, 0], [0, 0, 1, 1, 1, 9, 9, 1, 40], [300, 0, 0, 0, 0, 4, 4, 3, 17]
    _, _, out, _ = run_shared(prefix, rows, kv, heads, kv_heads, dim, torch.float16)
    assert int(out[1:3].count_nonzero()) == 0 and int(out[12:17].count_nonzero()) == 0


def test_attend_shared_large_scores():
    """Scores of hundreds, on either side of the join."""
    run_shared([-1, 0, 0, 0, 0], [0, 1, 1, 7, 40], [2000, 900, 1, 2000, 1000], 24, 4, 256, torch.float16, q_scale=60.0)


@pytest.mark.parametrize("rows", [[0, 1, 1, 1], [0, 9, 1, 30]])
def test_attend_shared_without_prefixes(rows):
    """Nothing shared: what `attend` gives.  Either is within (2^-11 + 3e-5) of the sum of
    p |v|, at most the largest |v| (6 x 1.1), of the same numbers (see `check`), and
    rounded once."""
    head, plan, out, _ = run_shared([-1] * 4, rows, [500, 700, 64, 1000], 24, 4, 256, torch.float16)
    plain = torch.empty_like(out)
    batch.attend(*head, plain, batch.attend_workspace("cuda", 256), max_rows=max(rows))
    tol = 2 * (2.0 ** -11 + 3e-5) * 6.6 + torch.finfo(out.dtype).eps * plain.double().abs() + 2.0 ** -24
    assert bool(((out.double() - plain.double()).abs() <= tol).all())


@pytest.mark.parametrize("rows", [1, 8])
@pytest.mark.parametrize("readers", [1, 2])
def test_attend_shared_nan_and_infinity(rows, readers):
    """A NaN or infinite score among a prefix's or a request's own tokens makes its
    rows NaN; the other requests' rows stay as they are."""
    kv, prefix = [300, 300] + [200] * readers + [100], [-1, -1] + [0] * readers + [1]
    new = [0, 0] + [rows] * readers + [rows]
    head, plan, out, ws = run_shared(prefix, new, kv, 24, 4, 256, torch.float16)
    table = head[5]
    last = -rows
    for value in (0x7F, 0xFF):
        for b in (0, 2):
            bad = [t.clone() for t in head[1:5]]
            bad[2].view(torch.uint8)[table[b, 0].long(), 7] = value
            got = torch.empty_like(out)
            batch.attend_shared(head[0], *bad, *head[5:], plan, got, ws, max_rows=rows)
            hit = slice(0, rows * readers) if b == 0 else slice(0, rows)
            assert bool(got[hit].isnan().all())
            assert torch.equal(got[last:], out[last:])
            if b == 2 and readers == 2:
                assert torch.equal(got[rows:2 * rows], out[rows:2 * rows])


@pytest.mark.parametrize("rows", [1, 10])
def test_attend_shared_bad_pages_and_plans(rows):
    """Table entries outside the pool count as absent tokens; a plan of another
    step is read within the step's bounds."""
    pool = make_pool(9, 4, 256, 5)
    table = i32([[0, -1, 2], [3, 4, 999], [-5, 5, 1], [6, 77, 7]])
    prefix = [-1, 0, 0, -1]
    head, plan, out, ws = run_shared(prefix, [0, rows, rows, rows], [600, 600, 600, 600], 24, 4, 256, torch.float16, pool=pool,
                                     table=table)
    assert _lib.device_error(clear=True) == 2
    good = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8], [0, 1, 2]])
    T = 3 * rows
    for wrong in ([0, 0, 0, 0, 900], [0, -5, T, T, T], [0, T, 0, T, 0]):
        bent = plan.clone()
        bent[:5] = i32(wrong)
        got = torch.full_like(out, 7.0)
        batch.attend_shared(*head[:5], good, *head[6:], bent, got, ws, max_rows=rows)
        assert _lib.device_error(clear=True) in (0, 1)
    bent = plan.clone()
    bent[5:9] = i32([900, 900, 900, -9])
    bent[13:] = i32([T, -1, 1 << 30] * rows)
    batch.attend_shared(*head[:5], good, *head[6:], bent, got, ws, max_rows=rows)
    assert _lib.device_error(clear=True) == 1


def test_attend_shared_lengths_beyond_the_table():
    pool = make_pool(6, 4, 256, 1)
    table = i32([[0, 1], [2, 3], [4, 5]])
    q = torch.randn(2, 24, 256, device="cuda").half()
    out, want = torch.empty_like(q), torch.empty_like(q)
    ws = batch.shared_workspace("cuda", 256, 2, 24)
    cu = np.array([0, 0, 1, 2])
    plan = make_plan([-1, 0, 0], [512, 100, 100], cu, 2)
    batch.attend_shared(q, *pool, table, i32(cu), i32([512, 100, 100]), plan, want, ws, max_rows=1)
    batch.attend_shared(q, *pool, table, i32(cu), i32([1 << 30, 100, 100]), plan, out, ws, max_rows=1)
    assert _lib.device_error(clear=True) == 1
    assert torch.equal(out, want)


def test_attend_shared_offsets_past_32_bits():
    """A pool of more than 4 GB of codes a tensor; the pages used lie at its end."""
    pages = 34000  # x 128 KB
    big = [torch.zeros(pages, PAGE, 4, w, dtype=torch.uint8, device="cuda") for w in (128, 128, 16, 16)]
    small = make_pool(6, 4, 256, 9)
    at = torch.tensor([33999, 33990, 20000, 33000, 32768, 16384])
    for b, s in zip(big, small):
        b[at] = s.view(torch.uint8)
    for new, prefix in (([0, 1, 1], [-1, 0, 0]), ([0, 8, 8], [-1, 0, 0]), ([0, 1, 0], [-1, 0, -1])):
        head, plan, out, ws = run_shared(prefix, new, [700, 500, 200], 24, 4, 256, torch.float16, pool=small,
                                         table=i32([[0, 1, 2], [3, 4, -1], [5, -1, -1]]))
        out2 = torch.empty_like(out)
        table = torch.where(head[5] >= 0, at.cuda()[head[5].clamp(min=0).long()], -1).to(torch.int32)
        batch.attend_shared(head[0], *big, table, *head[6:], plan, out2, ws, max_rows=8)
        assert torch.equal(out, out2)


# ----------------------------------------------------------------- together
def test_a_server_behind_two_prompts():
    """Prompts prefilled, read by requests that come and go: tables, plan, rotated
    append and attention on one stream, the later steps as one captured graph,
    against 64 bits over everything a request has seen."""
    heads, kv_heads, dim, dtype = 8, 2, 128, torch.bfloat16
    R, W, F, Tmax = 7, 6, 40, 820
    prefix_of = [-1, -1, 0, 0, 1, -1, 0]
    steps = [[300, 517, 0, 0, 0, 0, 0], [0, 0, 70, 3, 1, 9, 0], [0, 0, 1, 1, 1, 1, 5], [0, 0, 1, 1, 1, 1, 1],
             [0, 0, 1, 1, 1, 1, 1], [0, 0, -1, 1, 1, 0, 1], [0, 0, 2, 1, 1, 4, 1]]
    pool = make_pool(F, kv_heads, dim, 0)
    inv, qw, kw = freqs_of(32), weight_of(dim, 1), weight_of(dim, 2)
    lengths, held, new = i32([0] * R), i32([0] * R), i32([0] * R)
    ring, state = i32(range(F)), i32([0, F])
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    e = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, kv, held_out, state_out, slots, pos, req, far = e(R + 1), e(R), e(R), e(2), e(Tmax), e(Tmax), e(Tmax), e(Tmax)
    plan, ws = batch.prefix_plan("cuda", R, Tmax), batch.shared_workspace("cuda", dim, Tmax, heads)
    x = torch.zeros(Tmax, heads + 2 * kv_heads, dim, dtype=dtype, device="cuda")
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)
    q_out, out = torch.empty(Tmax, heads, dim, dtype=dtype, device="cuda"), torch.empty(Tmax, heads, dim, dtype=dtype,
                                                                                       device="cuda")
    whom = i32(prefix_of)

    def step():
        batch.build_tables(lengths, new, held, ring, state, table, cu, kv, held_out, state_out, slots, pos, req)
        batch.share_prefixes(whom, kv, cu, pos, req, plan, far)
        batch.append_rotated(q, k, v, q_out, *pool, slots, far, inv, q_weight=qw, k_weight=kw)
        batch.attend_shared(q_out, *pool, table, cu, kv, plan, out, ws, max_rows=Tmax)
        lengths.copy_(kv)
        held.copy_(held_out)
        state.copy_(state_out)

    seen = [([], []) for _ in range(R)]  # K (as held) and V rows of each request
    graph = None
    stream = torch.cuda.Stream()
    for i, counts in enumerate(steps):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda"))
        new.copy_(i32(counts))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            if i < 2:
                step()
            else:
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=stream):
                        step()
                graph.replay()
        torch.cuda.current_stream().wait_stream(stream)
        at = 0
        for b, n in enumerate(counts):
            if n < 0:
                seen[b] = ([], [])
            if n <= 0:
                continue
            rows = slice(at, at + n)
            before = sum(len(t) for t in seen[prefix_of[b]][0]) if prefix_of[b] >= 0 else 0
            mine = sum(len(t) for t in seen[b][0])
            p = before + mine + torch.arange(n, device="cuda")
            assert torch.equal(far[rows], p.int())
            y, _ = obatch.rotate(k[rows], p, inv, False, kw)
            seen[b][0].append(obatch.dequant(*obatch.quantise(y)))
            seen[b][1].append(obatch.dequant(*obatch.quantise(v[rows].double())))
            y, mag = obatch.rotate(q[rows], p, inv, False, qw)
            close(q_out[rows], y, mag, dtype)
            ks, vs = (sum((seen[g][j] for g in ([prefix_of[b]] if prefix_of[b] >= 0 else []) + [b]), []) for j in range(2))
            ks, vs = (torch.cat(t).repeat_interleave(heads // kv_heads, 1) for t in (ks, vs))
            s = torch.einsum("nhd,thd->hnt", q_out[rows].double(), ks) * dim ** -0.5
            j = torch.arange(len(ks), device="cuda")
            s = s.masked_fill(j[None] > p[:, None], -torch.inf).softmax(-1)
            check(out[rows], torch.einsum("hnt,thd->nhd", s, vs), torch.einsum("hnt,thd->nhd", s, vs.abs()), dtype)
            at += n
    assert lengths.tolist() == [300, 517, 2, 8, 6, 16, 9]


def test_two_graphs_with_workspaces_of_their_own():
    """Two captured calls replayed on two streams at once."""
    calls = []
    for seed in (1, 2):
        head, plan, out, ws = run_shared([-1, 0, 0, 0], [0, 1, 9, 1], [3000, 40, 300, 500], 24, 4, 256, torch.float16, seed=seed)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        got = torch.zeros_like(out)
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(5):
                batch.attend_shared(*head, plan, got, ws, max_rows=9)
        calls.append((graph, stream, got, out, head, plan, ws))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream, *_ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, out, *_ in calls:
        assert torch.equal(got, out)
