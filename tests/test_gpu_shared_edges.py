"""The operators for requests that share prefixes (qwarz_b200.batch) at their edges: plans
that do not fit, denied prefixes, weights, the ends of the types' ranges, long steps."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import batch as obatch
from qwarz_b200 import _lib, batch
from tests import test_gpu_shared as shared
from tests.test_gpu_batch import check, i32, make_pool, make_tables
from tests.test_gpu_shared import freqs_of, make_plan, make_rows, make_slots, run_shared, weight_of

pytestmark = pytest.mark.gpu
PAGE = 256


@pytest.fixture(autouse=True)
def clean_errors(cuda):
    _lib.device_error(clear=True)
    yield
    assert _lib.device_error(clear=True) == 0  # a test that expects a bit clears it itself


# ------------------------------------------------------- plans that do not fit
def bent_step(seed, many):
    """A step with a wide request (so that no prefix is read directly): one prefix whose item is
    shared by many CTAs, or forty whose items lie within one."""
    if many:
        prefix, rows, kv = [-1] * 40, [0] * 40, [600] * 40
        for g in range(40):
            prefix += [g, g]
            rows += [10, 1 + g % 3]
            kv += [200 + g, 40 + 9 * g]
        layout = (8, 8, 64)
    else:
        prefix, rows, kv, layout = [-1, 0, 0, 0, -1], [0, 10, 1, 1, 2], [600, 300, 40, 300, 50], (24, 4, 256)
    heads, kv_heads, dim = layout
    pages = sum(-(-n // PAGE) for n in kv)
    pool, table = make_pool(pages, kv_heads, dim, seed), make_tables(kv, 3, pages, seed)
    cu = np.concatenate([[0], np.cumsum(rows)])
    return prefix, rows, kv, layout, pool, table, cu, make_plan(prefix, kv, cu, int(cu[-1]))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("how", ["outside", "emptied", "later", "range"])
def test_rows_the_plan_does_not_list(how, many):
    """Rows behind a prefix that the plan does not list (entries outside the step's rows, an
    emptied range, one that begins a row late, one that is none) see their own tokens alone and
    set an error bit, whatever an earlier call left in the workspace; the others are as ever."""
    prefix, rows, kv, (heads, kv_heads, dim), pool, table, cu, plan = bent_step(3, many)
    R, T = len(kv), int(cu[-1])
    ws = batch.shared_workspace("cuda", dim, T, heads)
    ws.fill_(0xFF)
    q = [torch.randn(T, heads, dim, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").half() for s in (1, 2)]
    args = (*pool, table, i32(cu), i32(kv))
    batch.attend_shared(q[0], *args, plan, torch.empty_like(q[0]), ws, max_rows=10)
    bent, listed = plan.clone(), plan[3 * R + 1:]
    if how == "outside":
        at = torch.tensor([0, 3, 10])
        bent[3 * R + 1 + at] = i32([T, -1, 1 << 30])
        gone = listed[at.cuda()]
    elif how == "emptied":
        bent[:R + 1] = 0
        gone = listed[listed >= 0]
    else:
        bent[0] = 1 if how == "later" else -5
        gone = listed[:1 if how == "later" else int(plan[1])]
    missing = torch.zeros(T, dtype=torch.bool, device="cuda")
    missing[gone.long()] = True
    room = torch.full((T + 6, heads, dim), 7.0, dtype=torch.float16, device="cuda")
    out = room[3:-3]
    batch.attend_shared(q[1], *args, bent, out, ws, max_rows=10)
    assert _lib.device_error(clear=True) == 1
    both, mag = obatch.attend_shared(q[1], *args, prefix, out, dim ** -0.5)
    alone, mag_alone = obatch.attend_shared(q[1], *args, [-1] * R, out, dim ** -0.5)
    some = missing[:, None, None]
    check(out, torch.where(some, alone, both), torch.where(some, mag_alone, mag), torch.float16)
    assert bool((room[:3] == 7).all()) and bool((room[-3:] == 7).all())


def test_a_wide_reader_of_an_emptied_prefix():
    """The only reader has too many rows to read its prefix by itself, and the plan lists none."""
    heads, kv_heads, dim, kv = 24, 4, 256, [600, 300]
    pool, table, cu = make_pool(5, kv_heads, dim, 1), i32([[0, 1, 2], [3, 4, -1]]), np.array([0, 0, 10])
    plan = make_plan([-1, 0], kv, cu, 10)
    q = torch.randn(10, heads, dim, device="cuda").half()
    out, ws = torch.empty_like(q), batch.shared_workspace("cuda", dim, 10, heads)
    args = (q, *pool, table, i32(cu), i32(kv))
    batch.attend_shared(*args, plan, out, ws, max_rows=10)
    plan[:3] = 0
    batch.attend_shared(*args, plan, out, ws, max_rows=10)
    assert _lib.device_error(clear=True) == 1
    want, mag = obatch.attend_shared(*args, [-1, -1], out, dim ** -0.5)
    check(out, want, mag, torch.float16)


# --------------------------------------------------------------------- weights
@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("rows", [[0, 1, 1, 40], [0, 1, 1, 1], [0, 130, 7, 9]])
def test_weights_add_up_to_one(heads, kv_heads, dim, rows):
    """Where every V is 1 the output is exactly 1, with some keys that draw most of the weight.

    The sum of the weights takes what is multiplied with V, so both are FP32 sums of the same
    numbers: at most 3,000 additions of 2^-24 each on either side, and 2^-25 a weight against a
    largest one of 2^6 where earlier weights were scaled down, 3,000 x (2^-23 + 2^-31) at the very
    worst and, over chains of at most 750 weights, below 2^-12, half of FP16's step below 1."""
    kv = [2000, 300, 7, 700]
    pool = make_pool(14, kv_heads, dim, 3)
    pool[1].fill_(0x22)
    pool[3].view(torch.uint8).fill_(0x38)
    cu = np.concatenate([[0], np.cumsum(rows)])
    T, prefix = int(cu[-1]), [-1, 0, 0, 0]
    q = 2 * torch.randn(T, heads, dim, generator=torch.Generator(device="cuda").manual_seed(dim), device="cuda").half()
    out = torch.empty_like(q)
    batch.attend_shared(q, *pool, make_tables(kv, 8, 14, 3), i32(cu), i32(kv), make_plan(prefix, kv, cu, T), out,
                        batch.shared_workspace("cuda", dim, T, heads), max_rows=max(rows))
    assert bool((out == 1).all()), f"{float((out != 1).float().mean()):.2%}, {float(out.min())} to {float(out.max())}"


# ------------------------------------------------------ prefixes without tokens
def test_a_denied_prefix():
    """A prefix whose rows get no page has no tokens in the step: its readers, which have pages
    and are granted, would have wrong positions.  It counts as none and sets a bit."""
    R, T, W = 4, 13, 4
    e = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1]])
    cu, kv, held, state, slots, pos, req, far = e(R + 1), e(R), e(R), e(2), e(T), e(T), e(T), e(T)
    batch.build_tables(i32([250, 9, 300, 30]), i32([10, 1, 0, 2]), i32([1, 1, 2, 1]), i32([-1] * 8), i32([0, 0]), table, cu, kv,
                       held, state, slots, pos, req)
    assert kv.tolist() == [0, 10, 300, 32] and _lib.device_error(clear=True) == 16
    plan = batch.prefix_plan("cuda", R, T)
    batch.share_prefixes(i32([-1, 0, -1, 2]), kv, cu, pos, req, plan, far)
    assert _lib.device_error(clear=True) == 1
    want, why = obatch.share_prefixes([-1, 0, -1, 2], kv.tolist(), cu.tolist(), pos.tolist(), req.tolist())
    assert why and plan.tolist() == sum(want[:4], []) and far.tolist() == want[4]
    assert want[1] == [-1, -1, -1, 2] and far[10:].tolist() == [9, 330, 331]


def test_an_empty_prefix_is_no_error():
    """One without rows and tokens is a prefix all the same."""
    plan, far = batch.prefix_plan("cuda", 2, 1), i32([-7])
    batch.share_prefixes(i32([-1, 0]), i32([0, 6]), i32([0, 0, 1]), i32([5]), i32([1]), plan, far)
    assert plan.tolist() == [0, 1, 1, -1, 0, 1, -1, 0] and far.tolist() == [5]


# ------------------------------------------------------------------ most rows
def test_share_most_rows():
    """Arrays of 2^31 - 9 rows: the positions of the last ones are written, and nothing else is read."""
    T = (1 << 31) - 9
    req = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    pos = torch.full((T,), 5, dtype=torch.int32, device="cuda")
    req[:6], req[-3:] = 1, 1
    plan = batch.prefix_plan("cuda", 2, T)
    plan.fill_(-7)
    batch.share_prefixes(i32([-1, 0]), i32([40, 6]), i32([0, 0, 6]), pos, req, plan, pos)
    assert plan[:14].tolist() == [0, 6, 6, -1, 0, 1, -1, 0, 1, 2, 3, 4, 5, -1] and plan[-2:].tolist() == [-1, -1]
    assert pos[:7].tolist() == [45] * 6 + [5] and pos[-4:].tolist() == [5, 45, 45, 45]
    assert int((plan[13:] != -1).sum()) == 0 and int((pos != 5).sum()) == 9


# ------------------------------------------------------------- Q's whole range
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("heads,dim,freqs", [(24, 256, 32), (5, 128, 64), (3, 64, 16), (70, 64, 24)])
@pytest.mark.parametrize("rows", [1, 250])
def test_rotated_smallest_and_largest_q(rows, heads, dim, freqs, eps, neighbours):
    """Q heads whose squares 32 bits do not hold are normed as any other: 18 x 2^-24 of the two
    terms (see `close`), the output's half step of 2^-8, and its half step below 2^-126."""
    scales = [1.0, 2.0 ** -90, 2.0 ** -60, 2.0 ** -20, 2.0 ** 30, 2.0 ** 63, 2.0 ** 80, 2.0 ** 120, 2.0 ** -126]
    T = len(scales) * rows
    q, k, v, _ = make_rows(T, heads, 1, dim, torch.bfloat16, 8)
    q.mul_(torch.tensor(scales * rows, device="cuda").bfloat16()[:, None, None])
    q[2, 1] = 0.0
    P = T // PAGE + 1
    pool = [torch.zeros(P, PAGE, 1, w, dtype=torch.uint8, device="cuda") for w in (dim // 2, dim // 2, dim // 16, dim // 16)]
    out = torch.empty_like(q.contiguous())
    w, positions, inv = weight_of(dim, 3), i32(range(5, 5 + T)), freqs_of(freqs)
    batch.append_rotated(q, k, v, out, *pool, make_slots(T, P, 4), positions, inv, neighbours, q_weight=w, eps=eps)
    packed = q.contiguous()  # and in place
    batch.append_rotated(packed, k, v, packed, *pool, make_slots(T, P, 4), positions, inv, neighbours, q_weight=w, eps=eps)
    assert torch.equal(packed.view(torch.int16), out.view(torch.int16))
    if eps == 0.0:  # 0 / 0, as the formula says
        assert bool(out[2, 1].isnan().all())
        out[2, 1] = q[2, 1] = 0.0
    y, mag = obatch.rotate(q, positions, inv, neighbours, w, float(np.float32(eps)))
    if eps == 0.0:
        y[2, 1] = mag[2, 1] = 0.0
    off = mag * 18 * 2.0 ** -24
    tol = off + (y.abs() + off) * 2.0 ** -8 + 2.0 ** -134
    assert bool(((out.double() - y).abs() <= tol).all()), float(((out.double() - y).abs() / tol).max())


# -------------------------------------------------------------------- storage
def test_rotated_arrays_side_by_side():
    """Outputs that touch inputs and each other, and arrays between two rows of q_out."""
    T, heads, kv_heads, dim = 7, 6, 2, 64
    q, k, v, _ = make_rows(T, heads, kv_heads, dim, torch.float16, 4)
    slots, positions, inv = make_slots(T, 1, 4), i32(range(T)), freqs_of(16)
    codes, scales = PAGE * kv_heads * dim // 2, PAGE * kv_heads * dim // 16
    got = []
    for packed in (False, True):
        if packed:  # rows of q_out 4 MB apart, the first one with everything else behind it
            room = torch.zeros(T, 1 << 21, dtype=torch.float16, device="cuda")
            out = room[:, :heads * dim].view(T, heads, dim)
            at = heads * dim
            rest = []
            for n in (T * kv_heads * dim * 2,) * 2 + (codes, codes, scales, scales):
                rest.append(room[0, at:at + n // 2])
                at += n // 2
            kh, vh = (t.view(T, kv_heads, dim) for t in rest[:2])
            pool = [t.view(torch.uint8).view(1, PAGE, kv_heads, -1) for t in rest[2:]]
        else:
            out = torch.zeros(T, heads, dim, dtype=torch.float16, device="cuda")
            kh, vh = (torch.zeros(T, kv_heads, dim, dtype=torch.float16, device="cuda") for _ in range(2))
            pool = [torch.zeros(1, PAGE, kv_heads, w, dtype=torch.uint8, device="cuda") for w in (32, 32, 4, 4)]
        batch.append_rotated(q, k, v, out, *pool, slots, positions, inv, k_held=kh, v_held=vh)
        got.append([out, kh, vh, *pool])
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ------------------------------------------------------------------- more steps
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [[0, 1, 1], [0, 8, 8], [0, 1, 40]])
def test_attend_shared_infinite_query(rows, dtype):
    """A query element that is not finite makes its row and head NaN and nothing else."""
    head, plan, out, ws = run_shared([-1, 0, 0], rows, [3000, 300, 200], 24, 4, 256, dtype)
    for value in (float("inf"), float("nan")):
        q = head[0].clone()
        q[-1, 5, 100] = value
        got = torch.empty_like(out)
        batch.attend_shared(q, *head[1:], plan, got, ws, max_rows=max(rows))
        assert bool(got[-1, 5].isnan().all())
        got[-1, 5] = out[-1, 5]
        assert torch.equal(got, out)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (64, 8, 128), (14, 2, 64)])
def test_attend_shared_long_chunks(heads, kv_heads, dim):
    """Prompt chunks of 1,100 and 2,000 rows, decode rows and a window behind two prefixes."""
    run_shared([-1, -1, 0, 1, 0, 0, 1], [0, 0, 1100, 2000, 1, 7, 1], [700, 257, 1100, 2300, 500, 40, 9], heads, kv_heads, dim,
               torch.bfloat16)


@pytest.mark.parametrize("heads,kv_heads,dim,freqs", [(64, 8, 128, 64), (48, 8, 256, 32), (49, 7, 128, 16), (128, 4, 64, 32)])
def test_rotated_wide_layouts(heads, kv_heads, dim, freqs):
    """More Q heads than one warp's task holds, in long steps and short ones."""
    for T in (1101, 5):
        shared.test_rotated(T, heads, kv_heads, dim, freqs, False, True, torch.bfloat16)


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (8, 8, 64)])
def test_attend_shared_many_long_prefixes(heads, kv_heads, dim):
    """As many prefixes as before, too long for their readers to read them by themselves."""
    P = 150
    kv = [400 + 13 * i % 1700 for i in range(P)] + [1 + 7 * i % 300 for i in range(P + 50)]
    run_shared([-1] * P + list(range(P)) + list(range(50)), [0] * P + [1] * (P + 50), kv, heads, kv_heads, dim, torch.float16)


@pytest.mark.parametrize("prefix", [3060, 3080])
def test_attend_shared_on_either_side_of_a_rule(prefix):
    """50 rows behind a prefix whose tokens x KV heads x rows are just below 600 K, and just above."""
    run_shared([-1] + [0] * 50, [0] + [1] * 50, [prefix] + [1 + 31 * i % 290 for i in range(50)], 24, 4, 256, torch.bfloat16)
