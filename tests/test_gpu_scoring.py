"""Token log probabilities (qwarz_b200.scoring) against a plain 64-bit form."""
from __future__ import annotations

import pytest
import torch

from oracle import batch as obatch
from qwarz_b200 import _lib, scoring

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_errors(cuda):
    _lib.device_error(clear=True)
    yield
    assert _lib.device_error(clear=True) == 0


def run(logits, ids, top, ws=None):
    T = logits.shape[0]
    dev = logits.device
    got = (torch.full((T,), 9.0, device=dev), torch.full((T,), 9.0, device=dev), torch.full((T, top), 9.0, device=dev),
           torch.full((T, top), -9, dtype=torch.int32, device=dev))
    ws = scoring.workspace(dev, T, logits.shape[1], top) if ws is None else ws
    scoring.token_logprobs(logits, ids, *got, ws)
    return got


def check(logits, ids, top):
    """FP32 sums of up to some hundred terms a chain (at most 512 x 2^-24 = 3e-5
    relative, 1e-6 as a random walk), scores to 2^-23 of their distance from the
    maximum: 1e-5 (1 + |value|)."""
    got, want = run(logits, ids, top), obatch.token_logprobs(logits, ids.long(), top)
    assert torch.equal(got[3].long(), want[3])
    for a, b in zip(got[:3], want[:3]):
        b = b.float().double()  # what FP32 can hold of it
        same = (a.double() == b) | (a.isnan() & b.isnan())
        err = torch.where(same, 0.0, (a.double() - b).abs())
        assert bool((err <= 1e-5 * (1 + torch.where(b.isfinite(), b.abs(), 0.0))).all()), float(err.max())
    again = run(logits, ids, top)
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(got, again))


def logits_of(T, V, dtype, seed, pad=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, V + pad, generator=g, device="cuda") * scale
    ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    return x.to(dtype)[:, :V], ids


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,top,pad", [(1, 1, 1, 0), (1, 7, 7, 0), (3, 33, 32, 1), (5, 4096, 0, 0), (2, 8191, 5, 2),
                                         (2, 8193, 20, 3), (7, 50257, 20, 0), (3, 151001, 32, 5), (300, 1000, 3, 7),
                                         (1500, 257, 2, 0), (1, 400003, 8, 0)])
def test_shapes(dtype, T, V, top, pad):
    check(*logits_of(T, V, dtype, V + top, pad), top)


def test_int32_ids_and_row_views():
    x, ids = logits_of(6, 5000, torch.bfloat16, 1, pad=24)
    check(x[1::2], ids[1::2].to(torch.int32).contiguous(), 4)  # every other row
    x, ids = logits_of(4, 5000, torch.float32, 2)
    check(x.expand(4, 5000)[:1].expand(4, 5000), ids, 4)       # one row four times, stride 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_values(dtype):
    """Constant rows, few distinct values, two equal maxima far apart, -0 and +0:
    the lowest index wins."""
    x = torch.zeros(5, 30000, device="cuda")
    x[1] = (torch.arange(30000, device="cuda") % 3).float()
    x[2, 29999] = x[2, 17] = 4.0
    x[3, ::2] = -0.0
    x[4] = -5.0
    check(x.to(dtype), torch.tensor([0, 2, 17, 1, 29999], device="cuda"), 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_sorted_rows(dtype):
    """Ascending rows overflow every list that is made from the row's beginning."""
    up = torch.arange(60000, device="cuda") * (1.0 if dtype == torch.float16 else 1e-3)
    x = torch.stack([up, up.flip(0)]).to(dtype)
    check(x, torch.tensor([59999, 4], device="cuda"), 20)


def test_impossible_tokens():
    """-inf logits: some, all but a few, all but fewer than the top asks, all."""
    x, _ = logits_of(5, 40000, torch.float32, 3)
    x[0, ::3] = -torch.inf
    x[1, 25:] = -torch.inf
    x[2, :39990] = -torch.inf
    x[3] = -torch.inf
    x[3, 12345] = 2.0
    x[4] = -torch.inf
    ids = torch.tensor([0, 3, 39999, 12345, 7], device="cuda")
    check(x, ids, 20)
    lp, ent, top, _ = run(x, ids, 20)
    assert lp[0] == -torch.inf and lp[3] == 0.0 and ent[3] == 0.0 and lp[4] == -torch.inf and ent[4] == 0.0
    assert bool((top[4] == -torch.inf).all())


def test_nan_and_infinity():
    x, ids = logits_of(3, 9000, torch.float32, 4)
    x[0, 5000] = torch.nan
    x[1, 3] = torch.inf
    lp, ent, top, at = run(x, ids, 4)
    assert bool(lp[:2].isnan().all()) and bool(ent[:2].isnan().all()) and bool(top[:2].isnan().all())
    assert 5000 not in at[0].tolist() and at[1, 0] == 3
    check(x[2:], ids[2:], 4)


def test_large_offsets():
    """All logits far from zero: nothing overflows, differences stay exact."""
    x, ids = logits_of(4, 20000, torch.float32, 5)
    x += torch.tensor([[1000.0], [-1000.0], [30000.0], [0.0]], device="cuda")
    check(x, ids, 5)
    wide = torch.tensor([[3e38, -3e38, 0.0, 1.0]], device="cuda")
    check(wide, torch.tensor([0], device="cuda"), 4)


def test_ids_outside():
    x, ids = logits_of(3, 1000, torch.bfloat16, 6)
    ids[0] = -1
    lp = run(x, ids, 2)[0]
    assert lp[0] == 0.0
    ids[1] = 1000
    lp = run(x, ids, 2)[0]
    assert lp[1].isnan() and _lib.device_error(clear=True) == 4


def test_workspace_of_a_larger_call():
    """A workspace made for a size serves every smaller one, in any type."""
    ws = scoring.workspace("cuda", 64, 60000, 20)
    for T, V, dtype in ((64, 60000, torch.float32), (1, 60000, torch.float32), (63, 300, torch.float16), (17, 59999, torch.bfloat16)):
        x, ids = logits_of(T, V, dtype, T)
        got, want = run(x, ids, 20, ws), run(x, ids, 20)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1, 4, 32])
def test_nan_ranks_after_impossible_tokens(dtype, top):
    """Rows of -inf with few finite logits and NaN at their beginning, in later
    parts, and everywhere: NaN takes no place from a -inf token."""
    x = torch.full((7, 50001), -torch.inf, device="cuda")
    x[0, 0] = torch.nan
    x[1, :40] = torch.nan
    x[1, [100, 30000, 50000]] = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    x[2, ::2] = torch.nan
    x[3] = torch.nan
    x[3, 49999] = -torch.inf
    x[4, :] = torch.nan
    x[5, 1:49000] = torch.nan
    x[5, 20000] = 5.0
    x[6, 3] = torch.inf
    x[6, 4:9] = torch.nan
    check(x.to(dtype), torch.tensor([0, 30000, 1, 49999, 7, 20000, -1], device="cuda"), top)
    check(x[:, :40].to(dtype), torch.tensor([0, 39, 1, 2, 7, 20, -1], device="cuda"), top)
