"""Refusals of the operators for requests that share prefixes: nothing is
launched (no GPU).  The plain forms agree with each other."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import batch as obatch
from oracle import nvfp4
from qwarz_b200 import _lib, batch, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def addr():
    buf = ctypes.create_string_buffer(1 << 20)
    yield (ctypes.addressof(buf) + 63) // 64 * 64


def refused(lib, rc, needle):
    assert rc == _lib.QWZ_EINVAL and needle in lib.qwz_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "required"), ({1: None}, "required"), ({2: None}, "required"), ({5: None}, "required"),
    ({3: None}, "positions"), ({4: None}, "positions"), ({6: None}, "positions"), ({7: 0}, "requests"),
    ({7: (1 << 14) + 1}, "requests"), ({8: -1}, "rows"),
    ({5: 0}, "share storage"), ({5: 2}, "share storage"), ({5: 3}, "share storage"), ({5: 4}, "share storage"),
    ({6: 1}, "share storage"), ({6: 4}, "share storage"), ({6: 5}, "share storage"), ({6: (3, 4)}, "share storage"),
    ({6: (5, 44)}, "share storage"),
])
def test_share(lib, addr, change, needle):
    args = [addr + 1024 * i for i in range(7)] + [4, 16, None]
    for i, value in change.items():
        if i in (5, 6) and value is not None:  # the address of another argument
            value = args[value] if isinstance(value, int) else args[value[0]] + value[1]
        args[i] = value
    refused(lib, lib.qwz_batch_share_prefixes(*args), needle)


ROTATE = {"q": 0, "k": 1, "v": 2, "q_out": 3, "slots": 8, "positions": 9, "inv_freq": 10, "q_weight": 11, "k_weight": 12,
          "k_held": 13, "v_held": 14, "rows": 15, "q_stride": 16, "k_stride": 17, "v_stride": 18, "q_out_stride": 19,
          "q_heads": 20, "kv_heads": 21, "dim": 22, "freqs": 23, "neighbours": 24, "eps": 25, "pages": 26, "dtype": 27}


def rotate_args(addr):
    return [addr + 65536 * i for i in range(4)] + [addr + 0x80000 + 4096 * i for i in range(9)] + [None, None] + \
        [2, 1024, 256, 256, 1024, 4, 1, 256, 32, 0, 1e-6, 8, 0, None]


@pytest.mark.parametrize("change,needle", [
    ({"q": None}, "q and q_out"), ({"q_out": None}, "q and q_out"), ({"q": 8}, "q and q_out"), ({"k": None}, "k, v and slots"),
    ({"slots": None}, "slots"), ({"positions": None}, "positions"), ({"inv_freq": None}, "inv_freq"),
    ({"q_weight": 4}, "q_weight"), ({"k_weight": 8}, "k_weight"), ({"rows": -1}, "rows"),
    ({"q_stride": 1016}, "q: the row stride"), ({"q_out_stride": 1028}, "q_out: the row stride"),
    ({"k_stride": 248}, "k: the row stride"), ({"q_heads": 0}, "num_q_heads"), ({"dim": 96}, "head_dim"),
    ({"freqs": 4}, "num_freqs"), ({"freqs": 136}, "num_freqs"), ({"freqs": -8}, "num_freqs"), ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"pages": 0}, "num_pages"), ({"dtype": 2}, "dtype"),
])
def test_rotated(lib, addr, change, needle):
    args = rotate_args(addr)
    for name, value in change.items():
        i = ROTATE[name]
        args[i] = args[i] + value if i < 15 and isinstance(value, int) else value
    refused(lib, lib.qwz_batch_append_rotated(*args), needle)


@pytest.mark.parametrize("change,needle", [
    # q_out over a part of q, over another row of it, at another stride, over k, over v; held values over k, q_out and q
    ({"q_out": ("q", 16)}, "q_out must be q"), ({"q_out": ("q", 2048)}, "q_out must be q"),
    ({"q_out": ("q", 0), "q_out_stride": 2048}, "q_out must be q"), ({"q_out": ("k", 0)}, "k or v"),
    ({"q_out": ("v", 0)}, "k or v"), ({"k_held": ("k", 0)}, "k_held"), ({"v_held": ("q_out", 512)}, "k_held"),
    ({"v_held": ("q", 0)}, "k_held"),
    # rows of one packed tensor: q_out reaches into k's columns
    ({"q_stride": 1536, "k": ("q", 2048), "k_stride": 1536, "q_out": ("q", 16), "q_out_stride": 1536}, "q_out must be q"),
    ({"k": ("q_out", 1024), "k_stride": 1536, "q_out_stride": 1536}, "k or v"),
    ({"k_held": ("k_weight", 65536), "v_held": ("k_weight", 66000 // 16 * 16)}, "k_held and v_held must not share storage"),
])
def test_rotated_shared_storage(lib, addr, change, needle):
    args = rotate_args(addr)
    for name, value in change.items():
        args[ROTATE[name]] = args[ROTATE[value[0]]] + value[1] if isinstance(value, tuple) else value
    refused(lib, lib.qwz_batch_append_rotated(*args), needle)


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "q and out"), ({9: 2}, "q and out"), ({5: None}, "block_table"), ({8: None}, "plan"),
    ({10: None}, "workspace"), ({11: 16}, "workspace smaller"), ({11: "plain"}, "workspace smaller"), ({12: -1}, "rows"),
    ({13: (1 << 14) + 1}, "requests"), ({14: 0}, "max_rows"), ({15: 0}, "table_width"), ({16: 0}, "num_pages"),
    ({17: 23}, "num_q_heads"), ({19: 80}, "head_dim"), ({20: 24 * 256 - 8}, "q: the row stride"), ({22: 0.0}, "sm_scale"),
    ({23: 2}, "dtype"), ({}, "out must not share"),
])
def test_attend_shared(lib, addr, change, needle):
    size = lib.qwz_batch_shared_workspace_bytes(256, 4, 24)
    args = [addr + 256 * i for i in range(11)] + [size, 4, 2, 1, 4, 8, 24, 4, 256, 6144, 6144, 0.0625, 0, None]
    for i, value in change.items():
        if value == "plain":
            value = lib.qwz_batch_attend_workspace_bytes(256)
        args[i] = addr + 2 if i == 9 else value
    refused(lib, lib.qwz_batch_attend_shared(*args), needle)


def test_without_work(lib, addr):
    args = [addr + 256 * i for i in range(11)] + [16, 0, 2, 1, 4, 8, 24, 4, 256, 6144, 6144, 0.0625, 0, None]
    assert lib.qwz_batch_attend_shared(*args) == 0
    args = rotate_args(addr)
    args[ROTATE["rows"]] = 0
    args[0] = args[3] = args[9] = None
    assert lib.qwz_batch_append_rotated(*args) == 0


def test_workspace_sizes(lib):
    plain = lib.qwz_batch_attend_workspace_bytes(128)
    none = lib.qwz_batch_shared_workspace_bytes(128, 0, 8)
    assert plain < none < plain + (1 << 20)
    # two parts of a row and head: output, maximum and sum, a word
    assert lib.qwz_batch_shared_workspace_bytes(128, 4, 6) == none + 2 * 24 * 4 * (128 + 3)
    none = lib.qwz_batch_shared_workspace_bytes(256, 0, 64)
    assert lib.qwz_batch_shared_workspace_bytes(256, 1 << 20, 64) == none + 2 * (64 << 20) * 4 * 259
    for bad in ((96, 1, 8), (128, -1, 8), (128, 1, 0), (128, 1, 1 << 15)):
        assert lib.qwz_batch_shared_workspace_bytes(*bad) == 0
    with pytest.raises(ValueError):
        batch.shared_workspace("cpu", 96, 1, 8)


def test_python_refuses_cpu_tensors():
    t = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        batch.share_prefixes(t, t, t, t, t, t, t)
    x = torch.zeros(1, 4, 64, dtype=torch.float16)
    pool = [torch.zeros(1, 256, 1, w, dtype=torch.uint8) for w in (32, 32, 4, 4)]
    with pytest.raises(ValueError, match="CUDA"):
        batch.append_rotated(x, x, x, x, *pool, t, t, torch.zeros(8))
    with pytest.raises(ValueError, match="CUDA"):
        batch.attend_shared(x, *pool, t, t, t, t, x, t, 1)
    assert batch.prefix_plan("cpu", 5, 7).numel() == 23


def test_plain_quantiser_is_the_writers():
    """On 16-bit rows the exact quotients round as the 32-bit ones of the writer."""
    x = torch.randn(64, 2, 64, generator=torch.Generator().manual_seed(1)) * torch.logspace(-4, 4, 64)[:, None, None]
    for dtype in (torch.float16, torch.bfloat16):
        rows = x.to(dtype).float()
        codes, scales = obatch.quantise(rows.double())
        want, want_scales = nvfp4.quantize_rows(rows.numpy().reshape(-1, 64))
        assert (codes.numpy().reshape(-1, 32) == want).all() and (scales.numpy().reshape(-1, 4) == want_scales).all()


def test_plain_rotation_is_relative():
    """Products of rotated rows depend on the difference of their positions."""
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(1, 3, 64, generator=g), torch.randn(1, 3, 64, generator=g)
    freq = 10000.0 ** (-torch.arange(16) / 16)
    for neighbours in (False, True):
        dots = []
        for a, b in ((5, 3), (100005, 100003)):
            y = obatch.rotate(q, torch.tensor([a]), freq, neighbours)[0]
            z = obatch.rotate(k, torch.tensor([b]), freq, neighbours)[0]
            dots.append((y * z).sum(-1))
        assert torch.allclose(dots[0], dots[1], atol=1e-9)
        assert torch.equal(obatch.rotate(q, torch.tensor([0]), freq, neighbours)[0], q.double())
