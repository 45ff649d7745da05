"""append_rotated refuses outputs that share storage with what it reads or with each
other, as include/qwz_b200.h says (nothing is launched; no GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from qwarz_b200 import _lib, build
from tests.test_shared_args import ROTATE

# (what passes the checks would be launched on host addresses)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="refusals are tested without a GPU")
CACHES = {"k_cache": 4, "v_cache": 5, "k_scales": 6, "v_scales": 7}
INDEX = ROTATE | CACHES
MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def addr():
    buf = ctypes.create_string_buffer(32 * MB)
    yield (ctypes.addressof(buf) + 63) // 64 * 64


def make_args(addr):
    """2 rows of 4/1/256, 8 pages; every array a MB of its own."""
    at = [addr + i * MB for i in range(15)]
    return at + [2, 1024, 256, 256, 1024, 4, 1, 256, 32, 0, 1e-6, 8, 0, None]


BYTES = {"q": 4096, "k": 1024, "v": 1024, "q_out": 4096, "k_cache": 8 * 256 * 128, "v_cache": 8 * 256 * 128,
         "k_scales": 8 * 256 * 16, "v_scales": 8 * 256 * 16, "slots": 8, "positions": 8, "inv_freq": 128, "q_weight": 1024,
         "k_weight": 1024, "k_held": 1024, "v_held": 1024}
WRITTEN = ("q_out", "k_held", "v_held", "k_cache", "v_cache", "k_scales", "v_scales")
PAIRS = [(w, o) for w in WRITTEN for o in BYTES if o != w and (w, o) != ("q_out", "q")]


@pytest.mark.parametrize("written,other", PAIRS)
@pytest.mark.parametrize("end", [False, True])
def test_refused(lib, addr, written, other, end):
    """The other array begins in the written one's last 16 bytes, or ends in its first."""
    args = make_args(addr)
    step = -((BYTES[other] - 1) // 16 * 16) if end else (BYTES[written] - 1) // 16 * 16
    args[INDEX[other]] = args[INDEX[written]] + step
    assert lib.qwz_batch_append_rotated(*args) == _lib.QWZ_EINVAL
    assert "share" in lib.qwz_last_error().decode()
