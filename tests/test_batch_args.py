"""Refusals of the many-request operators: nothing is launched (no GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from qwarz_b200 import _lib, batch, build, scoring


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def addr():
    buf = ctypes.create_string_buffer(1 << 16)
    yield (ctypes.addressof(buf) + 63) // 64 * 64


def refused(lib, rc, needle):
    assert rc == _lib.QWZ_EINVAL and needle in lib.qwz_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "required"), ({10: None}, "slots"), ({13: 0}, "requests"), ({14: 0}, "table_width"),
    ({15: 0}, "ring_size"), ({16: -1}, "rows"), ({8: "held"}, "share storage"),
])
def test_tables(lib, addr, change, needle):
    args = [addr + 256 * i for i in range(13)] + [4, 8, 16, 32, None]
    for i, value in change.items():
        args[i] = args[2] if value == "held" else value
    refused(lib, lib.qwz_batch_tables(*args), needle)


@pytest.mark.parametrize("out,other,at", [
    (7, 1, 0), (8, 0, 0), (8, 1, 0), (9, 0, 0), (9, 2, 4), (6, 1, 0), (6, 4, 0), (10, 0, 0), (11, 2, 0), (12, 3, 0),
    (7, 0, 4), (7, 0, -4), (6, 5, 64), (5, 0, 0), (5, 3, 0), (3, 2, 0),   # in part; tables and ring, which are written too
])
def test_tables_shared_storage(lib, addr, out, other, at):
    """An array that is written and shares bytes with one that is read is refused:
    every CTA reads all of the inputs while others write."""
    args = [addr + 256 * i for i in range(13)] + [4, 8, 16, 32, None]
    args[out] = args[other] + at
    refused(lib, lib.qwz_batch_tables(*args), "share storage")


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "k, v and slots"), ({2: None}, "required"), ({0: "odd"}, "aligned"), ({10: 4 * 256 - 8}, "k: the row stride"),
    ({11: 4 * 256 + 4}, "v: the row stride"), ({12: 0}, "num_kv_heads"), ({13: 96}, "head_dim"), ({14: 0}, "num_pages"),
    ({15: 2}, "dtype"), ({9: -1}, "rows"),
])
def test_append(lib, addr, change, needle):
    args = [addr + 256 * i for i in range(7)] + [None, None, 2, 1024, 1024, 4, 256, 8, 0, None]
    for i, value in change.items():
        args[i] = addr + 2 if value == "odd" else value
    refused(lib, lib.qwz_batch_append(*args), needle)


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "q and out"), ({8: "odd"}, "q and out"), ({1: None}, "required"), ({5: None}, "block_table"),
    ({9: None}, "workspace"), ({10: 16}, "workspace smaller"), ({11: -1}, "rows"), ({13: 0}, "max_rows"),
    ({14: 0}, "table_width"), ({15: 0}, "num_pages"), ({16: 23}, "num_q_heads"), ({16: 65 * 4}, "num_q_heads"),
    ({17: 0}, "num_kv_heads"), ({18: 80}, "head_dim"), ({19: 24 * 256 - 8}, "q: the row stride"),
    ({20: 24 * 256 + 4}, "out: the row stride"), ({21: 0.0}, "sm_scale"), ({21: float("inf")}, "sm_scale"),
    ({22: 2}, "dtype"),
])
def test_attend(lib, addr, change, needle):
    size = lib.qwz_batch_attend_workspace_bytes(256)
    args = [addr + 256 * i for i in range(10)] + [size, 4, 2, 1, 4, 8, 24, 4, 256, 6144, 6144, 0.0625, 0, None]
    for i, value in change.items():
        args[i] = addr + 2 if value == "odd" else value
    refused(lib, lib.qwz_batch_attend(*args), needle)


@pytest.mark.parametrize("change", [{11: 0}, {0: None, 8: None, 11: 0}, {5: None, 6: None, 7: None, 12: 0}])
def test_attend_without_work(lib, addr, change):
    """No rows or no requests: nothing is launched, whatever the pointers (those
    of empty tensors are null); the sizes are checked all the same."""
    size = lib.qwz_batch_attend_workspace_bytes(256)
    args = [addr + 256 * i for i in range(10)] + [size, 4, 2, 1, 4, 8, 24, 4, 256, 6144, 6144, 0.0625, 0, None]
    for i, value in change.items():
        args[i] = value
    assert lib.qwz_batch_attend(*args) == _lib.QWZ_OK
    args[16] = 23
    refused(lib, lib.qwz_batch_attend(*args), "num_q_heads")


def test_workspace_sizes(lib):
    assert lib.qwz_batch_attend_workspace_bytes(100) == 0
    sizes = [lib.qwz_batch_attend_workspace_bytes(d) for d in (64, 128, 256)]
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    assert lib.qwz_token_logprobs_workspace_bytes(4, 0, 1, 0) == 0
    assert lib.qwz_token_logprobs_workspace_bytes(4, 10, 33, 0) == 0
    assert lib.qwz_token_logprobs_workspace_bytes(4, 10, 3, 3) == 0
    a, b = (lib.qwz_token_logprobs_workspace_bytes(r, 1000, 8, 1) for r in (4, 5))
    assert 0 < a < b


@pytest.mark.parametrize("change,needle", [
    ({0: None}, "required"), ({0: "odd"}, "aligned"), ({5: None}, "top_logprobs"), ({7: None}, "workspace"),
    ({8: 16}, "workspace smaller"), ({9: -1}, "rows"), ({10: 0}, "vocab"), ({11: 33}, "top"), ({11: 11}, "top"),
    ({12: 9}, "row stride"), ({13: 3}, "dtype"),
])
def test_logprobs(lib, addr, change, needle):
    args = [addr, addr, 0] + [addr + 256 * i for i in range(5)] + [1 << 30, 2, 10, 3, 10, 1, None]
    for i, value in change.items():
        args[i] = addr + 1 if value == "odd" else value
    refused(lib, lib.qwz_token_logprobs(*args), needle)


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU fallback"):
        batch.build_tables(*[t] * 13)
    x = torch.zeros(2, 4, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        batch.append(x, x, *[t] * 5)
    with pytest.raises(ValueError, match="no CPU fallback"):
        batch.attend(x, *[t] * 9, max_rows=1)
    with pytest.raises(ValueError, match="no CPU fallback"):
        scoring.token_logprobs(torch.zeros(2, 8), *[t] * 6)


@pytest.mark.parametrize("current", [0, 1])
def test_launches_on_the_tensors_device(monkeypatch, current):
    """The call runs with the tensors' device current and on its stream, whichever was current before."""
    seen, now = [], [current]

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.was, now[0] = now[0], self.dev

        def __exit__(self, *_):
            now[0] = self.was

    class Lib:
        def qwz_op(self, *args):
            seen.append((now[0], args))
            return 0

    monkeypatch.setattr(batch, "_current_device", lambda: now[0])
    monkeypatch.setattr(batch, "_raw_stream", lambda dev: 100 + dev)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(batch._lib, "load", Lib)
    batch._launch(1, "qwz_op", 7, 8)
    assert seen == [(1, (7, 8, 101))] and now == [current]


@pytest.mark.parametrize("rows,stride", [(1, 1001), (1, 0), (1, 256), (0, 1001), (0, 0)])
def test_stride_of_one_row(rows, stride):
    """The row stride of at most one row means nothing, whatever the view gives."""
    assert batch._rows("k", torch.empty_strided((rows, 4, 64), (stride, 64, 1)), 4, 64) == (rows, 256)
    assert batch._rows("k", torch.empty_strided((2, 4, 64), (1001, 64, 1)), 4, 64) == (2, 1001)
