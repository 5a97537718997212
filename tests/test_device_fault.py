"""Reading the fault word from Python."""

import types

import pytest
import torch

from kernels import _native, ops


def test_word_reaches_the_caller(monkeypatch):
    """The library's answer, its status and the device's index, with a library that stands in for it."""
    asked = []

    def answer(device, bits):
        asked.append(device)
        bits._obj.value = 1
        return _native.QS_OK if device < 2 else _native.QS_EINVAL

    monkeypatch.setattr(_native, "lib", lambda: types.SimpleNamespace(qs_device_fault=answer, qs_last_error=lambda: b"no such device"))
    assert _native.device_fault() == 1 and _native.device_fault(1) == 1 and asked == [0, 1]
    with pytest.raises(_native.QsError):
        _native.device_fault(2)


@pytest.mark.gpu
def test_products_leave_it_clear():
    w = torch.zeros((256, 144 * 4), dtype=torch.uint8, device="cuda")
    x = torch.zeros((300, 34 * 32), dtype=torch.uint8, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        assert not ops.matmul(w, 12, x, out_dtype=dtype).any()
    assert _native.device_fault() == 0
