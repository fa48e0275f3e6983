"""csrc/pynative.cpp: the CPython binding of the device entries."""
import ctypes as C

import numpy as np
import pytest

import rustorch_amd as ra
from rustorch_amd import _lib as L


def test_native_binding_converts_arguments_and_reports_errors():
    """Addresses, streams and shapes as objects, errors as the tuple errors.check takes."""
    class Buf:
        ptr = 16

    class Handle:
        _as_parameter_ = C.c_void_p(0)

    call = L.native.rt_gqa_decode_online_bf16
    for stream in (None, 0, C.c_void_p(), Handle()):
        for buf in (16, np.int64(16), Buf()):
            assert call(stream, buf, buf, buf, buf, 8, 3, 1, 64, 10)[:4] == (L.RT_ERR_HEAD_COUNT_MISMATCH, -1, 8, 3)
    with pytest.raises(ra.Overflow) as e:
        ra.LlmKernels.gqa_decode_online_bf16(None, 16, 16, 16, 16, 8, 2, 11, 64, 10)
    assert (e.value.requested, e.value.max) == (11, 10)
    with pytest.raises(ra.ZeroDim):
        ra.flash_forward_bf16_dev(ra.AttentionShape.new(1, 1, 4, 0), 16, 16, 16, 16)
    for bad in ("x", 1.5, [16]):
        with pytest.raises(TypeError):
            call(None, bad, 16, 16, 16, 8, 2, 1, 64, 10)
    with pytest.raises(TypeError):
        call(None, 16, 16, 16, 16, 8, 2, 1, 64)
    with pytest.raises(TypeError):
        call(None, 16, 16, 16, 16, 8, 2, 1.0, 64, 10)


def test_an_address_is_taken_from_each_object_by_itself():
    """Objects of one class that hold their address in different ways, in any order: what one call saw is nothing to the next."""
    class Gpu:
        """A tensor's protocol, or only the address."""

        def __init__(self, tensor, contiguous=True, cuda=True):
            if tensor:
                self.is_cuda, self.is_contiguous, self.data_ptr = cuda, (lambda: contiguous), (lambda: 32)
            else:
                self.ptr = 48

    call = L.native.rt_gqa_decode_online_bf16
    mismatch = (L.RT_ERR_HEAD_COUNT_MISMATCH, -1, 8, 3)
    for buf in (Gpu(False), Gpu(True), Gpu(False), Gpu(True), Gpu(False)):
        assert call(None, buf, 16, buf, 16, 8, 3, 1, 64, 10)[:4] == mismatch
    for bad in (Gpu(True, contiguous=False), Gpu(True, cuda=False)):
        for _ in range(2):
            with pytest.raises(AssertionError):
                call(None, bad, 16, 16, 16, 8, 3, 1, 64, 10)
    broken = Gpu(True)
    broken.data_ptr = lambda: 1 // 0
    for _ in range(2):
        with pytest.raises(ZeroDivisionError):
            call(None, broken, 16, 16, 16, 8, 3, 1, 64, 10)
    half = Gpu(False)
    half.is_cuda = True  # says so, and has an address alone
    assert call(None, half, 16, half, 16, 8, 3, 1, 64, 10)[:4] == mismatch


def test_a_tensor_that_is_not_on_the_gpu_is_refused():
    torch = pytest.importorskip("torch")
    call = L.native.rt_gqa_decode_online_bf16
    for _ in range(2):
        with pytest.raises(AssertionError):
            call(None, torch.zeros(4), 16, 16, 16, 8, 3, 1, 64, 10)
    # (and a class that comes behind it)
    class Buf:
        ptr = 16

    assert call(None, Buf(), 16, Buf(), 16, 8, 3, 1, 64, 10)[:4] == (L.RT_ERR_HEAD_COUNT_MISMATCH, -1, 8, 3)
