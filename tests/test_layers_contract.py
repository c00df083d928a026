"""CPU: what the layer operators promise about workspaces, sizes, dispatch and derivatives; nothing here
reaches a GPU (calls of the C ABI return before any CUDA call)."""
import ctypes

import pytest
import torch

import qrb200
from qrb200 import _lib

FP8 = torch.float8_e4m3fn
BF = torch.bfloat16


def size_of(fn, *args):
    n = ctypes.c_size_t()
    assert getattr(_lib.lib(), fn)(*args, ctypes.byref(n)) == _lib.QRB200_OK
    return n.value


# ---------------------------------------------------------------------- workspaces

def test_workspace_sizes_allow_for_any_start():
    """The buffers are used from the first byte on 16, so a size holds 15 bytes more than they do."""
    # 40 rows of 8 bf16 elements, 9 apart: a copy of 40 * 16 bytes, rounded up to 768
    assert size_of("qrb200_linear_workspace_bytes", 16, 9, 16, 8, 0, 40, 4, 8, 1) == 768 + 15
    # without a copy nothing is needed at all
    assert size_of("qrb200_linear_workspace_bytes", 16, 8, 16, 8, 0, 40, 4, 8, 1) == 0
    assert size_of("qrb200_linear_backward_workspace_bytes", 16, 9, 0, 16, 8, 16, 8, 0, 1, 0, 0, 40, 8, 8) == 768 + 15
    # short rows share a block, and a block leaves one row of partial sums
    assert size_of("qrb200_rms_norm_backward_workspace_bytes", 2, 8, 0, 0) == 8 * 4 + 15


@pytest.mark.parametrize("start", [17, 18, 24, 31])
def test_workspace_off_16_bytes_has_to_be_larger(start):
    """What the start wastes is not counted as room: such a workspace was used as it stood, for 16-byte stores."""
    L, skip = _lib.lib(), -start % 16
    linear = lambda size: L.qrb200_linear(16, 9, 16, 8, 0, None, None, None, None, 0, 16, 4, None, 40, 4, 8, 1, 1, 0,  # noqa: E731
                                          start, size, None)
    back = lambda size: L.qrb200_linear_backward(16, 9, None, 16, 8, 16, 8, 0, 16, None, None, 40, 8, 8, 1, start, size, None)  # noqa: E731
    for size in (0, 767, 768, 768 + skip - 1):
        assert linear(size) == _lib.QRB200_ERR_WORKSPACE
        assert back(size) == _lib.QRB200_ERR_WORKSPACE
    for size in (0, 31, 32, 32 + skip - 1):
        assert L.qrb200_rms_norm_backward(16, 8, 16, 8, None, 8, 16, 0, 16, None, 16, 2, 8, 1e-6, 0, 0, start, size,
                                          None) == _lib.QRB200_ERR_WORKSPACE


# ---------------------------------------------------------------------- sizes

def test_sums_too_long_for_int_indices_are_refused():
    """Kernels step past k by up to 32768 elements: their int index must not pass 2^31 on the way."""
    L, n, most = _lib.lib(), ctypes.c_size_t(), 2 ** 31 - 65537
    size = lambda k, t: L.qrb200_linear_workspace_bytes(16, k, 16, k, 0, 1, 1, k, t, ctypes.byref(n))  # noqa: E731
    for t in (_lib.QRB200_BF16, _lib.QRB200_E4M3):
        assert size(most, t) == _lib.QRB200_OK
        for k in (most + 1, 2 ** 31 - 32768, 2 ** 31 - 257, 2 ** 31):
            assert size(k, t) == _lib.QRB200_ERR_INVALID_ARG
            assert L.qrb200_linear(16, k, 16, k, 0, None, None, None, None, 0, 16, 1, None, 1, 1, k, t, _lib.QRB200_BF16, 0, None, 0,
                                   None) == _lib.QRB200_ERR_INVALID_ARG
