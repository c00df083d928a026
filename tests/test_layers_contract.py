"""CPU: what the layer operators promise about workspaces, sizes, dispatch and derivatives; nothing here
reaches a GPU (calls of the C ABI return before any CUDA call)."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import qrb200
from qrb200 import _lib

FP8 = torch.float8_e4m3fn
BF = torch.bfloat16


def meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


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


# ---------------------------------------------------------------------- what listens below autograd

class Seen(torch.utils._python_dispatch.TorchDispatchMode):
    """Records the layer operators that reach a dispatch mode."""

    def __init__(self):
        super().__init__()
        self.ops = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "qrb200":
            self.ops.append(func._opname)
        return func(*args, **(kwargs or {}))


def test_dispatch_modes_see_the_operators():
    with Seen() as seen:
        qrb200.rms_norm(meta(2, 8))
        qrb200.rms_norm(meta(2, 8), residual=meta(2, 8), out_dtype=FP8)
        qrb200.linear(meta(2, 8), meta(4, 8), activation="gelu")
        qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), x_scale=meta(2, dtype=torch.float32))
    assert seen.ops == ["rms_norm", "rms_norm", "linear", "linear"]


def test_dispatch_modes_see_the_gradients():
    x, w = meta(2, 8).requires_grad_(), meta(4, 8).requires_grad_()
    with Seen() as seen:
        y, h = qrb200.rms_norm(x, residual=meta(2, 8))
        dx, dw = torch.autograd.grad(qrb200.linear(y, w, activation="silu").sum() + h.sum(), (x, w))
    assert seen.ops == ["rms_norm", "linear", "linear_backward", "rms_norm_backward"]
    assert dx.shape == x.shape and dw.shape == w.shape


def test_fake_tensors_of_a_gpu():
    """Shapes without the GPU: nothing is allocated there."""
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        x, w = (torch.empty(*s, dtype=BF, device="cuda") for s in ((2, 3, 8), (4, 8)))
        y, h = qrb200.rms_norm(x, residual=x.float())
        z = qrb200.linear(y, w, activation="gelu")
        q8, s, h8 = qrb200.rms_norm(x, residual=x, out_dtype=FP8)
    assert z.shape == (2, 3, 4) and z.dtype == BF and z.device.type == "cuda" and h.dtype == torch.float32
    assert q8.shape == (2, 3, 8) and q8.dtype == FP8 and s.shape == (2, 3) and h8.dtype == BF


def called(graph):
    return [n.target._opname for n in graph.nodes if getattr(n.target, "namespace", "") == "qrb200"]


def test_a_trace_holds_the_operators():
    from torch.fx.experimental.proxy_tensor import make_fx

    def forward(x, w):
        return qrb200.linear(qrb200.rms_norm(x), w, activation="silu")

    def gradients(x, w):
        return torch.autograd.grad(forward(x, w).sum(), (x, w))
    assert called(make_fx(forward)(meta(2, 8), meta(4, 8)).graph) == ["rms_norm", "linear"]
    assert called(make_fx(gradients)(meta(2, 8).requires_grad_(), meta(4, 8).requires_grad_()).graph) == [
        "rms_norm", "linear", "linear_backward", "rms_norm_backward"]


def test_exported_and_compiled_programs_hold_the_operators():
    class Block(torch.nn.Module):
        def forward(self, x, w):
            return qrb200.linear(qrb200.rms_norm(x), w, activation="silu")
    qrb200.rms_norm(meta(2, 8))
    assert called(torch.export.export(Block(), (meta(2, 8), meta(4, 8))).graph) == ["rms_norm", "linear"]
    graphs = []

    def keep(gm, inputs):
        graphs.append(called(gm.graph))
        return gm.forward
    from torch._dynamo.backends.common import aot_autograd
    torch._dynamo.reset()
    step = torch.compile(Block(), backend=aot_autograd(fw_compiler=keep), fullgraph=True, dynamic=True)
    for rows in (2, 5):
        x, w = meta(rows, 8).requires_grad_(), meta(4, 8).requires_grad_()
        dx, dw = torch.autograd.grad(step(x, w).sum(), (x, w))
        assert dx.shape == x.shape and dw.shape == w.shape
    assert graphs[:2] == [["rms_norm", "linear"], ["linear_backward", "rms_norm_backward"]]


def test_the_slope_comes_with_gradients():
    """linear's want_slope is for linear_backward: without the slope that takes the activation for the identity."""
    qrb200.api.load_torch_ops()
    x, w = meta(2, 8).requires_grad_(), meta(4, 8)
    y, slope = torch.ops.qrb200.linear(x, w, None, None, _lib.ACT_SILU, None, None, None, True)
    assert y.requires_grad and slope is not None and slope.shape == (2, 4) and slope.dtype == torch.int16 and not slope.requires_grad
    # asked for, it is there without an activation as well, as it is without gradients
    for grad in (False, True):
        x = meta(2, 8).requires_grad_(grad)
        assert torch.ops.qrb200.linear(x, w, None, None, _lib.ACT_NONE, None, None, None, True)[1] is not None
        assert torch.ops.qrb200.linear(x, w, None, None, _lib.ACT_SILU, None, None, None, False)[1] is None


def test_the_first_call_may_be_a_compiled_one():
    """The libraries are loaded while a whole-program graph is traced; in a process of its own, where nothing has been."""
    code = """if True:
        import torch, qrb200
        x, w = (torch.empty(*s, dtype=torch.bfloat16, device="meta") for s in ((2, 8), (4, 8)))
        step = torch.compile(lambda x, w: qrb200.quantize_rows(qrb200.linear(qrb200.rms_norm(x), w))[1], backend="aot_eager", fullgraph=True)
        assert step(x, w).shape == (2,)
        """
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(qrb200.__file__).resolve().parents[1], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


def test_outputs_share_no_memory():
    """The residual's gradient is dx itself where the types are the same: the operator returns it once, because what
    compiles a program may write over one output while it still needs the other."""
    qrb200.api.load_torch_ops()
    op = torch.ops.qrb200.rms_norm_backward
    for want_dx in (False, True):
        dx, dres, dw = op(meta(2, 8), meta(2, 8), None, meta(8), 1e-6, want_dx, True, True)
        assert dx.shape == (2, 8) and dres is None and dw.shape == (8,)
        dx, dres, _ = op(meta(2, 8), meta(2, 8, dtype=torch.float32), None, meta(8), 1e-6, want_dx, True, True)
        assert (dx is not None) == want_dx and dres.dtype == torch.float32
    x, r = meta(2, 8).requires_grad_(), meta(2, 8).requires_grad_()
    y, h = qrb200.rms_norm(x, residual=r)
    dx, dr = torch.autograd.grad(y.sum() + h.sum(), (x, r))
    assert dx.shape == dr.shape == (2, 8)
    y, h = qrb200.rms_norm(meta(2, 8), residual=r)
    assert torch.autograd.grad(y.sum(), r)[0].shape == (2, 8)


# ---------------------------------------------------------------------- derivatives there are not

def tangents(call, *shapes, dual):
    """call() on tensors of these shapes, the one at `dual` with a tangent."""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        ts = [meta(*s) if isinstance(s, tuple) else s for s in shapes]
        ts[dual] = fw.make_dual(ts[dual], torch.empty_like(ts[dual]))
        return call(*ts)


F32_4 = meta(4, dtype=torch.float32)


@pytest.mark.parametrize("call", [
    lambda: tangents(lambda x: qrb200.rms_norm(x), (2, 8), dual=0),
    lambda: tangents(lambda x: qrb200.rms_norm(x, out_dtype=FP8), (2, 8), dual=0),
    lambda: tangents(lambda x, w: qrb200.rms_norm(x, w), (2, 8), (8,), dual=1),
    lambda: tangents(lambda x, r: qrb200.rms_norm(x, residual=r), (2, 8), (2, 8), dual=1),
    lambda: tangents(lambda x, w: qrb200.linear(x, w), (2, 8), (4, 8), dual=0),
    lambda: tangents(lambda x, w: qrb200.linear(x, w, activation="gelu"), (2, 8), (4, 8), dual=1),
    lambda: tangents(lambda x, w, b: qrb200.linear(x, w, b), (2, 8), (4, 8), (4,), dual=2),
    lambda: tangents(lambda x, w, r: qrb200.linear(x, w, residual=r), (2, 8), (4, 8), (2, 4), dual=2),
    lambda: tangents(lambda x, w, s: qrb200.linear(x, w, weight_scale=s), meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), F32_4, dual=2),
    lambda: tangents(lambda x: qrb200.quantize_rows(x), (2, 8), dual=0),
    lambda: tangents(lambda x, w: qrb200.linear(x.requires_grad_(), w), (2, 8), (4, 8), dual=1),
    lambda: torch.func.jvp(lambda x: qrb200.linear(x, meta(4, 8)), (meta(2, 8),), (meta(2, 8),)),
    lambda: torch.func.jvp(lambda x: qrb200.rms_norm(x), (meta(2, 8),), (meta(2, 8),)),
])
def test_forward_mode_is_refused(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call", [lambda x: qrb200.rms_norm(x), lambda x: qrb200.linear(x, meta(8, 8), activation="silu")])
def test_forward_over_reverse_is_refused(call):
    """A tangent of the gradient that comes in is not dropped on the way back either."""
    import torch.autograd.forward_ad as fw
    x = meta(2, 8).requires_grad_()
    y = call(x)
    with fw.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(y, x, fw.make_dual(torch.empty_like(y), torch.empty_like(y)))


def test_gradients_of_8_bits_are_refused():
    w = meta(4, 8).requires_grad_()
    w8, scale = qrb200.quantize_rows(w)
    with pytest.raises(RuntimeError, match="not implemented"):
        scale.sum().backward()
    # quantizing what requires a gradient is fine where none is asked for
    with torch.no_grad():
        w8, scale = qrb200.quantize_rows(w)
    assert not scale.requires_grad and qrb200.linear(meta(2, 8, dtype=FP8), w8, weight_scale=scale).shape == (2, 4)


# ---------------------------------------------------------------------- arguments of the wrong kind

@pytest.mark.parametrize("call", [
    lambda: qrb200.rms_norm([1.0, 2.0]),
    lambda: qrb200.rms_norm(None),
    lambda: qrb200.rms_norm(meta(2, 8), weight=1.0),
    lambda: qrb200.rms_norm(meta(2, 8), residual=[0.0]),
    lambda: qrb200.rms_norm(meta(2, 8), eps="1e-6"),
    lambda: qrb200.rms_norm(meta(2, 8), eps=None),
    lambda: qrb200.rms_norm(meta(2, 8), out_dtype="bf16"),
    lambda: qrb200.quantize_rows([1.0, 2.0]),
    lambda: qrb200.quantize_rows(None),
    lambda: qrb200.linear(meta(2, 8), None),
    lambda: qrb200.linear(None, meta(4, 8)),
    lambda: qrb200.linear(meta(2, 8), meta(4, 8), 1.0),
    lambda: qrb200.linear(meta(2, 8), meta(4, 8), residual=0),
    lambda: qrb200.linear(meta(2, 8), meta(4, 8), out_dtype="bf16"),
    lambda: qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), x_scale=0.5),
])
def test_arguments_of_another_kind(call):
    """TypeError, as the documentation says, and not the operator registry's RuntimeError."""
    with pytest.raises(TypeError):
        call()


# ---------------------------------------------------------------------- scales

@pytest.mark.parametrize("m", [1, 2, 40, 3000])
def test_scales_of_16_bit_operands_are_refused(m):
    """From C as from Python: one kernel multiplied by them and the others did not."""
    L, bad = _lib.lib(), _lib.QRB200_ERR_INVALID_ARG
    for t in (_lib.QRB200_BF16, _lib.QRB200_F16):
        for xs, ws in ((16, None), (None, 16), (16, 16)):
            assert L.qrb200_linear(16, 8, 16, 8, 0, xs, ws, None, None, 0, 16, 4, None, m, 4, 8, t, t, 0, None, 0, None) == bad
    with pytest.raises(ValueError):
        qrb200.linear(meta(m, 8), meta(4, 8), weight_scale=F32_4)
