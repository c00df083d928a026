"""CPU: the layer operators' refusals and output shapes (nothing here reaches a GPU), and the layer
C ABI's checks of its arguments, each of which returns before any CUDA call."""
import ctypes

import pytest
import torch

import qrb200
from qrb200 import _lib

FP8 = torch.float8_e4m3fn
BF = torch.bfloat16


def meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_host_tensors_are_refused():
    for call in (lambda: qrb200.rms_norm(torch.ones(2, 8)), lambda: qrb200.quantize_rows(torch.ones(2, 8)),
                 lambda: qrb200.linear(torch.ones(2, 8, dtype=BF), torch.ones(4, 8, dtype=BF))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_rms_norm_shapes():
    x, w = meta(2, 3, 40), meta(40, dtype=torch.float32)
    y = qrb200.rms_norm(x, w)
    assert y.shape == x.shape and y.dtype == BF
    y, h = qrb200.rms_norm(x, w, residual=meta(2, 3, 40, dtype=torch.float32))
    assert y.dtype == BF and h.dtype == torch.float32 and h.shape == x.shape
    q, s, h = qrb200.rms_norm(x, residual=meta(2, 3, 40), out_dtype=FP8)
    assert q.dtype == FP8 and q.shape == x.shape and s.shape == (2, 3) and s.dtype == torch.float32 and h.dtype == BF
    q, s = qrb200.quantize_rows(meta(5, 7, dtype=torch.float32))
    assert q.shape == (5, 7) and s.shape == (5,)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: qrb200.rms_norm(meta(2, 8, dtype=torch.float64))),
    (TypeError, lambda: qrb200.rms_norm(meta(2, 8, dtype=torch.int32))),
    (TypeError, lambda: qrb200.rms_norm(meta(2, 8), meta(8, dtype=torch.float16))),
    (TypeError, lambda: qrb200.rms_norm(meta(2, 8), residual=meta(2, 8, dtype=torch.float16))),
    (TypeError, lambda: qrb200.rms_norm(meta(2, 8), out_dtype=torch.float32)),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8), meta(7))),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8), meta(1, 8))),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8), residual=meta(1, 8))),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8), eps=-1.0)),
    (ValueError, lambda: qrb200.rms_norm(torch.empty((), dtype=BF, device="meta"))),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8), torch.ones(8, dtype=BF))),
    (ValueError, lambda: qrb200.rms_norm(meta(2, 8).requires_grad_(), out_dtype=FP8)),
    (TypeError, lambda: qrb200.quantize_rows(meta(2, 8, dtype=FP8))),
    (TypeError, lambda: qrb200.linear(meta(2, 8, dtype=torch.float32), meta(4, 8, dtype=torch.float32))),
    (TypeError, lambda: qrb200.linear(meta(2, 8), meta(4, 8, dtype=torch.float16))),
    (TypeError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), meta(4, dtype=torch.float32))),
    (TypeError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), residual=meta(2, 4, dtype=torch.float16))),
    (TypeError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), out_dtype=torch.float32)),
    (TypeError, lambda: qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), out_dtype=torch.float32)),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 7))),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(8))),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), meta(8))),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), residual=meta(1, 4))),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), activation="tanh")),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), activation=["relu"])),
    (ValueError, lambda: qrb200.linear(meta(2, 8), meta(4, 8), x_scale=meta(2, dtype=torch.float32))),
    (ValueError, lambda: qrb200.linear(meta(2, 8).requires_grad_(), meta(4, 8), x_scale=meta(2, dtype=torch.float32))),
    (ValueError, lambda: qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), x_scale=meta(3, dtype=torch.float32))),
    (TypeError, lambda: qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), weight_scale=meta(4))),
    (ValueError, lambda: qrb200.linear(meta(2, 8, dtype=FP8), meta(4, 8, dtype=FP8), meta(4).requires_grad_())),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call()


def test_linear_shapes():
    assert qrb200.linear(meta(8), meta(4, 8)).shape == (4,)
    y = qrb200.linear(meta(2, 3, 8, dtype=FP8), meta(4, 8, dtype=FP8), x_scale=meta(2, 3, dtype=torch.float32),
                      weight_scale=meta(1, dtype=torch.float32), out_dtype=torch.float16)
    assert y.shape == (2, 3, 4) and y.dtype == torch.float16


def _norm(**kw):
    a = dict(x=16, ldx=8, w=None, wt=0, r=None, ldr=8, st=0, y=16, s=None, h=None, rows=2, dim=8, eps=0.0, t=1, ot=1)
    a.update(kw)
    return _lib.lib().qrb200_rms_norm(a["x"], a["ldx"], a["w"], a["wt"], a["r"], a["ldr"], a["st"], a["y"], a["s"], a["h"],
                                      a["rows"], a["dim"], a["eps"], a["t"], a["ot"], None)


def test_norm_abi_checks():
    bad = _lib.QRB200_ERR_INVALID_ARG
    for kw in (dict(t=3), dict(t=9), dict(ot=0), dict(rows=-1), dict(dim=-1), dict(eps=-1.0), dict(eps=float("nan")),
               dict(x=None), dict(y=None), dict(ot=3), dict(w=16, wt=2), dict(r=16, st=2, h=16), dict(r=16, st=1),
               dict(rows=1 << 31), dict(dim=1 << 30), dict(ldx=-1)):
        assert _norm(**kw) == bad, kw
    assert _norm(rows=0, x=None, y=None) == _lib.QRB200_OK
    assert _norm(dim=0, x=None, y=None) == _lib.QRB200_OK
    L = _lib.lib()
    assert L.qrb200_quantize_rows(16, 8, 16, None, 2, 8, 0, None) == bad
    assert L.qrb200_quantize_rows(16, 8, 16, 16, 2, 8, 3, None) == bad
    assert L.qrb200_quantize_rows(None, 8, None, None, 0, 8, 0, None) == _lib.QRB200_OK
    n = ctypes.c_size_t()
    assert L.qrb200_rms_norm_backward_workspace_bytes(4, 8, 0, 0, None) == bad
    assert L.qrb200_rms_norm_backward_workspace_bytes(4, 8, 0, 0, ctypes.byref(n)) == _lib.QRB200_OK and n.value >= 32
    back = lambda **k: L.qrb200_rms_norm_backward(  # noqa: E731
        k.get("dy", 16), 8, k.get("h", 16), 8, None, 8, k.get("w", 16), k.get("wt", 0), 16, None, 16, k.get("rows", 2), 8, 1e-6,
        k.get("t", 0), k.get("st", 0), k.get("ws"), k.get("wsb", 0), None)
    for kw in (dict(t=3), dict(st=1), dict(wt=1), dict(w=None), dict(dy=None), dict(h=None), dict(rows=-1)):
        assert back(**kw) == bad, kw
    assert back(ws=16, wsb=1) == _lib.QRB200_ERR_WORKSPACE


def _linear(**kw):
    a = dict(x=16, ldx=8, w=16, ldw=8, tr=0, y=16, ldy=4, r=None, ldr=4, slope=None, m=2, n=4, k=8, t=1, ot=1, act=0, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().qrb200_linear(a["x"], a["ldx"], a["w"], a["ldw"], a["tr"], None, None, None, a["r"], a["ldr"], a["y"], a["ldy"],
                                    a["slope"], a["m"], a["n"], a["k"], a["t"], a["ot"], a["act"], a["ws"], a["wsb"], None)


def test_linear_abi_checks():
    bad = _lib.QRB200_ERR_INVALID_ARG
    for kw in (dict(t=0), dict(t=7), dict(ot=2), dict(t=3, ot=0), dict(t=3, ot=1, tr=1), dict(t=3, ot=1, slope=16), dict(act=5),
               dict(act=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(m=1 << 31), dict(x=None), dict(w=None), dict(y=None),
               dict(ldx=7), dict(ldw=7), dict(ldy=3), dict(tr=1, ldw=3), dict(r=16, ldr=-1)):
        assert _linear(**kw) == bad, kw
    # odd rows need an aligned copy, and the caller's workspace has to hold it
    assert _linear(m=40, ldx=9, ws=16, wsb=16) == _lib.QRB200_ERR_WORKSPACE
    assert _linear(m=0, x=None, w=None, y=None) == _lib.QRB200_OK
    assert _linear(n=0, ldy=0, x=None, w=None, y=None) == _lib.QRB200_OK
    L, n = _lib.lib(), ctypes.c_size_t()
    size = lambda ldx, k: (L.qrb200_linear_workspace_bytes(16, ldx, 16, 16, 0, 2, 4, k, 1, ctypes.byref(n)), n.value)  # noqa: E731
    assert size(16, 16) == (_lib.QRB200_OK, 0)
    assert size(17, 16)[1] >= 2 * 16 * 2
    assert L.qrb200_linear_workspace_bytes(16, 8, 16, 8, 0, 2, 4, 8, 0, ctypes.byref(n)) == bad
    back = lambda **k: L.qrb200_linear_backward(  # noqa: E731
        k.get("dy", 16), k.get("lddy", 8), None, k.get("x", 16), 8, k.get("w", 16), 8, 0, 16, 16, None, 2, k.get("n", 8), 8, k.get("t", 1),
        k.get("ws"), k.get("wsb", 0), None)
    for kw in (dict(t=0), dict(t=3), dict(dy=None), dict(x=None), dict(w=None), dict(lddy=7), dict(n=-1)):
        assert back(**kw) == bad, kw
    assert back(lddy=9, ws=16, wsb=16) == _lib.QRB200_ERR_WORKSPACE
    assert L.qrb200_layer_status(None) == bad
