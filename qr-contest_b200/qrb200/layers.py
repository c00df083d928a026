"""Layer operators: what is done with an orthogonal factor once it is a weight.

:func:`rms_norm` -- root-mean-square norm of rows with the residual's addition, its output in the
input's type or in 8 bits (e4m3) with a scale a row; :func:`linear` -- matrix product with bias,
activation and residual in its epilogue, on 16-bit operands or on 8-bit ones with scales;
:func:`quantize_rows` -- lays a weight out in 8 bits once.  A root-mean-square norm commutes with an
orthogonal ``Q`` (:func:`qrb200.geqrf_q`), which is why activations can be rotated before they are
held in 8 bits.

All take CUDA tensors, run on the current stream without synchronising, and raise ``TypeError`` or
``ValueError`` on arguments they do not take.  Leading dimensions are free; rows may be slices or
expanded views (one row stride: read in place, anything else is copied first).  ``rms_norm`` and
``linear`` are differentiable once in every floating input where all types are 16 bits or more (the
operators' own autograd formulas, in C++), in reverse mode: a second derivative, a forward-mode one or one of an
8-bit output is refused, not dropped.  The same inputs give the same bits.
"""
from __future__ import annotations

import torch

from . import _lib, api

_ACTIVATIONS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
                "gelu_tanh": _lib.ACT_GELU_TANH, "silu": _lib.ACT_SILU}
_FP8 = torch.float8_e4m3fn


class _Ops:
    """The operators' handles, looked up once; ``fast_*`` take plain CUDA tensors without the operator
    registry and return NotImplemented for anything else."""

    loaded = False

    @classmethod
    def load(cls):
        api.load_torch_ops()
        ns = torch.ops.qrb200
        cls.rms_norm = ns.rms_norm.default
        cls.rms_norm_backward = ns.rms_norm_backward.default
        cls.quantize_rows = ns.quantize_rows.default
        cls.linear = ns.linear.default
        cls.linear_backward = ns.linear_backward.default
        from . import _layers
        cls.fast_rms_norm = staticmethod(_layers.rms_norm)
        cls.fast_linear = staticmethod(_layers.linear)
        cls.loaded = True


def _load():
    _Ops.load()


_load._dynamo_marked_constant = True  # run, not traced, where the first call is in a compiled program


def _check(what, optional=(), eps=0.0, out_dtype=None):
    """Kinds of arguments that the registry would refuse with a RuntimeError."""
    for name, t in what:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"qrb200: {name} must be a tensor, got {type(t).__name__}")
    for name, t in optional:
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"qrb200: {name} must be a tensor or None, got {type(t).__name__}")
    if not isinstance(eps, (float, int)) and not hasattr(eps, "__float__"):
        raise TypeError(f"qrb200: eps must be a number, got {type(eps).__name__}")
    if out_dtype is not None and not isinstance(out_dtype, torch.dtype):
        raise TypeError(f"qrb200: out_dtype must be a torch.dtype or None, got {type(out_dtype).__name__}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
             eps: float = 1e-6, out_dtype: torch.dtype | None = None):
    """``h = x + residual``; ``y = h * (mean(h**2, -1) + eps)**-0.5 * weight``.

    ``x`` is ``(..., d)`` in float32, bfloat16 or float16; ``weight`` ``(d,)`` in x's type or float32;
    ``residual`` in x's shape, in x's type or float32.  ``h`` is rounded to the residual's type (it is the
    stream that later layers read) and ``y`` is the norm of that.  Returns ``y``, or ``(y, h)`` with a
    residual.  With ``out_dtype=torch.float8_e4m3fn`` it returns ``(y, scale)`` or ``(y, scale, h)``:
    ``scale`` is float32, one a row, ``max(max|y| / 448, 2**-126)``, and ``y * scale[..., None]`` the value.
    """
    if not _Ops.loaded:
        _load()
    if not torch.compiler.is_compiling():
        got = _Ops.fast_rms_norm(x, weight, residual, eps, out_dtype)
        if got is not NotImplemented:
            return got
    _check((("x", x),), (("weight", weight), ("residual", residual)), eps, out_dtype)
    y, scale, h = _Ops.rms_norm(x, weight, residual, eps, out_dtype)
    if scale is None:
        return y if h is None else (y, h)
    return (y, scale) if h is None else (y, scale, h)


def quantize_rows(x: torch.Tensor):
    """Rows of ``x`` (``(..., d)``; float32, bfloat16, float16) in e4m3 with a float32 scale each, by
    :func:`rms_norm`'s rule: returns ``(q, scale)``.  For a weight ``(n, k)`` that is one scale per
    output feature."""
    if not _Ops.loaded:
        _load()
    _check((("x", x),))
    return _Ops.quantize_rows(x)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           activation: str | None = None, residual: torch.Tensor | None = None,
           x_scale: torch.Tensor | None = None, weight_scale: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    ``x`` is ``(..., k)`` and ``weight`` ``(n, k)``, both bfloat16, float16 or float8_e4m3fn (a transposed view is
    read in place for 16-bit types); ``bias`` ``(n,)`` and ``residual`` ``(..., n)`` are in the output's type, which is
    x's, or bfloat16 (default) or float16 for 8-bit operands.  ``activation``: None, ``"relu"``, ``"gelu"``,
    ``"gelu_tanh"``, ``"silu"``.  8-bit operands are multiplied by ``x_scale`` (one float32, or one a row of x) and
    ``weight_scale`` (one, or one an output feature).  Sums are float32; the result is rounded once.
    """
    if not _Ops.loaded:
        _load()
    try:
        act = _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"qrb200: unknown activation {activation!r}") from None
    if not torch.compiler.is_compiling():
        got = _Ops.fast_linear(x, weight, bias, residual, act, x_scale, weight_scale, out_dtype)
        if got is not NotImplemented:
            return got
    _check((("x", x), ("weight", weight)), (("bias", bias), ("residual", residual), ("x_scale", x_scale),
                                            ("weight_scale", weight_scale)), out_dtype=out_dtype)
    return _Ops.linear(x, weight, bias, residual, act, x_scale, weight_scale, out_dtype, False)[0]
