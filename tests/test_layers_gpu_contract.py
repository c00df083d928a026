"""GPU: what the layer operators promise about workspaces, streams, waits and the ends of their ranges.

Bounds are derived beside each test; u is the unit roundoff of a type (2^-8 bf16, 2^-11 f16, 2^-24 f32)."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _give_memory_back():
    """No bounded wait ran out in here; leaves no cached blocks behind."""
    yield
    from qrb200 import _lib
    assert not _lib.layer_timed_out()
    torch.cuda.empty_cache()


def q():
    import qrb200
    return qrb200


def rnd(*shape, dtype=F32, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * gain).to(dtype)


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------------- workspaces

class Workspace:
    """`size` bytes that start `off` bytes past a 256-byte boundary, in front of and behind bytes of 0xA5."""

    def __init__(self, size, off):
        self.all = torch.full((size + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
        assert self.all.data_ptr() % 256 == 0
        self.first, self.size, self.ptr = 256 + off, size, self.all.data_ptr() + 256 + off

    def untouched(self):
        return bool((self.all[:self.first] == 0xA5).all()) and bool((self.all[self.first + self.size:] == 0xA5).all())


@pytest.mark.parametrize("off", [0, 1, 2, 4, 8, 15])
def test_workspace_starts_anywhere(off):
    """Same bits as with a workspace of torch's, and nothing written outside it."""
    from qrb200 import _lib
    L, n = _lib.lib(), ctypes.c_size_t()
    ok = _lib.QRB200_OK
    # a product whose operands are both copied
    x, w = rnd(40, 37, dtype=BF, seed=1), rnd(50, 37, dtype=BF, seed=2)
    want = q().linear(x, w)
    y = torch.empty_like(want)
    assert L.qrb200_linear_workspace_bytes(x.data_ptr(), 37, w.data_ptr(), 37, 0, 40, 50, 37, 1, ctypes.byref(n)) == ok
    ws = Workspace(n.value, off)
    assert L.qrb200_linear(x.data_ptr(), 37, w.data_ptr(), 37, 0, None, None, None, None, 0, y.data_ptr(), 50, None, 40, 50, 37, 1, 1, 0,
                           ws.ptr, ws.size, stream()) == ok
    assert torch.equal(y, want) and ws.untouched()
    # its gradients, with dz, partial sums and copies in the workspace
    dy = rnd(40, 50, dtype=BF, seed=3)
    slope = torch.ops.qrb200.linear(x, w, None, None, _lib.ACT_SILU, None, None, None, True)[1]
    want = torch.ops.qrb200.linear_backward(dy, slope, x, w, True, True, True)
    got = [torch.empty_like(t) for t in want]
    assert L.qrb200_linear_backward_workspace_bytes(dy.data_ptr(), 50, 1, x.data_ptr(), 37, w.data_ptr(), 37, 0, 1, 1, 1, 40, 50, 37,
                                                    ctypes.byref(n)) == ok
    ws = Workspace(n.value, off)
    assert L.qrb200_linear_backward(dy.data_ptr(), 50, slope.data_ptr(), x.data_ptr(), 37, w.data_ptr(), 37, 0, *(t.data_ptr() for t in got),
                                    40, 50, 37, 1, ws.ptr, ws.size, stream()) == ok
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and ws.untouched()
    # the norm's gradients, by vectors and by single elements
    for dim in (64, 65):
        h, dy, w = rnd(300, dim, seed=4), rnd(300, dim, seed=5), rnd(dim, seed=6)
        want = torch.ops.qrb200.rms_norm_backward(dy, h, None, w, 1e-6, True, False, True)
        dx, dw = torch.empty_like(h), torch.empty_like(w)
        assert L.qrb200_rms_norm_backward_workspace_bytes(300, dim, 0, 0, ctypes.byref(n)) == ok
        ws = Workspace(n.value, off)
        assert L.qrb200_rms_norm_backward(dy.data_ptr(), dim, h.data_ptr(), dim, None, 0, w.data_ptr(), 0, dx.data_ptr(), None,
                                          dw.data_ptr(), 300, dim, 1e-6, 0, 0, ws.ptr, ws.size, stream()) == ok
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[2]) and ws.untouched()


# ---------------------------------------------------------------------- what listens below autograd

def test_a_trace_answers_for_its_own_inputs():
    """A traced or compiled step gives on other inputs what the operators give there, to the bit."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def forward(x, w):
        return q().linear(q().rms_norm(x), w, activation="silu")

    def step(x, w):
        return torch.autograd.grad(forward(x, w).sum(), (x, w))
    first = rnd(33, 64, dtype=BF, seed=1), rnd(40, 64, dtype=BF, seed=2)
    other = rnd(33, 64, dtype=BF, seed=3), rnd(40, 64, dtype=BF, seed=4)
    assert torch.equal(make_fx(forward)(*first)(*other), forward(*other))
    first, other = ([t.requires_grad_() for t in ts] for ts in (first, other))
    want = step(*other)
    assert all(torch.equal(a, b) for a, b in zip(make_fx(step)(*first)(*(t.detach() for t in other)), want))
    torch._dynamo.reset()
    compiled = torch.compile(forward, backend="aot_eager", fullgraph=True)
    for x, w in (first, other):
        y = compiled(x, w)
        assert torch.equal(y, forward(x, w))
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), (x, w)), step(x, w)))


def test_the_slope_comes_with_gradients():
    """The operator's slope is the same with and without something to differentiate, and so are the gradients made
    from it: a traced step may be run on tensors that require gradients."""
    from qrb200 import _lib
    x, w, dy = rnd(33, 64, dtype=BF, seed=1), rnd(40, 64, dtype=BF, seed=2), rnd(33, 40, dtype=BF, seed=3)
    op = torch.ops.qrb200.linear
    for act in (_lib.ACT_NONE, _lib.ACT_SILU):
        y, slope = op(x, w, None, None, act, None, None, None, True)
        xg = x.clone().requires_grad_()
        yg, slope_g = op(xg, w, None, None, act, None, None, None, True)
        assert torch.equal(y, yg) and torch.equal(slope, slope_g)
        dx, = torch.autograd.grad(yg, xg, dy)
        assert torch.equal(dx, torch.ops.qrb200.linear_backward(dy, slope_g, x, w, True, False, False)[0])


def test_forward_mode_is_refused():
    """On the short way from Python too."""
    import torch.autograd.forward_ad as fw
    x, w = rnd(5, 64, dtype=BF, seed=1), rnd(40, 64, dtype=BF, seed=2)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        for call in (lambda: q().rms_norm(d), lambda: q().linear(d, w), lambda: q().rms_norm(x, residual=d, out_dtype=FP8),
                     lambda: q().quantize_rows(d)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(q().linear(x, w), q().linear(x.clone(), w))


# ---------------------------------------------------------------------- waits

def test_status_waits_for_every_stream():
    """Torch's side streams do not block the default one, and what still runs there has not reported yet."""
    from qrb200 import _lib
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    _lib.layer_timed_out()  # whatever a first call takes longer for
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # cycles: 0.1 s
        done.record()
    assert not _lib.layer_timed_out()
    assert done.query()


# ---------------------------------------------------------------------- contexts

IN_TWO_CONTEXTS = """if True:
    # each kernel that asks for more than 48 KB of shared memory, before and after the context is made again
    import ctypes, numpy, torch
    from qrb200 import _lib
    L, rt = _lib.lib(), ctypes.CDLL("libcudart.so.12")
    rng = numpy.random.default_rng(1)

    def check(rc):
        assert rc == 0, (rc, L.qrb200_last_cuda_error())

    def bf16(*shape):
        return (rng.standard_normal(shape, numpy.float32).view(numpy.uint32) >> 16).astype(numpy.uint16)

    class Array:
        def __init__(self, host):
            self.host, self.p = host, ctypes.c_void_p()
            check(rt.cudaMalloc(ctypes.byref(self.p), ctypes.c_size_t(host.nbytes)))
            check(rt.cudaMemcpy(self.p, host.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(host.nbytes), 1))

        def back(self):
            check(rt.cudaDeviceSynchronize())
            out = numpy.empty_like(self.host)
            check(rt.cudaMemcpy(out.ctypes.data_as(ctypes.c_void_p), self.p, ctypes.c_size_t(out.nbytes), 2))
            return out
    m, n, k = 300, 256, 256
    hosts = [bf16(m, k), bf16(n, k), bf16(k), bf16(5000, k), bf16(4096, k)]

    def run():
        x, w, gain, many, wide = map(Array, hosts)
        y, u, dx, dw = (Array(numpy.zeros(s, numpy.uint16)) for s in ((m, n), (5000, 4096), (m, k), (k,)))
        check(L.qrb200_linear(x.p, k, w.p, k, 0, None, None, None, None, 0, y.p, n, None, m, n, k, 1, 1, 0, None, 0, None))
        check(L.qrb200_linear(many.p, k, wide.p, k, 0, None, None, None, None, 0, u.p, 4096, None, 5000, 4096, k, 1, 1, 0, None, 0, None))
        check(L.qrb200_rms_norm_backward(x.p, k, x.p, k, None, 0, gain.p, 1, dx.p, None, dw.p, m, k, 1e-6, 1, 1, None, 0, None))
        return [t.back() for t in (y, u, dx, dw)]
    first = run()
    check(rt.cudaDeviceReset())
    second = run()
    assert all(numpy.array_equal(a, b) and a.any() for a, b in zip(first, second))
    """


def test_a_context_that_is_made_again():
    """In a process of its own: what the library remembers of a context goes with it."""
    import subprocess
    import sys
    from pathlib import Path
    done = subprocess.run([sys.executable, "-c", IN_TWO_CONTEXTS], cwd=Path(q().__file__).resolve().parents[1], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ---------------------------------------------------------------------- waits that run out

@pytest.fixture(scope="module")
def nowait():
    """The library whose bounded waits run out at once: no kernel of it waits for anything, none fails otherwise."""
    from qrb200 import _lib
    h = ctypes.CDLL(str(_lib.NOWAIT_LIB_PATH))
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(h, name)
        fn.restype, fn.argtypes = res, args
    return h


# one CTA a tile; a cluster of several; the persistent pairs, with and without rows that TMA can address
@pytest.mark.parametrize("m,n,k", [(40, 20000, 64), (16, 256, 4096), (2048, 2048, 256), (2048, 2049, 256), (300, 520, 4096)])
@pytest.mark.parametrize("residual,slope", [(False, False), (True, False), (True, True)])
def test_waits_that_run_out_are_reported(nowait, m, n, k, residual, slope):
    """The call returns, the flag is up and every output is NaN; the flag comes down, and the context works on."""
    from qrb200 import _lib
    x, w = rnd(m, k, dtype=BF, seed=1), rnd(n, k, dtype=BF, seed=2)
    r, y = rnd(m, n, dtype=BF, seed=3), torch.zeros(m, n, dtype=BF, device="cuda")
    s = torch.zeros(m, n, dtype=torch.int16, device="cuda")
    timed_out = ctypes.c_int32(-1)
    assert nowait.qrb200_layer_status(ctypes.byref(timed_out)) == _lib.QRB200_OK and timed_out.value == 0
    assert nowait.qrb200_linear(x.data_ptr(), k, w.data_ptr(), k, 0, None, None, None, r.data_ptr() if residual else None, n, y.data_ptr(), n,
                                s.data_ptr() if slope else None, m, n, k, 1, 1, _lib.ACT_GELU, None, 0, stream()) == _lib.QRB200_OK
    assert nowait.qrb200_layer_status(ctypes.byref(timed_out)) == _lib.QRB200_OK and timed_out.value == 1
    assert bool(torch.isnan(y).all())
    assert not slope or bool((s == -1).all())  # 65535: NaN
    assert nowait.qrb200_layer_status(ctypes.byref(timed_out)) == _lib.QRB200_OK and timed_out.value == 0
    assert bool(torch.isfinite(q().linear(x, w, residual=r)).all()) and not _lib.layer_timed_out()


# ---------------------------------------------------------------------- the ends of the ranges

def test_scales_of_empty_rows():
    """The largest of no elements is 0, so the scale is the smallest one, 2^-126, and not what was there."""
    import ctypes
    from qrb200 import _lib
    L = _lib.lib()
    for rows in (1, 5, 1000):
        for call in (lambda s: L.qrb200_quantize_rows(None, 0, None, s, rows, 0, _lib.QRB200_BF16, stream()),
                     lambda s: L.qrb200_rms_norm(None, 0, None, 0, None, 0, 0, None, s, None, rows, 0, 1e-6, _lib.QRB200_F32, _lib.QRB200_E4M3,
                                                 stream())):
            scale = torch.full((rows + 1,), 7.0, device="cuda")
            assert call(ctypes.c_void_p(scale.data_ptr())) == _lib.QRB200_OK
            assert bool((scale[:rows] == 2.0 ** -126).all()) and float(scale[rows]) == 7.0
    y, s = q().quantize_rows(torch.empty(3, 4, 0, dtype=BF, device="cuda"))
    assert y.shape == (3, 4, 0) and s.shape == (3, 4) and bool((s == 2.0 ** -126).all())


@pytest.mark.parametrize("gain", [1e-16, 1e15])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,dim", [(300, 64), (5, 4096), (300, 65), (2, 3001), (3, 20000)])
def test_norm_gradient_of_tiny_and_huge_rows(rows, dim, dtype, gain):
    """eps = 0 and rows of about 1e-16 or 1e15: the cube of the root's inverse leaves float32, the gradient does not.
    Sums of float32 against their magnitudes: 2^-17 as for ordinary rows (squares and their sums are normal numbers)."""
    x = rnd(rows, dim, dtype=dtype, seed=1, gain=gain).requires_grad_()
    w, dy = (rnd(dim, dtype=dtype, seed=2) + 1).requires_grad_(), rnd(rows, dim, dtype=dtype, seed=3)
    dx, dw = torch.autograd.grad(q().rms_norm(x, w, eps=0.0), (x, w), dy)
    h, g = x.detach().double(), dy.double() * w.detach().double()
    r = h.square().mean(-1, keepdim=True).rsqrt()
    want = r * g - r ** 3 * (g * h).mean(-1, keepdim=True) * h
    size = (r * g).abs() + r ** 3 * (g * h).abs().mean(-1, keepdim=True) * h.abs()
    u = {F32: 2.0 ** -24, BF: 2.0 ** -8}[dtype]
    assert bool(((dx.double() - want).abs() <= u * (1 + 2 ** -10) * want.abs() + 2.0 ** -17 * size).all())
    terms = dy.double() * h * r
    assert bool(((dw.double() - terms.sum(0)).abs() <= u * (1 + 2 ** -10) * terms.sum(0).abs() + 2.0 ** -16 * terms.abs().sum(0)).all())


# ---------------------------------------------------------------------- gradients in an activation's tail

@pytest.mark.parametrize("m", [40, 512, 6000])
@pytest.mark.parametrize("act,bias", [("gelu", -3.0), ("gelu", -4.0), ("gelu", -5.0), ("gelu_tanh", -4.0), ("silu", -10.0), ("silu", -14.0)])
def test_gradients_in_a_tail(act, bias, m):
    """Features whose z all lie where act' is small still learn.  act' is held as its root in steps of 2^-15, so it is
    off by 2 |act'|^(1/2) 2^-16 + 2^-32, and by 2^-9 of itself through the formula's approximations out there; dz is
    rounded to bf16 (u = 2^-8) for dw and dx, not for db; sums are added as in any product."""
    n, k, u = 16, 64, 2.0 ** -8
    x, w = rnd(m, k, dtype=BF, seed=1).requires_grad_(), rnd(n, k, dtype=BF, seed=2, gain=0.02).requires_grad_()
    b = torch.full((n,), bias, dtype=BF, device="cuda").requires_grad_()
    dy = rnd(m, n, dtype=BF, seed=3).abs()
    dx, dw, db = torch.autograd.grad(q().linear(x, w, b, activation=act), (x, w, b), dy)
    x64, w64, z = x.detach().double(), w.detach().double(), None
    z = (x64 @ w64.T + bias).requires_grad_()
    f = {"gelu": lambda t: t * torch.special.ndtr(t), "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)),
         "silu": lambda t: t * torch.sigmoid(t)}[act]
    slope, = torch.autograd.grad(f(z).sum(), z)
    dz = dy.double() * slope
    ddz = dy.double() * (2.0 ** -15 * slope.abs().sqrt() + 2.0 ** -32 + 2.0 ** -9 * slope.abs())
    rdz = ddz + u * (1 + 2 ** -10) * dz.abs()
    for got, want, err, mag, steps in ((dw, dz.T @ x64, rdz.T @ x64.abs(), dz.abs().T @ x64.abs(), m), (dx, dz @ w64, rdz @ w64.abs(), dz.abs() @ w64.abs(), n),
                                       (db, dz.sum(0), ddz.sum(0), dz.abs().sum(0), m)):
        tol = u * (1 + 2 ** -10) * want.abs() + err * (1 + u) + (steps / 16 + 16) * 2.0 ** -23 * (mag + err)
        assert bool(((got.double() - want).abs() <= tol).all())
    # all terms of db have one sign, so its bound is one on its relative error
    assert bool((db.double() / dz.sum(0) - 1).abs().max() < 2.0 ** -5)


# ---------------------------------------------------------------------- strides

def bits(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,dim", [(40, 96), (300, 96), (40, 2048), (400, 2048), (7, 16392)])
def test_norm_of_strided_rows(rows, dim, fp8, dtype):
    """Rows that all start on 16 bytes give the bits of their contiguous copies, whatever lies between them; so do, among
    themselves, rows that do not, which are read one element at a time.  The stream is the same everywhere.  Between the
    two the sums are added in another order: each y is within u + 2^-18 of the exact one (u = 2^-8, 2^-24), so two of them
    are within twice that, and in 8 bits within twice 2^-4 of a value or 2^-10 of the scale."""
    wide = rnd(rows, dim + 72, dtype=dtype, seed=1)
    w, res = rnd(dim, dtype=dtype, seed=2) + 1, rnd(rows, dim, dtype=dtype, seed=3)
    call = lambda x: q().rms_norm(x, w, residual=res, out_dtype=FP8 if fp8 else None)  # noqa: E731
    on, off = [0, 16, 64], [1, 3, 17]  # elements
    for starts in (on, off):
        for c in starts:
            x = wide[:, c:c + dim]
            assert (x.data_ptr() % 16 == 0) == (starts is on) and not x.is_contiguous()
            got = call(x)
            if starts is on:
                same = call(x.contiguous())
            else:  # the same rows at another odd distance
                other = torch.empty(rows, dim + 41, dtype=dtype, device="cuda")[:, 5:5 + dim]
                same = call(other.copy_(x))
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, same))
            plain = call(x.contiguous())
            assert torch.equal(got[-1], plain[-1])  # the stream
            if fp8:
                assert bool(((got[1] - plain[1]).abs() <= 2.0 ** -17 * plain[1]).all())
                a, b, s = got[0].double() * got[1].double()[:, None], plain[0].double() * plain[1].double()[:, None], plain[1].double()[:, None]
                tol = 2 * (torch.maximum(2.0 ** -4 * torch.maximum(a.abs(), b.abs()) * (1 + 2.0 ** -4), 2.0 ** -10 * s * (1 + 2.0 ** -12)))
            else:
                a, b = got[0].double(), plain[0].double()
                tol = 2 * ({BF: 2.0 ** -8, F32: 2.0 ** -24}[dtype] + 2.0 ** -18) * (1 + 2.0 ** -7) * b.abs() + 2.0 ** -133
            assert bool(((a - b).abs() <= tol).all())


# ---------------------------------------------------------------------- the operators' registration

@pytest.mark.parametrize("kept", [BF, F32])
def test_operators_keep_their_schemas(kept):
    """Torch's own checks of an operator: no output shares memory with an input or another output, the meta kernel agrees
    with the CUDA one, and a compiled step gives what the operator gives."""
    from qrb200 import _lib
    q().api.load_torch_ops()
    ops, grad = torch.ops.qrb200, lambda *ts: [t.clone().requires_grad_() for t in ts]  # noqa: E731
    x, g, r, w, b = (rnd(5, 64, dtype=BF, seed=1), rnd(64, dtype=BF, seed=2), rnd(5, 64, dtype=kept, seed=3), rnd(40, 64, dtype=BF, seed=4),
                     rnd(40, dtype=BF, seed=5))
    dy, dh, dz = rnd(5, 64, dtype=BF, seed=6), rnd(5, 64, dtype=kept, seed=7), rnd(5, 40, dtype=BF, seed=8)
    slope = ops.linear(x, w, b, None, _lib.ACT_SILU, None, None, None, True)[1]
    for op, args in ((ops.rms_norm, (x, g, r, 1e-6, None)), (ops.rms_norm, (*grad(x, g, r), 1e-6, None)), (ops.rms_norm, (x, None, None, 1e-6, FP8)),
                     (ops.rms_norm_backward, (dy, r, dh, g, 1e-6, True, True, True)),
                     (ops.rms_norm_backward, (dy, r, None, None, 1e-6, False, True, False)),
                     (ops.quantize_rows, (r,)),
                     (ops.linear, (x, w, b, None, _lib.ACT_GELU, None, None, None, True)),
                     (ops.linear, (*grad(x, w, b), None, _lib.ACT_GELU, None, None, None, False)),
                     (ops.linear_backward, (dz, slope, x, w, True, True, True)), (ops.linear_backward, (dz, None, x, w, False, True, False))):
        torch.library.opcheck(op.default, args)
    # the same numbers by way of autograd, with the residual's gradient where it is dx and where it is not
    xg, rg = grad(x, r)
    y, h = q().rms_norm(xg, g, residual=rg)
    dx, dr = torch.autograd.grad((y, h), (xg, rg), (dy, dh))
    want = ops.rms_norm_backward(dy, h.detach(), dh, g, 1e-6, True, True, False)
    assert torch.equal(dx, want[0]) and torch.equal(dr, want[0] if kept == BF else want[1])
    dr, = torch.autograd.grad(q().rms_norm(x, g, residual=rg), rg, (dy, dh))
    assert torch.equal(dr, want[0] if kept == BF else want[1])
