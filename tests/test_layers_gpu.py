"""GPU: rms_norm, quantize_rows, linear and their gradients against plain float64 formulas.

Bounds.  u(T) is the unit roundoff of a type (2^-8 bf16, 2^-11 f16, 2^-24 f32, 2^-4 e4m3) and an output is
rounded once, so |y - y64| <= u |y64| + what float32 arithmetic before it costs:
  norm     sums of squares are added by up to 64 sequential terms and a tree, then a root and two products:
           2^-18 relative; sums of signed terms are held against the sum of their magnitudes, 2^-17.
  product  the accumulator drops up to one unit in the last place (2^-23) at each of the k / 16 (k / 32) steps and
           in the alignment inside a step: (k / 16 + 16) 2^-23 sum |x w|; activations have a slope below 1.13 and
           are themselves good to 2^-19 (|z| + 1).
  dz       is rounded to the operands' type: u sum |dz| |w|; act' is held to 2^-15.
Each type's smallest subnormal covers what lies below its range.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _give_memory_back():
    """Leaves no cached blocks behind: with none, what the next module allocates comes from the device again."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

BF, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
SUB = {BF: 2.0 ** -133, F16: 2.0 ** -25, F32: 2.0 ** -149}
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def q():
    import qrb200
    return qrb200


def rnd(*shape, dtype=F32, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * gain).to(dtype)


def within(got, want, tol):
    got, bad = got.double(), None
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs() - tol
    off = torch.where(torch.isnan(want) | (got == want), torch.full_like(off, -1.0), off)
    bad = off > 0
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(off.max()):.3g} over its bound"


# ---------------------------------------------------------------------- rms_norm

def norm64(x, w, res, eps, kept):
    h = x.double() if res is None else (x.double() + res.double()).to(kept).double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = h * r * (1.0 if w is None else w.double())
    return h, r, y


def check_norm(x, w, res, eps=1e-6, fp8=False):
    kept = x.dtype if res is None else res.dtype
    h64, _, y64 = norm64(x, w, res, eps, kept)
    got = q().rms_norm(x, w, residual=res, eps=eps, out_dtype=FP8 if fp8 else None)
    got = got if isinstance(got, tuple) else (got,)
    if res is not None:
        within(got[-1], x.double() + res.double(), U[kept] * (1 + 2 ** -12) * (x.double() + res.double()).abs() + SUB[kept])
        # the norm is that of the stream as it is kept
        _, _, y64 = norm64(got[-1], w, None, eps, kept)
    if fp8:
        s64 = (y64.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
        within(got[1], s64, 2.0 ** -18 * s64)
        s = got[1].double().unsqueeze(-1)
        within(got[0].double() * s, y64, torch.maximum(2.0 ** -4 * y64.abs(), 2.0 ** -10 * s) * (1 + 2.0 ** -12) + 2.0 ** -18 * y64.abs())
    else:
        within(got[0], y64, (U[x.dtype] + 2.0 ** -18) * y64.abs() + SUB[x.dtype])
    return got


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,kept", [(F32, F32), (BF, BF), (BF, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (300, 64), (5, 512), (700, 513), (2, 4096), (350, 4096), (3, 8200),
                                      (400, 1000), (2, 16384), (301, 16384), (2, 16390), (1, 40000)])
def test_norm(rows, dim, dtype, kept, fp8):
    x, w = rnd(rows, dim, dtype=dtype, seed=1, gain=3), rnd(dim, dtype=dtype, seed=2) + 1
    check_norm(x, w, rnd(rows, dim, dtype=kept, seed=3), fp8=fp8)
    check_norm(x, w.float(), None, fp8=fp8)
    check_norm(x, None, None, eps=0.5, fp8=fp8)


@pytest.mark.parametrize("fp8", [False, True])
def test_norm_strides(fp8):
    big = rnd(40, 3, 200, dtype=BF, seed=4)
    w = rnd(96, dtype=BF, seed=5)
    for x in (big[:, :, :96], big[:, :, 1:97], big[:, 1, 8:104], big[::2, 0, 3:99], big[:7, 0, :96].transpose(0, 1).contiguous().t(),
              big[0, 0, :96].expand(6, 96), big[0, 0, :96], big[:, :, 100:196].transpose(0, 1)):
        res = rnd(*x.shape, dtype=F32, seed=6)
        got = check_norm(x, w, res, fp8=fp8)
        same = q().rms_norm(x.contiguous(), w, residual=res, out_dtype=FP8 if fp8 else None)
        assert all(torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, b.view(torch.uint8) if b.dtype == FP8 else b)
                   for a, b in zip(got, same)) or not x.is_contiguous()


def test_norm_special_rows():
    x = rnd(12, 256, dtype=F32, seed=7)
    x[0] = 0
    x[1, 5], x[2, 7], x[3, 9] = float("nan"), float("inf"), float("-inf")
    x[4] = 1e-30
    x[5] *= 1e18
    y = q().rms_norm(x)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and bool(torch.isnan(y[1]).all())
    for i, c in ((2, 7), (3, 9)):  # an infinity: its own place is inf * 0, the others 0
        assert bool(torch.isnan(y[i, c])) and int(torch.isnan(y[i]).sum()) == 1 and float(y[i].nan_to_num(0).abs().max()) == 0
    within(y[4:], norm64(x[4:], None, None, 1e-6, F32)[2], 2.0 ** -18 * norm64(x[4:], None, None, 1e-6, F32)[2].abs() + 2 ** -149)
    y8, s = q().rms_norm(x, out_dtype=FP8)
    assert float(s[0]) == 2.0 ** -126 and float(y8[0].float().abs().max()) == 0
    assert bool(torch.isnan(s[1:4]).all()) and bool(torch.isnan(y8[1].float()).all())
    assert bool(torch.isfinite(s[4:]).all())
    check_norm(x[4:], None, None, fp8=True)
    # the rows beside them are not touched, and a masked-out row of the lowest value is a row like others
    low = torch.full((2, 64), torch.finfo(BF).min, dtype=BF, device="cuda")
    assert not bool(q().rms_norm(low).any())  # its square overflows: r = 0
    # in 8 bits too, where h w would overflow float32 but y = (h r) w does not; beside ordinary rows
    for rows, dim, w in ((2, 64, 2.0), (700, 72, 2.0), (3, 4096, 3.0), (400, 2047, 2.0), (2, 20000, 2.0)):
        low = rnd(rows, dim, dtype=BF, seed=12)
        low[::2] = torch.finfo(BF).min
        q8, s8 = q().rms_norm(low, torch.full((dim,), w, dtype=BF, device="cuda"), out_dtype=FP8)
        assert not bool(q8[::2].float().any()) and bool((s8[::2] == 2.0 ** -126).all())
        check_norm(low[1::2], torch.full((dim,), w, dtype=BF, device="cuda"), None, fp8=True)
    big = torch.full((4, 256), 1e-3, device="cuda")
    w = torch.full((256,), 3e38, device="cuda")
    q8, s8 = q().rms_norm(big, w, eps=0.0, out_dtype=FP8)
    assert bool((q8.float() == 448).all()) and bool(((s8 - 3e38 / 448).abs() <= 2e33).all())
    # an in-place stream
    from qrb200 import _lib
    a, r = rnd(4, 64, dtype=BF, seed=8), rnd(4, 64, dtype=BF, seed=9)
    want = q().rms_norm(a, residual=r)
    out = torch.empty_like(a)
    rc = _lib.lib().qrb200_rms_norm(a.data_ptr(), 64, None, 0, r.data_ptr(), 64, 1, out.data_ptr(), None, r.data_ptr(), 4, 64, 1e-6, 1, 1,
                                    torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(out, want[0]) and torch.equal(r, want[1])


def test_norm_empty():
    for shape in ((0, 8), (3, 0), (2, 0, 8)):
        y, h = q().rms_norm(torch.empty(*shape, device="cuda"), residual=torch.empty(*shape, device="cuda"))
        assert y.shape == h.shape == shape
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    q().rms_norm(x, w).sum().backward()
    assert float(w.grad.abs().max()) == 0


@pytest.mark.parametrize("dtype,kept", [(F32, F32), (BF, BF), (BF, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (700, 64), (1300, 513), (5, 2048), (333, 4096), (200, 5000), (400, 16384), (3, 16390)])
def test_norm_gradients(rows, dim, dtype, kept):
    eps = 1e-3
    x, res = rnd(rows, dim, dtype=dtype, seed=1, gain=2).requires_grad_(), rnd(rows, dim, dtype=kept, seed=2).requires_grad_()
    w = (rnd(dim, dtype=F32 if dtype == BF and kept == F32 else dtype, seed=3) + 1).detach().requires_grad_()
    dy, dh = rnd(rows, dim, dtype=dtype, seed=4), rnd(rows, dim, dtype=kept, seed=5)
    y, h = q().rms_norm(x, w, residual=res, eps=eps)
    dx, dw, dr = torch.autograd.grad((y, h), (x, w, res), (dy, dh))
    assert (dx.dtype, dw.dtype, dr.dtype) == (dtype, w.dtype, kept)
    hd, g, wd = h.detach().double(), dy.double(), w.detach().double()
    r = (hd.square().mean(-1, keepdim=True) + eps).rsqrt()
    c = r ** 3 * (g * wd * hd).mean(-1, keepdim=True)
    want = dh.double() + r * g * wd - c * hd
    tol = 2.0 ** -17 * (dh.double().abs() + (r * g * wd).abs() + r ** 3 * (g * wd * hd).abs().mean(-1, keepdim=True) * hd.abs())
    within(dx, want, U[dtype] * (1 + 2 ** -10) * want.abs() + tol + SUB[dtype])
    within(dr, want, U[kept] * (1 + 2 ** -10) * want.abs() + tol + SUB[kept])
    terms = g * hd * r
    within(dw, terms.sum(0), U[w.dtype] * (1 + 2 ** -10) * terms.sum(0).abs() + 2.0 ** -16 * terms.abs().sum(0) + SUB[w.dtype])
    # the same bits again, and the parts alone
    again = torch.autograd.grad(q().rms_norm(x, w, residual=res, eps=eps), (x, w, res), (dy, dh))
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and torch.equal(dr, again[2])
    xs = x.detach().clone().requires_grad_()
    only, = torch.autograd.grad(q().rms_norm(xs, w.detach(), eps=eps), xs, dy)
    hs = xs.detach().double()
    r = (hs.square().mean(-1, keepdim=True) + eps).rsqrt()
    want = r * g * wd - r ** 3 * (g * wd * hs).mean(-1, keepdim=True) * hs
    tol = 2.0 ** -17 * ((r * g * wd).abs() + r ** 3 * (g * wd * hs).abs().mean(-1, keepdim=True) * hs.abs())
    within(only, want, U[dtype] * (1 + 2 ** -10) * want.abs() + tol + SUB[dtype])


def test_norm_gradient_heads():
    """Only the stream is used, or only the norm; expanded and strided gradients."""
    x, w = rnd(33, 100, seed=1).requires_grad_(), rnd(100, seed=2).requires_grad_()
    res = rnd(33, 100, seed=3).requires_grad_()
    y, h = q().rms_norm(x, w, residual=res)
    dx, dw = torch.autograd.grad(h.sum(), (x, w))
    assert bool((dx == 1).all()) and bool((dw == 0).all())
    y, h = q().rms_norm(x, w, residual=res)
    a = torch.autograd.grad(y.sum(), (x, w, res))
    y, h = q().rms_norm(x, w, residual=res)
    b = torch.autograd.grad(y, (x, w, res), torch.ones(33, 100, device="cuda"))
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and torch.equal(a[0], a[2])


def test_norm_gradient_differences():
    """Central differences of a float32 norm: 2^-9 steps along a random direction.  Rounding: y is good to 2^-20, so
    the quotient to 2^-20 sqrt(sum (dy y)^2) * 2^9 (its errors are independent), taken eight times; curvature: the
    third derivative of h r is below 6 |v|^3 r^3 a unit, i.e. a relative (2^-9)^2."""
    rows, dim, e = 40, 96, 2.0 ** -9
    x, w, v = rnd(rows, dim, seed=1), rnd(dim, seed=2), rnd(rows, dim, seed=3)
    vw, dy = rnd(dim, seed=5), rnd(rows, dim, seed=4)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(q().rms_norm(xg, wg), (xg, wg), dy)
    loss = lambda a, b: (q().rms_norm(a, b).double() * dy.double()).sum()  # noqa: E731
    noise = 8 * 2.0 ** -20 * float((dy * q().rms_norm(x, w)).double().square().sum().sqrt()) / e
    for grad, diff in ((dx, (loss(x + e * v, w) - loss(x - e * v, w)) / (2 * e)), ):
        want = float((grad.double() * v.double()).sum())
        assert abs(float(diff) - want) <= noise + 16 * e * e * float((dy.double().abs() * v.double().abs()).sum())
    diff = (loss(x, w + e * vw) - loss(x, w - e * vw)) / (2 * e)
    assert abs(float(diff) - float((dw.double() * vw.double()).sum())) <= noise


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (4, 33), (500, 512), (3, 20000)])
def test_quantize_rows(rows, dim, dtype):
    x = rnd(rows, dim, dtype=dtype, seed=1, gain=0.02)
    y, s = q().quantize_rows(x)
    s64 = (x.double().abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    within(s, s64, 2.0 ** -22 * s64)
    sd = s.double().unsqueeze(-1)
    within(y.double() * sd, x.double(), torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * sd) * (1 + 2.0 ** -12))
    assert bool((y.float().abs().amax(-1) == 448).all())


# ---------------------------------------------------------------------- linear

def act64(z, name):
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    return z, torch.ones_like(z)


def check_linear(x, w, b=None, act=None, res=None, xs=None, ws=None, out=None):
    y = q().linear(x, w, b, activation=act, residual=res, x_scale=xs, weight_scale=ws, out_dtype=out)
    k = x.shape[-1]
    x64, w64 = x.double(), w.double()
    if xs is not None:
        x64 = x64 * xs.double().expand(x.shape[:-1]).unsqueeze(-1)
    if ws is not None:
        w64 = w64 * ws.double().expand(w.shape[0]).unsqueeze(-1)
    z = x64 @ w64.T
    mag = x64.abs() @ w64.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    want = act64(z, act)[0]
    tol = 1.13 * (k / 16 + 16) * 2.0 ** -23 * mag + 2.0 ** -19 * (z.abs() + 1) * (act is not None)
    if res is not None:
        want = want + res.double()
    within(y, want, U[y.dtype] * (1 + 2 ** -10) * want.abs() + tol + SUB[y.dtype])
    return y


SIZES = [(1, 1, 1), (1, 4096, 512), (1, 300, 8200), (2, 2500, 264), (3, 1203, 2049), (4, 2368, 1040), (4, 40, 5000), (1, 5000, 77), (3, 5, 7), (16, 128, 64), (17, 130, 200), (33, 257, 96), (64, 512, 1000), (65, 100, 4096),
         (128, 256, 128), (130, 384, 72), (200, 1001, 513), (256, 512, 512), (300, 640, 2050), (1000, 2000, 264), (513, 4224, 128),
         (2048, 2048, 64)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(m, n, k, dtype):
    x, w = rnd(m, k, dtype=dtype, seed=1), rnd(n, k, dtype=dtype, seed=2, gain=k ** -0.5)
    b, res = rnd(n, dtype=dtype, seed=3), rnd(m, n, dtype=dtype, seed=4)
    plain = check_linear(x, w)
    for i, act in enumerate(ACTS):
        check_linear(x, w, b if i % 2 else None, act, res if i != 2 else None)
    # the weight as a transposed view, read in place (up to 4 tokens by another kernel, in another order)
    wt = w.t().contiguous().t()
    assert torch.equal(check_linear(x, wt), plain) or m <= 4
    assert torch.equal(q().linear(x, w), plain)


# enough 256 x 256 tiles for the persistent kernel; edges inside tiles, rows off 16 bytes
LARGE = [(2048, 2048, 256), (1793, 2304, 520), (2305, 1793, 77), (16400, 264, 136), (300, 16400, 40), (4000, 2056, 1032)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_linear_large(m, n, k, dtype):
    x, w = rnd(m, k, dtype=dtype, seed=1), rnd(n, k, dtype=dtype, seed=2, gain=k ** -0.5)
    b, res = rnd(n, dtype=dtype, seed=3), rnd(m, n, dtype=dtype, seed=4)
    plain = check_linear(x, w)
    for i, act in enumerate(ACTS):
        check_linear(x, w, b if i % 2 else None, act, res if i != 2 else None)
    assert torch.equal(check_linear(x, w.t().contiguous().t()), plain)
    assert torch.equal(q().linear(x, w), plain)
    wide = rnd(m, n + 13, dtype=dtype, seed=6)
    check_linear(x, w, b, "silu", wide[:, 5:5 + n])
    check_linear(x, w, b, None, wide[0, :n].expand(m, n))


@pytest.mark.parametrize("m,n,k", LARGE)
def test_linear_large_8bit(m, n, k):
    x8, xs = q().quantize_rows(rnd(m, k, seed=1))
    w8, ws = q().quantize_rows(rnd(n, k, seed=2, gain=k ** -0.5))
    check_linear(x8, w8, rnd(n, dtype=BF, seed=3), "gelu", rnd(m, n, dtype=BF, seed=4), xs, ws)
    check_linear(x8, w8, None, None, None, xs, ws, F16)


@pytest.mark.parametrize("out", [None, F16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_8bit(m, n, k, out):
    x8, xs = q().quantize_rows(rnd(m, k, seed=1))
    w8, ws = q().quantize_rows(rnd(n, k, seed=2, gain=k ** -0.5))
    dt = out or BF
    check_linear(x8, w8, xs=xs, ws=ws, out=out)
    check_linear(x8, w8, rnd(n, dtype=dt, seed=3), "gelu", rnd(m, n, dtype=dt, seed=4), xs, ws, out)
    check_linear(x8, w8, None, "silu", None, xs[:1], ws[:1], out)
    check_linear((rnd(m, k, seed=1)).to(FP8), w8, None, None, None, None, None, out)


def test_linear_strides():
    big, n, k = rnd(50, 3, 400, dtype=BF, seed=1), 72, 136
    w = rnd(n + 3, k + 5, dtype=BF, seed=2, gain=0.1)
    for x in (big[:, :, :k], big[:, 1, 8:8 + k], big[:, 2, 3:3 + k], big[0, 0, :k], big[:, :, 11:11 + k].transpose(0, 1),
              big[0, 0, :k].expand(9, k), big[:k, 0, :40].t()):
        kk = x.shape[-1]
        for ww in (w[:n, :kk], w[1:n + 1, 3:3 + kk], w[:n, :kk].t().contiguous().t(), w[:n, 5:5 + kk].clone()):
            res = rnd(*x.shape[:-1], n, dtype=BF, seed=5)
            y = check_linear(x, ww, rnd(n, dtype=BF, seed=4), "relu", res)
            same = q().linear(x.contiguous(), ww.contiguous(), rnd(n, dtype=BF, seed=4), activation="relu", residual=res)
            assert torch.equal(y, same) or x.numel() <= 4 * kk
    # the residual as a slice of a wider stream, and expanded
    x, ww = big[:, 0, :k], w[:n, :k]
    wide = rnd(50, 200, dtype=BF, seed=6)
    check_linear(x, ww, None, "silu", wide[:, 5:5 + n])
    check_linear(x, ww, None, "silu", wide[0, :n].expand(50, n))


def test_linear_special():
    # empty sums: y = act(bias) + residual
    b, res = rnd(24, dtype=BF, seed=1), rnd(10, 24, dtype=BF, seed=2)
    y = check_linear(torch.empty(10, 0, dtype=BF, device="cuda"), torch.empty(24, 0, dtype=BF, device="cuda"), b, "gelu", res)
    assert y.shape == (10, 24)
    assert q().linear(torch.empty(0, 8, dtype=BF, device="cuda"), torch.empty(24, 8, dtype=BF, device="cuda")).shape == (0, 24)
    assert q().linear(rnd(3, 8, dtype=BF), torch.empty(0, 8, dtype=BF, device="cuda")).shape == (3, 0)
    # a NaN or an infinity stays in its own row
    x, w = rnd(40, 64, dtype=BF, seed=3), rnd(48, 64, dtype=BF, seed=4)
    clean = q().linear(x, w, activation="relu")
    x[7, 3], x[20, 0] = float("nan"), float("inf")
    for act in ACTS:
        y = q().linear(x, w, activation=act)
        assert bool(torch.isnan(y[7]).all()) and not bool(torch.isfinite(y[20]).any() and act is None)
    y = q().linear(x, w, activation="relu")
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(y[keep], clean[keep])
    # large |z|: the activations' limits, no overflow on the way
    z = torch.tensor([[-200.0, -60.0, -10.0, 0.0, 10.0, 60.0, 200.0]], dtype=BF, device="cuda")
    for act in ACTS[1:]:
        y = q().linear(z, torch.eye(7, dtype=BF, device="cuda"), activation=act)
        assert torch.equal(y[0, 3:], z[0, 3:]), act
        assert float(y[0, :2].abs().max()) <= 60 * math.exp(-60) * (1 + 2.0 ** -8), act  # silu(-60) is not 0
        assert float(y[0, 2].abs()) < 1e-3


def test_linear_other_stream():
    x, w = rnd(300, 512, dtype=BF, seed=1), rnd(256, 512, dtype=BF, seed=2)
    want = q().linear(x, w, activation="silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = q().linear(x, w, activation="silu")
        n = q().rms_norm(y)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want) and torch.equal(n, q().rms_norm(want))


def test_layers_in_a_graph():
    """A captured chain replays on new inputs."""
    x, w = rnd(5, 256, dtype=BF, seed=1), rnd(256, 256, dtype=BF, seed=2, gain=0.06)
    w8, ws = q().quantize_rows(w)

    def step():
        y8, s, h = q().rms_norm(x, residual=x, out_dtype=FP8)
        return q().linear(y8, w8, x_scale=s, weight_scale=ws, residual=h)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(rnd(5, 256, dtype=BF, seed=3))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, step())


GRAD_SIZES = [(1, 1, 1), (3, 5, 7), (16, 128, 64), (70, 130, 200), (64, 512, 1000), (1000, 100, 64), (300, 257, 513),
              (4100, 64, 128), (256, 512, 512), (700, 1000, 264), (2048, 2048, 2048), (2300, 1993, 2050)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", GRAD_SIZES)
def test_linear_gradients(m, n, k, act, dtype):
    x, w = rnd(m, k, dtype=dtype, seed=1).requires_grad_(), rnd(n, k, dtype=dtype, seed=2, gain=k ** -0.5)
    if m % 2:
        w = w.t().contiguous().t()
    w.requires_grad_()
    b, res = rnd(n, dtype=dtype, seed=3).requires_grad_(), rnd(m, n, dtype=dtype, seed=4).requires_grad_()
    dy = rnd(m, n, dtype=dtype, seed=5)
    y = q().linear(x, w, b, activation=act, residual=res)
    dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, res), dy)
    assert torch.equal(dr, dy)
    x64, w64, g = x.detach().double(), w.detach().double(), dy.double()
    z = x64 @ w64.T + b.detach().double()
    noise = (k / 16 + 16) * 2.0 ** -23 * (x64.abs() @ w64.abs().T + b.detach().double().abs())  # of z
    slope = act64(z, act)[1]
    dz = g * slope
    # act' at a z that is off by the noise, held to 2^-15 (|act''| <= 0.8); relu's kink may fall either way
    dslope = torch.zeros_like(z) if act is None else 0.8 * noise + 2.0 ** -15 + 2.0 ** -18 * (z.abs() + 1)
    if act == "relu":
        dslope = (z.abs() <= noise).double()
    u = U[dtype]
    ddz = g.abs() * dslope
    rdz = ddz + (u * dz.abs() * (1 + 2 ** -10) + SUB[dtype] if act is not None else 0)
    for got, want, mag, err, steps in (
            (dx, dz @ w64, dz.abs() @ w64.abs(), rdz @ w64.abs(), n), (dw, dz.T @ x64, dz.abs().T @ x64.abs(), rdz.T @ x64.abs(), m)):
        within(got, want, u * (1 + 2 ** -10) * want.abs() + err * (1 + u) + (steps / 16 + 16) * 2.0 ** -23 * (mag + err) + SUB[dtype])
    want = dz.sum(0)
    within(db, want, u * (1 + 2 ** -10) * want.abs() + ddz.sum(0) * (1 + u) + 2.0 ** -16 * dz.abs().sum(0) + SUB[dtype])
    again = torch.autograd.grad(q().linear(x, w, b, activation=act, residual=res), (x, w, b), dy)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and torch.equal(db, again[2])


def test_linear_gradient_differences():
    """Central differences of the f16 layer along directions that f16 steps of 2^-5 hold exactly.  y is rounded to
    2^-11 of itself, independently, so the quotient is off by 2^-11 sqrt(sum (dy y)^2) / 2^-5, taken six times; the
    third derivative of an activation is below 2: (2^-5)^2 / 3 sum |dy| |v|^3 at most; gradients are rounded to 2^-11."""
    m, n, k, e = 64, 48, 80, 2.0 ** -5
    w = rnd(n, k, dtype=F16, seed=2, gain=k ** -0.5)
    # multiples of 2^-6 below 8, directions of +-1: x +- e v is exact in f16
    x = (rnd(m, k, seed=1).clamp(-4, 4) * 64).round().div(64).to(F16)
    v = torch.sign(rnd(m, k, seed=3)).to(F16)
    vb = torch.sign(rnd(n, seed=6)).to(F16)
    b = (rnd(n, seed=7) * 64).round().div(64).to(F16)
    dy = rnd(m, n, dtype=F16, seed=4)
    for act in (None, "gelu", "gelu_tanh", "silu"):
        xg, bg = x.clone().requires_grad_(), b.clone().requires_grad_()
        y = q().linear(xg, w, bg, activation=act)
        dx, db = torch.autograd.grad(y, (xg, bg), dy)
        loss = lambda a, c: (q().linear(a, w, c, activation=act).double() * dy.double()).sum()  # noqa: E731
        noise = 6 * 2.0 ** -11 * float((dy.double() * y.detach().double()).square().sum().sqrt()) / e
        dv = (v.double() @ w.double().T)
        bend = e * e / 3 * float((dy.double().abs() * dv.abs() ** 3).sum()) if act else 0.0
        want = float((dx.double() * v.double()).sum())
        got = float((loss(x + e * v, b) - loss(x - e * v, b)) / (2 * e))
        assert abs(got - want) <= noise + bend + 6 * 2.0 ** -11 * float(dx.double().norm()), act
        bend = e * e / 3 * float(dy.double().abs().sum()) if act else 0.0
        want = float((db.double() * vb.double()).sum())
        got = float((loss(x, b + e * vb) - loss(x, b - e * vb)) / (2 * e))
        assert abs(got - want) <= noise + bend + 6 * 2.0 ** -11 * float(db.double().norm()), act


def test_linear_gradient_special():
    x = rnd(6, 32, dtype=BF, seed=1).requires_grad_()
    w = rnd(8, 32, dtype=BF, seed=2).requires_grad_()
    b = rnd(8, dtype=BF, seed=3).requires_grad_()
    # expanded gradient of a sum
    a = torch.autograd.grad(q().linear(x, w, b, activation="gelu").sum(), (x, w, b))
    c = torch.autograd.grad(q().linear(x, w, b, activation="gelu"), (x, w, b), torch.ones(6, 8, dtype=BF, device="cuda"))
    assert all(torch.equal(s, t) for s, t in zip(a, c))
    # a NaN reaches the gradients it belongs to
    xn = x.detach().clone()
    xn[2, 0] = float("nan")
    xn.requires_grad_()
    dx, db = torch.autograd.grad(q().linear(xn, w, b, activation="silu").sum(), (xn, b))
    assert bool(torch.isnan(dx[2]).all()) and not bool(torch.isnan(dx[[0, 1, 3, 4, 5]]).any()) and bool(torch.isnan(db).all())
    # no tokens, no features: zero gradients
    x0 = torch.empty(0, 32, dtype=BF, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(q().linear(x0, w, b, activation="relu").sum(), (w, b))
    assert not bool(dw.any()) and not bool(db.any())
    w0 = torch.empty(0, 32, dtype=BF, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(q().linear(x, w0).sum(), (x,))
    assert not bool(dx.any())
    # the residual alone
    res = rnd(6, 8, dtype=BF, seed=4).requires_grad_()
    dr, = torch.autograd.grad(q().linear(x.detach(), w.detach(), residual=res), (res,), c[0].new_ones(6, 8))
    assert bool((dr == 1).all())


def test_no_wait_ran_out():
    from qrb200 import _lib
    assert not _lib.layer_timed_out()


def test_both_ways_in():
    """The short way from Python and torch.ops are the same operator; what the short way does not take goes the other."""
    from qrb200 import layers
    x, w, r = rnd(7, 96, dtype=BF, seed=1), rnd(96, dtype=BF, seed=2), rnd(7, 96, dtype=BF, seed=3)
    W = rnd(40, 96, dtype=BF, seed=4)
    layers._Ops.loaded or layers._Ops.load()
    y, _, h = torch.ops.qrb200.rms_norm(x, w, r, 1e-6, None)
    a, b = q().rms_norm(x, w, residual=r)
    assert torch.equal(a, y) and torch.equal(b, h)
    assert torch.equal(q().linear(x, W, activation="silu"), torch.ops.qrb200.linear(x, W, None, None, 4, None, None, None, False)[0])
    # eps as an int, a tensor subclass, a function mode, a transform: not the short way, the same result
    one = q().rms_norm(x, w, eps=1.0)
    assert torch.equal(q().rms_norm(x, w, eps=1), one)

    class Sub(torch.Tensor):
        pass
    assert torch.equal(q().rms_norm(x.as_subclass(Sub), w, eps=1.0).as_subclass(torch.Tensor), one)

    class Mode(torch.overrides.TorchFunctionMode):
        seen = 0

        def __torch_function__(self, func, types, args=(), kwargs=None):
            Mode.seen += 1
            return func(*args, **(kwargs or {}))
    with Mode():
        assert torch.equal(q().rms_norm(x, w, eps=1.0), one)
    assert Mode.seen
    with torch.inference_mode():
        assert torch.equal(q().rms_norm(x, w, eps=1.0), one)
    with torch.no_grad():
        assert not q().linear(x.clone().requires_grad_(), W).requires_grad
    for bad in (lambda: q().rms_norm(x.double()), lambda: q().linear(x, W, out_dtype=F32), lambda: q().rms_norm(x, r)):
        with pytest.raises((TypeError, ValueError)):
            bad()
    p = torch.nn.Parameter(W)
    y = q().linear(x, p)
    assert y.requires_grad and torch.autograd.grad(y.sum(), p)[0].shape == W.shape
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(q().linear(x, p).square().sum(), p, create_graph=True)


def test_offsets_past_32_bits():
    """Rows whose offsets pass 2^31 elements (and 2^32 bytes)."""
    rows, ld = 33000, 66048
    wide = torch.empty(rows, ld, dtype=BF, device="cuda")  # 4.4 GB, of which the views below are filled
    last = slice(rows - 40, rows)
    for c in (0, 65000, 65001):
        x = wide[:, c:c + 136]
        x.copy_(rnd(rows, 136, dtype=BF, seed=1))
        w, W = rnd(136, dtype=BF, seed=2), rnd(264, 136, dtype=BF, seed=3)
        y, h = q().rms_norm(x, w, residual=x)
        y1, h1 = q().rms_norm(x[last].clone(), w, residual=x[last].clone())
        assert torch.equal(y[last], y1) and torch.equal(h[last], h1)
        z = q().linear(x, W, activation="gelu", residual=wide[:, :264] if c else None)
        if not c:
            check_linear(x[last].clone(), W, act="gelu")
            want = q().linear(x.contiguous(), W, activation="gelu")
        else:
            want = q().linear(x.contiguous(), W, activation="gelu", residual=wide[:, :264].contiguous())
        assert torch.equal(z, want)
        t = q().linear(x[rows - 1], W)
        check_linear(x[rows - 1].clone(), W)
        assert torch.equal(t, q().linear(x[rows - 1].clone(), W))
        wide[:, :264].copy_(rnd(rows, 264, dtype=BF, seed=4))


@pytest.mark.parametrize("m,n", [(1, 4096), (40, 520), (40, 519), (2100, 2056), (2100, 2049)])
def test_linear_in_place_residual(m, n):
    """y over its own residual, through the C ABI, in each kernel and with rows off 16 bytes."""
    from qrb200 import _lib
    x, w, r = rnd(m, 256, dtype=BF, seed=1), rnd(n, 256, dtype=BF, seed=2), rnd(m, n, dtype=BF, seed=3)
    want = q().linear(x, w, activation="silu", residual=r)
    rc = _lib.lib().qrb200_linear(x.data_ptr(), 256, w.data_ptr(), 256, 0, None, None, None, r.data_ptr(), n, r.data_ptr(), n, None,
                                  m, n, 256, _lib.QRB200_BF16, _lib.QRB200_BF16, _lib.ACT_SILU, None, 0,
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.QRB200_OK and torch.equal(r, want)


@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_linear_8bit_nan(m):
    x8, xs = q().quantize_rows(rnd(m, 96, seed=1))
    w8, ws = q().quantize_rows(rnd(72, 96, seed=2))
    x8.view(torch.uint8)[m // 2, 5] = 0x7F  # e4m3's NaN
    y = q().linear(x8, w8, x_scale=xs, weight_scale=ws)
    rows = torch.isnan(y).all(-1)
    assert bool(rows[m // 2]) and int(rows.sum()) == 1 and int(torch.isnan(y).any(-1).sum()) == 1


def test_chain_is_ordered():
    """Kernels that start before the ones ahead of them have ended still see what those wrote: a chain that is
    long and short by turns, against the same chain with a wait after every call."""
    W = [rnd(512, 512, dtype=BF, seed=i, gain=0.04) for i in range(3)]
    x0 = rnd(700, 512, dtype=BF, seed=9)

    def chain(wait):
        x, h = x0, x0
        for i in range(60):
            rows = (700, 3, 1, 260)[i % 4]
            y, h2 = q().rms_norm(x[:rows], residual=h[:rows])
            wait()
            y8, s = q().quantize_rows(y)
            wait()
            w8, t = q().quantize_rows(W[i % 3])
            wait()
            z = q().linear(y8, w8, x_scale=s, weight_scale=t, activation="silu", residual=h2)
            wait()
            u = q().linear(z, W[(i + 1) % 3], activation="gelu")
            wait()
            x = torch.cat((u, x[rows:]))
            h = torch.cat((z, h[rows:]))
        return x, h
    a = chain(lambda: None)
    b = chain(torch.cuda.synchronize)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
