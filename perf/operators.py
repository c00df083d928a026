"""Cases of the layer operators: the root-mean-square norm with the residual's addition (16-bit and
8-bit outputs, forward and backward) and the matrix product with bias, activation and residual in
its epilogue (16-bit operands, and 8-bit operands with scales; forward and backward).

``own`` chooses what ``run`` computes with: the operators' plain form in elementary torch
operations, or the library's entry points ``qrb200.rms_norm`` and ``qrb200.linear``."""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0
_TINY = 2.0 ** -126
_EPS = 1e-6


def listed():
    return [
        # one token of a decoding step: the stream takes the last layer's output and is normed to 8 bits
        {"name": "norm8 one token", "op": "norm8", "rows": 1, "dim": 4096, "dtype": "bf16", "residual": True},
        # a prompt's activations on their way into an 8-bit product, the stream kept beside them
        {"name": "norm8 prompt", "op": "norm8", "rows": 8192, "dim": 8192, "dtype": "bf16", "residual": True},
        # a width that no vector load divides, without a residual (the norm before the last product)
        {"name": "norm odd width", "op": "norm", "rows": 777, "dim": 2047, "dtype": "f16", "residual": False},
        # a training step of a block's norm: 16384 tokens, forward and backward
        {"name": "norm train", "op": "norm_train", "rows": 16384, "dim": 4096, "dtype": "bf16", "residual": True},
        # the same at the factorization's own order and type
        {"name": "norm train f32", "op": "norm_train", "rows": 1536, "dim": 512, "dtype": "f32", "residual": True},
        # one token through a square projection added to the stream
        {"name": "linear one token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "act": "none", "bias": True, "residual": True},
        # sixteen sequences decoding together, weights and activations in 8 bits
        {"name": "linear8 sixteen tokens", "op": "linear8", "m": 16, "n": 8192, "k": 8192, "act": "silu", "bias": False, "residual": False},
        # a prompt through the widening product of a feed-forward block
        {"name": "linear prompt", "op": "linear", "m": 4096, "n": 16384, "k": 4096, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False},
        # a prompt through an 8-bit projection added to the stream
        {"name": "linear8 prompt", "op": "linear8", "m": 8192, "n": 8192, "k": 4096, "act": "none", "bias": True, "residual": True},
        # sizes that fill no tile and rows that start off any 16-byte boundary
        {"name": "linear ragged", "op": "linear", "m": 1000, "n": 1001, "k": 513, "dtype": "f16", "act": "relu", "bias": True, "residual": True},
        # a training step of the widening product: the result and all gradients
        {"name": "linear train", "op": "linear_train", "m": 8192, "n": 8192, "k": 2048, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False},
        # a small layer trained on many tokens: the weight's gradient has few outputs and a long sum
        {"name": "linear train small", "op": "linear_train", "m": 4100, "n": 512, "k": 512, "dtype": "bf16", "act": "silu", "bias": True, "residual": True},
    ]


def _size(rng, lo, hi, odd):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if not odd and v >= 128:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "norm8", "norm_train", "linear", "linear8", "linear_train"])
    odd = rng.random() < 0.35
    if op.startswith("norm"):
        dim = _size(rng, 64, 16384, odd)
        rows = _size(rng, 64 if op == "norm_train" else 1, min(16384, (1 << 26) // dim), True)
        return {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "residual": rng.random() < 0.7}
    cap = 1 << (37 if op == "linear_train" else 38)
    n, k = _size(rng, 64, 16384, odd), _size(rng, 64, 16384, odd)
    m = _size(rng, 64 if op == "linear_train" else 1, max(64, min(8192, cap // (n * k))), rng.random() < 0.5)
    case = {"op": op, "m": m, "n": n, "k": k, "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
            "bias": rng.random() < 0.6, "residual": rng.random() < 0.5}
    if op != "linear8":
        case["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    return case


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rows_to_8(y):
    """Rows of ``y`` (float32) in 8 bits with a scale each."""
    scale = (y.abs().amax(-1) / _FP8_MAX).clamp_min(_TINY)
    return (y / scale[:, None]).to(_FP8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    dtype = _DTYPES[case.get("dtype", "bf16")]
    if case["op"].startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        # activations: a few channels are much larger than the others
        gain = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 12.0, 1.0)
        s["x"] = (_randn(g, rows, dim) * gain).to(dtype)
        s["residual"] = (2 * _randn(g, rows, dim) * gain).to(dtype) if case["residual"] else None
        s["weight"] = (1 + 0.2 * _randn(g, dim)).to(dtype)
        if case["op"] == "norm_train":
            s["dy"] = _randn(g, rows, dim).to(dtype)
            s["dh"] = _randn(g, rows, dim).to(dtype) if case["residual"] else None
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x, w = _randn(g, m, k), _randn(g, n, k) / math.sqrt(k)
        if case["op"] == "linear8":
            s["x"], s["x_scale"] = _rows_to_8(x)
            s["w"], s["w_scale"] = _rows_to_8(w)
        else:
            s["x"], s["w"] = x.to(dtype), w.to(dtype)
        s["bias"] = (0.3 * _randn(g, n)).to(dtype) if case["bias"] else None
        s["residual"] = _randn(g, m, n).to(dtype) if case["residual"] else None
        if case["op"] == "linear_train":
            s["dy"] = _randn(g, m, n).to(dtype)
    if case["op"].endswith("train"):  # the leaves whose gradients a training step asks for
        s["leaves"] = [s[p].requires_grad_() for p in ("x", "weight", "w", "bias") if s.get(p) is not None]
        if case["op"] == "norm_train" and case["residual"]:
            s["leaves"].append(s["residual"].requires_grad_())
    return s


# ---- the plain form: 32 bits, rounded once at the end -----------------------------------------

def _act(z, name):
    if name == "relu":
        return torch.clamp_min(z, 0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_norm(s):
    case, x = s["case"], s["x"].detach()
    dtype = x.dtype
    # the stream's sum is an output of its own, rounded once; the norm is the norm of what is kept
    h = x if s["residual"] is None else (x.float() + s["residual"].detach().float()).to(dtype)
    hf, w = h.float(), s["weight"].detach().float()
    r = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + _EPS)
    y = hf * r * w
    out = {"h": None if s["residual"] is None else h}
    if case["op"] == "norm8":
        out["y"], out["scale"] = _rows_to_8(y)
        return out
    out["y"] = y.to(dtype)
    if case["op"] == "norm_train":
        dy = s["dy"].float()
        gw = dy * w
        dx = r * gw - hf * (r * r * r * (gw * hf).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dtype)
        out["dresidual"] = None if s["residual"] is None else out["dx"]
        out["dweight"] = (dy * hf * r).sum(0).to(dtype)
    return out


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    dtype = torch.bfloat16 if case["op"] == "linear8" else s["x"].dtype
    if case["op"] == "linear8":
        x, w = x * s["x_scale"][:, None], w * s["w_scale"][:, None]
    z = x @ w.T
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["op"] == "linear_train":
        dz = s["dy"].float() * _act_grad(z, case["act"])
        out["dx"] = (dz @ w).to(dtype)
        out["dweight"] = (dz.T @ x).to(dtype)
        out["dbias"] = None if s["bias"] is None else dz.sum(0).to(dtype)
    return out


# ---- the library's calls ---------------------------------------------------------------------

_loaded = None


def _library():
    global _loaded
    if _loaded is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "qr-contest_b200"))
        import qrb200
        _loaded = qrb200
    return _loaded


def _own_norm(s):
    case, q = s["case"], _library()
    if case["op"] == "norm8":
        got = q.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS, out_dtype=_FP8)
        return {"y": got[0], "scale": got[1], "h": got[2] if s["residual"] is not None else None}
    got = q.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
    y, h = got if s["residual"] is not None else (got, None)
    out = {"y": y, "h": h}
    if case["op"] == "norm_train":
        heads, grads = ((y, h), (s["dy"], s["dh"])) if h is not None else ((y,), (s["dy"],))
        d = torch.autograd.grad(heads, s["leaves"], grads)
        out = {"y": y.detach(), "h": None if h is None else h.detach(), "dx": d[0], "dweight": d[1],
               "dresidual": d[2] if h is not None else None}
    return out


def _own_linear(s):
    case, q = s["case"], _library()
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "linear8":
        return {"y": q.linear(s["x"], s["w"], s["bias"], activation=act, residual=s["residual"],
                              x_scale=s["x_scale"], weight_scale=s["w_scale"])}
    y = q.linear(s["x"], s["w"], s["bias"], activation=act, residual=s["residual"])
    if case["op"] == "linear":
        return {"y": y}
    d = torch.autograd.grad(y, s["leaves"], s["dy"])
    return {"y": y.detach(), "dx": d[0], "dweight": d[1], "dbias": d[2] if s["bias"] is not None else None}


def run(state):
    norm = state["case"]["op"].startswith("norm")
    if own:
        return _own_norm(state) if norm else _own_linear(state)
    return _plain_norm(state) if norm else _plain_linear(state)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    e = {"bf16": 2, "f16": 2, "f32": 4}[case.get("dtype", "bf16")]
    if case["op"].startswith("norm"):
        rows, dim, res = case["rows"], case["dim"], case["residual"]
        size = rows * dim
        by = size * e * (1 + 2 * res) + dim * e  # x, residual and stream, weight
        if case["op"] == "norm8":
            by += size + rows * 4
        elif case["op"] == "norm":
            by += size * e
        else:  # y, dy, dx; dh; dweight
            by += size * e * (3 + res) + dim * e
        return {"bytes": by, "flops": size * (16 if case["op"] == "norm_train" else 6)}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "linear8":
        by = m * k + n * k + 4 * (m + n)
    else:
        by = (m * k + n * k) * e
    by += e * (n * case["bias"] + m * n * (1 + case["residual"]))
    if case["op"] == "linear_train":  # dy; dx, dweight, dbias
        by += e * (m * n + m * k + n * k + n * case["bias"])
        return {"bytes": by, "flops": 6 * m * n * k}
    return {"bytes": by, "flops": 2 * m * n * k}


# ---- the operators' definitions in 64 bits -----------------------------------------------------

def _f64(t):
    return None if t is None else t.detach().to(torch.float64)


def _exact_norm(s):
    case, dim, dtype = s["case"], s["x"].shape[-1], s["x"].dtype
    x, w, res = _f64(s["x"]), _f64(s["weight"]), _f64(s["residual"])
    total = x if res is None else x + res
    kept = total if res is None else total.to(dtype).to(torch.float64)  # the stream as it is kept
    inv = 1.0 / torch.sqrt(torch.einsum("ij,ij->i", kept, kept) / dim + _EPS)
    unit = kept * inv[:, None]
    y = torch.einsum("ij,j->ij", unit, w)
    out = {"y": y, "h": None if res is None else total}
    if case["op"] == "norm8":
        top = torch.linalg.vector_norm(y, ord=float("inf"), dim=-1)
        out["scale"] = torch.clamp(top / _FP8_MAX, min=_TINY)
        out["y"] = y / out["scale"][:, None]
    elif case["op"] == "norm_train":
        dy = _f64(s["dy"])
        dunit = torch.einsum("ij,j->ij", dy, w)
        along = torch.einsum("ij,ij->i", dunit, unit) / dim
        dx = (dunit - unit * along[:, None]) * inv[:, None]
        if s["dh"] is not None:
            dx = dx + _f64(s["dh"])
        out["dx"] = dx
        out["dresidual"] = None if res is None else dx
        out["dweight"] = torch.einsum("ij,ij->j", dy, unit)
    return out


def _exact_linear(s):
    case = s["case"]
    x, w = _f64(s["x"]), _f64(s["w"])
    z = torch.einsum("ik,jk->ij", x, w)
    if case["op"] == "linear8":
        z = z * torch.outer(_f64(s["x_scale"]), _f64(s["w_scale"]))
    if s["bias"] is not None:
        z = z + _f64(s["bias"])
    normal = torch.distributions.Normal(torch.zeros((), dtype=z.dtype, device=z.device), 1.0)
    c, a = math.sqrt(2 / math.pi), 0.044715
    if case["act"] == "gelu":
        phi = torch.special.ndtr(z)
        y, slope = z * phi, phi + z * torch.exp(normal.log_prob(z))
    elif case["act"] == "gelu_tanh":  # (1 + tanh u) / 2 = sigmoid(2u)
        p = torch.sigmoid(2 * c * z * (1 + a * z ** 2))
        y, slope = z * p, p + z * p * (1 - p) * 2 * c * (1 + 3 * a * z ** 2)
    elif case["act"] == "silu":
        p = torch.sigmoid(z)
        y, slope = z * p, p + z * p * (1 - p)
    elif case["act"] == "relu":
        y, slope = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).to(z.dtype)
    else:
        y, slope = z, None
    if s["residual"] is not None:
        y = y + _f64(s["residual"])
    out = {"y": y}
    if case["op"] == "linear_train":
        dz = _f64(s["dy"]) if slope is None else _f64(s["dy"]) * slope
        out["dx"] = torch.einsum("ij,jk->ik", dz, w)
        out["dweight"] = torch.einsum("ij,ik->jk", dz, x)
        out["dbias"] = None if s["bias"] is None else torch.einsum("ij->j", dz)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"].startswith("norm") else _exact_linear(s)
