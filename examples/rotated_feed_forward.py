"""A feed-forward block in a rotated basis: factorization, norm and products together.

    python examples/rotated_feed_forward.py [--width 512] [--hidden 2048] [--tokens 300]

The block reads a stream h = x + r and returns h + W2 gelu(W1 rms(h) + b1).  With an orthogonal Q (the
explicit factor of a batched QR) the stream can be kept as hQ: a root-mean-square norm without a weight
commutes with Q, so Q goes into the weights on both sides (W1 Q and Q^T W2; the norm's weight goes into W1
first) and the block computes the same thing while no single channel of its activations stands out.  That is
the form that is then served in 8 bits:

    rms_norm(residual, 8 bits) -> linear(8 bits, gelu) -> quantize_rows -> linear(8 bits, residual)

The same block in 16 bits is trained for a few steps through the operators' gradients.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qr-contest_b200"))
import qrb200  # noqa: E402

FP8 = torch.float8_e4m3fn


def orthogonal(n, seed=0):
    """A random orthogonal n x n matrix: the Q of a Gaussian one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    _, _, Q, info = qrb200.geqrf_q(torch.randn(1, n, n, generator=g, device="cuda"))
    qrb200.api.raise_on_info(info)
    return Q[0]


def block(width, hidden, seed=1):
    """Float32 weights of the block: the norm's weight, W1, b1, W2."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return 1 + 0.2 * rnd(width), rnd(hidden, width) * width ** -0.5, 0.1 * rnd(hidden), rnd(width, hidden) * hidden ** -0.5


def rotated(weights, Q):
    gain, W1, b1, W2 = weights
    return (W1 * gain) @ Q, b1, Q.T @ W2


def plain64(weights, x, r):
    """The block in float64, from its definition."""
    gain, W1, b1, W2 = (w.double() for w in weights)
    h = x.double() + r.double()
    n = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain
    z = n @ W1.T + b1
    return h + 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5)) @ W2.T


class Served:
    """The rotated block in 8 bits; its weights are laid out once."""

    def __init__(self, weights, Q):
        W1, b1, W2 = rotated(weights, Q)
        self.w1, self.s1 = qrb200.quantize_rows(W1)
        self.w2, self.s2 = qrb200.quantize_rows(W2.contiguous())
        self.b1 = b1.bfloat16()

    def __call__(self, x, r):
        """x and r in the rotated basis -> the stream after the block, in the rotated basis."""
        y, s, h = qrb200.rms_norm(x, residual=r, out_dtype=FP8)
        u = qrb200.linear(y, self.w1, self.b1, activation="gelu", x_scale=s, weight_scale=self.s1)
        u, s = qrb200.quantize_rows(u)
        return qrb200.linear(u, self.w2, residual=h, x_scale=s, weight_scale=self.s2)


class Trained(torch.nn.Module):
    """The block in 16 bits."""

    def __init__(self, weights):
        super().__init__()
        self.gain, self.w1, self.b1, self.w2 = (torch.nn.Parameter(w.bfloat16()) for w in weights)

    def forward(self, x, r):
        n, h = qrb200.rms_norm(x, self.gain, residual=r)
        return qrb200.linear(qrb200.linear(n, self.w1, self.b1, activation="gelu"), self.w2, residual=h)


def main(width=512, hidden=2048, tokens=300, steps=5, report=print):
    Q, weights = orthogonal(width), block(width, hidden)
    g = torch.Generator(device="cuda").manual_seed(2)
    loud = torch.where(torch.rand(width, generator=g, device="cuda") < 0.02, 12.0, 1.0)  # a few loud channels
    x, r = (torch.randn(tokens, width, generator=g, device="cuda") * loud for _ in range(2))
    want = plain64(weights, x, r)
    off = lambda y: float((y.double() - want).norm() / want.norm())  # noqa: E731

    served = Served(weights, Q)
    xr, rr = (x @ Q).bfloat16(), (r @ Q).bfloat16()
    eight = off(served(xr, rr).float() @ Q.T)
    report(f"8 bits, rotated:  {eight:.2e} off the float64 block")
    one = served(xr[:1], rr[:1])
    single = float((one.float() @ Q.T - want[:1].float()).norm() / want[:1].norm())
    report(f"  a single token: {single:.2e}")

    model = Trained(weights)
    sixteen = off(model(x.bfloat16(), r.bfloat16()).detach())
    report(f"16 bits:          {sixteen:.2e} off the float64 block")
    target = want.bfloat16().roll(1, 0).float()
    opt = torch.optim.Adam(model.parameters(), lr=2e-3)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (model(x.bfloat16(), r.bfloat16()).float() - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    report("training loss:    " + "  ".join(f"{v:.4f}" for v in losses))
    return eight, single, sixteen, losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("width", 512), ("hidden", 2048), ("tokens", 300)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    main(a.width, a.hidden, a.tokens)
