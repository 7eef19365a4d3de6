"""The operators for matrix-shaped parameters in plain 64-bit torch on the CPU, and tolerances for
them from a model of how the kernels round.

The kernels' products read operands of 22 significant bits and drop the smallest of four partial
products: two relative errors of 2^-22 at most per factor.  The float32 sums add theirs (2^-24 a
step of a walk, so less than one more 2^-22 at these lengths).  `tolerance` runs the plain form
again with every factor off by a random relative error of up to 2^-20 -- bfloat16's last two steps,
whose operands may carry 11 bits, by up to 2^-10 -- three times, takes the largest deviation from
the exact run and allows four times that.  (The errors that are modelled are twice what the
kernels may commit, the factor covers three draws standing for all.)  The result's own rounding
comes on top: half a step of its type, eps / 2 relative, and half of the smallest subnormal.
"""

from __future__ import annotations

import math

import torch

COEFFICIENTS = (3.4445, -4.775, 2.0315)
BLOCK = 128


class Exact:
    def __call__(self, x, coarse=False):
        return x


class Noisy:
    """Every factor with a random relative error."""

    def __init__(self, seed, dtype):
        self.gen = torch.Generator().manual_seed(seed)
        self.half = dtype == torch.bfloat16

    def __call__(self, x, coarse=False):
        u = 2.0 ** -10 if coarse and self.half else 2.0 ** -20
        return x * (1.0 + u * (2.0 * torch.rand(x.shape, generator=self.gen, dtype=x.dtype) - 1.0))


def _wide(g):
    return g.mT if g.shape[-2] > g.shape[-1] else g


def iterates(g, steps, coefficients, eps, r=Exact()):
    """Every iterate of the wide 64-bit matrix `g`."""
    a, b, c = coefficients
    xs = [r(g) / (g.square().sum().sqrt() + eps)]
    for k in range(steps):
        coarse, x = k >= steps - 2, xs[-1]
        s = r(x, coarse) @ r(x, coarse).mT
        p = b * s + c * (r(s, coarse) @ r(s, coarse))
        # one factor holds the diagonal, as large as it is
        p = r(p + a * torch.eye(len(p), dtype=p.dtype), coarse)
        xs.append(p @ r(x, coarse))
    return xs


def orthogonalize(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, r=Exact()):
    out = iterates(_wide(g), steps, coefficients, eps, r)[-1]
    return out.mT if g.shape[-2] > g.shape[-1] else out


def gradient(g, dy, steps=5, coefficients=COEFFICIENTS, eps=1e-7, r=Exact()):
    """With S = X X^T, P = b S + c S^2 and the cotangent Y of a X + P X, M = Y X^T + X Y^T and
    N = b M + c (M S + S M) give a Y + P Y + N X for X.  (All operands in 22 bits.)"""
    a, b, c = coefficients
    w, y = _wide(g), _wide(dy)
    fine = lambda x, coarse=False: r(x)  # noqa: E731
    for x in reversed(iterates(w, steps, coefficients, eps, fine)[:-1]):
        s = r(x) @ r(x).mT
        p = r(b * s + c * (r(s) @ r(s)) + a * torch.eye(len(s), dtype=s.dtype))
        z = r(y) @ r(x).mT
        m = z + z.mT
        ms = r(m) @ r(s)
        n = b * m + c * (ms + ms.mT)
        y = p @ r(y) + r(n) @ r(x)
    size = w.square().sum().sqrt()
    along = (y * w).sum() / (size * (size + eps)).clamp_min(1e-300)
    dx = (y - w * along) / (size + eps)
    return dx.mT if g.shape[-2] > g.shape[-1] else dx


def tolerance(fn, *args, dtype, **kw):
    """``(exact result, allowed deviation in the Frobenius norm)`` before the result's rounding."""
    exact = fn(*args, **kw)
    worst = max(float((fn(*args, **kw, r=Noisy(seed, dtype)) - exact).norm()) for seed in (1, 2, 3))
    return exact, 4.0 * worst


def assert_close(got, exact, allowed, what='', spread=False):
    """`got` against `exact` in the Frobenius norm; with `spread` (inputs whose deviations spread
    evenly over the elements) also one by one: eight times the mean square allows the largest of
    10^6 normal ones, and an element that is read or written in a wrong place shows."""
    fi = torch.finfo(got.dtype)
    half = fi.eps / 2 * exact.abs() + fi.smallest_normal * fi.eps / 2
    diff = (got.detach().double().cpu() - exact).abs()
    assert bool(torch.isfinite(diff).all()), what
    off = float((diff - half).clamp_min(0.0).norm())
    assert off <= allowed, f'{what}: off by {off:.3g} beyond rounding, {allowed:.3g} allowed'
    if spread and exact.numel() > 64:
        worst, each = float((diff - half).max()), 8.0 * allowed / math.sqrt(exact.numel())
        assert worst <= each, f'{what}: an element off by {worst:.3g}, {each:.3g} allowed'


def quantize(x):
    """``(codes, scales, values)`` of the 64-bit vector `x`."""
    n = x.numel()
    p = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    scales = (p.abs().amax(1) / 127.0).float()
    wide = scales.double()[:, None]
    codes = torch.where(wide > 0.0, (p / wide).round(), 0.0)
    return codes.view(-1)[:n], scales, (codes * wide).view(-1)[:n]


def rate(rows, cols, adjust):
    if adjust in (None, 'original'):
        return math.sqrt(max(1.0, rows / cols))
    return 0.2 * math.sqrt(max(rows, cols)) if adjust == 'match_rms_adamw' else 1.0
