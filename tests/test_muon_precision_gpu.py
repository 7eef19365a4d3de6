"""16-bit results of the orthogonalisation are the 64-bit form's, rounded once to their type.

For a result `z + e` that is rounded to the type, with `z` exact: each element ends no farther from
`z` than `|round(z) - z| + 2 |e|` (either both round to the same value, or `z` lies within `|e|` of a
border, and then `|round(z) - z|` is half a step less `|e|` at least).  So the whole deviation is at most
that of the rounded exact result and twice the norm of `e`, for which `plain.tolerance` gives what
operands of 22 bits and float32 sums may commit."""

from __future__ import annotations

import pytest
import torch

import muon_plain as plain
from torchopt_amd import orthogonalize
from torchopt_amd._C import muon_op

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# one workgroup; thin; tiles with steps one by one and by twos
SIZES = [(24, 60), (60, 200), (40, 1000), (128, 128), (200, 256), (260, 100), (100, 900), (512, 512)]


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def low_rank(m, n, rank):
    return randn(m, rank, seed=rank) @ randn(rank, n, seed=rank + 1)


def special(m, n):
    spread = torch.ones(m, n)
    spread[0, 0] = 1e4
    k = min(m, n)
    u, v = torch.linalg.qr(randn(m, k, seed=1))[0], torch.linalg.qr(randn(n, k, seed=2))[0]
    yield from ((f'rank {r}', low_rank(m, n, r)) for r in (1, 2, 3, 8))
    yield from [('identity', torch.eye(m, n)), ('ones', torch.ones(m, n)), ('one element', spread),
                ('decaying', u @ torch.diag(torch.arange(1.0, k + 1) ** -1.5) @ v.t()),
                ('full rank', randn(m, n, seed=3))]


def rounded_once(y, exact, allowed, what):
    rounding = float((exact.to(y.dtype).double() - exact).norm())
    off = float((y.double().cpu() - exact).norm())
    assert off <= rounding + 2.0 * allowed, \
        f'{what}: off by {off:.4g}; rounding alone {rounding:.4g}, arithmetic {allowed:.3g}'


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('m,n', SIZES)
def test_special_matrices_are_rounded_once(m, n, dtype):
    """The default coefficients, whose last steps magnify what is rounded before them: few large
    singular values among many small ones show it most."""
    for what, x in special(m, n):
        x = x.to(dtype)
        for steps in (5, 2, 1):
            exact, allowed = plain.tolerance(plain.orthogonalize, x.double(), dtype=F32, steps=steps)
            rounded_once(orthogonalize(x.cuda(), steps=steps), exact, allowed, f'{what}, {steps} steps')


@pytest.mark.parametrize('coefficients,steps', [((5.0, -10.0, 6.0), 2), ((3.0, -3.0, -0.1), 3),
                                                ((0.5, 1.0, 0.01), 3)])
def test_other_coefficients_are_rounded_once(coefficients, steps):
    kw = dict(steps=steps, coefficients=coefficients)
    for m, n in ((128, 128), (100, 900)):
        for rank in (1, 3, 8):
            x = low_rank(m, n, rank).to(BF16)
            exact, allowed = plain.tolerance(plain.orthogonalize, x.double(), dtype=F32, **kw)
            rounded_once(orthogonalize(x.cuda(), **kw), exact, allowed, f'{m} x {n}, rank {rank}')


@pytest.mark.parametrize('coefficients,steps', [((1.875, -1.25, 0.375), 5), ((1.875, -1.25, 0.375), 1),
                                                ((1.5, -0.5, 0.0), 6), ((2.0, -1.5, 0.5), 4),
                                                ((-1.5, 0.5, 0.0), 3)])
def test_gentle_coefficients_stay_near_one_rounding(coefficients, steps):
    """Series that converge may read the last step's operands in 11 bits, an eighth of bfloat16's
    rounding, where that stays below half a step.  Here they magnify it at most four times -- at singular
    value t by (|p'| + dP/dS |S + h I| + max |P|) / |P|, which is 3.1 at most for the quintics and 2.3 for
    the cubics -- which is half a rounding beside the result's own, independent of it, so sqrt(1.25) = 1.12
    times the result's alone.  A tenth more for few elements."""
    kw = dict(steps=steps, coefficients=coefficients)
    for m, n in ((128, 128), (100, 260), (512, 300), (3, 2000)):
        for rank in (1, 2, 3, 8, None):
            x = (low_rank(m, n, rank) if rank else randn(m, n, seed=5)).to(BF16)
            exact = plain.orthogonalize(x.double(), **kw)
            rounding = float((exact.to(BF16).double() - exact).norm())
            off = float((orthogonalize(x.cuda(), **kw).double().cpu() - exact).norm())
            assert off <= 1.23 * rounding, f'{m} x {n}, rank {rank}: {off / rounding:.3f}'


def test_step_of_low_rank_gradients_is_rounded_once():
    for m, n in ((128, 128), (260, 100), (512, 512)):
        gs = [low_rank(m, n, rank).to(BF16) for rank in (1, 3)]
        mine, kept = [g.cuda() for g in gs], [torch.zeros(m, n, dtype=BF16, device='cuda') for _ in gs]
        muon_op.forward_multi_(mine, kept, None, 0.0, nesterov=False, adjust_lr_fn='none')
        for g, y in zip(gs, mine):
            exact, allowed = plain.tolerance(plain.orthogonalize, g.double(), dtype=F32)
            rounded_once(y, exact, allowed, f'{m} x {n}')


def plain_float32(x, steps=5):
    """The definition in float32, on the CPU."""
    a, b, c = plain.COEFFICIENTS
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x


@pytest.mark.parametrize('m,n', [(1, 7), (1, 64), (2, 5), (7, 40), (8, 8), (16, 16), (16, 100), (24, 24), (32, 32),
                                 (33, 33), (32, 288), (64, 64), (64, 224)])
def test_float32_is_as_exact_as_plain_float32(m, n):
    """Operands of hi + lo are off by 5.2e-8 on average (half of all lo have an ulp of 2^-22, a quarter
    2^-23, ...), float32's by 3.4e-8, and the sums round alike: 1.53 times the plain form's error where
    the operands' rounding is all there is, over many matrices."""
    x = randn(64, m, n, seed=m + n)
    exact = torch.stack([plain.orthogonalize(g) for g in x.double()])
    off = float((orthogonalize(x.cuda()).double().cpu() - exact).norm())
    usual = float((plain_float32(x).double() - exact).norm())
    assert off <= 1.53 * usual, f'{m} x {n}: {off / usual:.2f}'


@pytest.mark.parametrize('m,n', [(100, 100), (128, 128), (100, 900), (200, 256), (512, 512)])
def test_gradients_at_rank_one(m, n):
    """Most of such a gradient is the cotangent times a in every step, and what is off in the multiple of
    the unit matrix in P is off everywhere.  A step's average errors, relative to a = 3.44: h + S_ii is
    rounded by 5.2e-8, which c (h + S)^2 makes 7.2e-8; P's diagonal by 5.2e-8; the cotangent by 5.2e-8 and
    in its sum by 3e-8 (6e-8): 1.1e-7 together; and lo lo, which is dropped, is c / a * 2^-22 / 3 = 4.7e-8 on
    the diagonal, always to one side.  1.6e-7 a step, if all of it adds up over the steps; 1.5 * 2^-23 are
    allowed."""
    x = low_rank(m, n, 1)
    dy = randn(m, n, seed=5)
    exact = plain.gradient(x.double(), dy.double())
    dx, = muon_op.orthogonalize_backward_multi([dy.cuda()], [x.cuda()])
    off = float((dx.double().cpu() - exact).norm() / exact.norm())
    assert off <= 5 * 1.5 * 2.0 ** -23, f'{off:.3g}'


def plain_float32_gradient(x, dy, steps=5):
    a, b, c = plain.COEFFICIENTS
    size = x.square().sum((1, 2), keepdim=True).sqrt()
    xs, g = [x / (size + 1e-7)], x
    for _ in range(steps - 1):
        s = xs[-1] @ xs[-1].mT
        xs.append(a * xs[-1] + (b * s + c * (s @ s)) @ xs[-1])
    y = dy
    for x in reversed(xs):
        s = x @ x.mT
        z = y @ x.mT
        m = z + z.mT
        ms = m @ s
        y = a * y + (b * s + c * (s @ s)) @ y + (b * m + c * (ms + ms.mT)) @ x
    along = (y * g).sum((1, 2), keepdim=True) / (size * (size + 1e-7))
    return (y - g * along) / (size + 1e-7)


@pytest.mark.parametrize('m,n', [(16, 16), (32, 288), (65, 65), (100, 100), (100, 300), (200, 256)])
def test_float32_gradients_are_as_exact_as_plain_float32(m, n):
    """As for the results: operands off by 1.53 times what float32's are, sums alike."""
    x, dy = randn(16, m, n, seed=m + n), randn(16, m, n, seed=m + n + 1)
    exact = torch.stack([plain.gradient(g, d) for g, d in zip(x.double(), dy.double())])
    dx, = muon_op.orthogonalize_backward_multi([dy.cuda()], [x.cuda()])
    off = float((dx.double().cpu() - exact).norm())
    usual = float((plain_float32_gradient(x, dy).double() - exact).norm())
    assert off <= 1.53 * usual, f'{m} x {n}: {off / usual:.2f}'
