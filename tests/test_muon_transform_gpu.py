"""`scale_by_muon` out of place on 16-bit leaves is what it is in place: the momentum bit for bit, the update
the 64-bit form's of that momentum, rounded once."""

from __future__ import annotations

import pytest
import torch

import muon_plain as plain
from test_muon_precision_gpu import rounded_once
from torchopt_amd import muon, orthogonalize
from torchopt_amd.transform import scale_by_muon

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SHAPES = [(40, 60), (16, 3, 3, 3), (100, 130)]


def randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('momentum', [0.95, 0.9])
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_out_of_place_is_in_place(dtype, momentum, nesterov):
    t = scale_by_muon(momentum=momentum, nesterov=nesterov, adjust_lr_fn='none')
    ps = [randn(*s, dtype=dtype).cuda() for s in SHAPES]
    inner, outer = t.init(ps), t.init(ps)
    for n in range(4):
        gs = [randn(*s, dtype=dtype, seed=10 * n + k) for k, s in enumerate(SHAPES)]
        mine, inner = t.update([g.cuda() for g in gs], inner)
        fresh, outer = t.update([g.cuda().requires_grad_() for g in gs], outer, inplace=False)
        for k, g in enumerate(gs):
            m = inner.momentum[k]
            assert outer.momentum[k].dtype == fresh[k].dtype == dtype
            assert torch.equal(m, outer.momentum[k]), f'step {n}, leaf {k}'
            m = m.double().cpu()
            u = (g.double() + momentum * m if nesterov else m).flatten(1)
            exact, allowed = plain.tolerance(plain.orthogonalize, u, dtype=F32)
            rounded_once(mine[k].flatten(1), exact, allowed, f'in place, step {n}, leaf {k}')
            rounded_once(fresh[k].detach().flatten(1), exact, allowed, f'out of place, step {n}, leaf {k}')


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_gradient_through_the_sums(dtype):
    """Of <d, update> with respect to gradient and momentum: 1 + mu and mu (1 + ...) times the series' own
    gradient, which is formed from the look-ahead in 32 bits and rounded to the type at the leaves."""
    g, m, d = (randn(40, 70, dtype=dtype, seed=k) for k in (1, 2, 3))
    t = scale_by_muon(momentum=0.5, adjust_lr_fn='none')
    leaves = g.cuda().requires_grad_(), m.cuda().requires_grad_()
    state = t.init([g.cuda()])._replace(momentum=[leaves[1]])
    (u,), state = t.update([leaves[0]], state, inplace=False)
    got = torch.autograd.grad(u, leaves, d.cuda())
    kept = (0.5 * m.double() + g.double()).to(dtype).double()
    series, allowed = plain.tolerance(plain.gradient, g.double() + 0.5 * kept, d.double(), dtype=F32)
    # (to the momentum it passes through the kept sum, whose cotangent is rounded to its type as well:
    # half of the series' gradient, off by half a step)
    half = torch.finfo(dtype).eps / 2
    for mine, factor in zip(got, (1.5, 0.25)):
        exact = factor * series
        off = (mine.double().cpu() - exact).norm()
        assert mine.dtype == dtype
        assert float(off) <= 3.0 * half * float(exact.norm()) + 2.0 * allowed


def test_float32_gradients_of_16_bit_parameters_keep_a_float32_momentum():
    """Where gradients are wider than the kept momentum, the sum is theirs."""
    g = randn(20, 30, seed=1).cuda()
    t = scale_by_muon()
    (u,), state = t.update([g], t.init([g.to(BF16)]), inplace=False)
    assert u.dtype == F32 and state.momentum[0].dtype == F32
    assert torch.equal(u, orthogonalize(g + 0.95 * g))


def test_functional_chain_in_and_out_of_place():
    ps = [randn(40, 60, dtype=BF16, seed=1).cuda(), randn(60, seed=2).cuda()]
    gs = [randn(40, 60, dtype=BF16, seed=3).cuda(), randn(60, seed=4).cuda()]
    both = muon(0.1, weight_decay=0.0)
    a, s = both.update([g.clone() for g in gs], both.init(ps), params=ps)
    b, r = both.update(gs, both.init(ps), params=ps, inplace=False)
    assert torch.equal(s[1].matrices.momentum[0], r[1].matrices.momentum[0])
    # The two series differ by 22-bit arithmetic (twice what one may be off, eight times its mean for a
    # single element, times the rate), so their roundings may be neighbours, a step of 2^-7 at most
    # apart; the product with the rate then rounds each by another 2^-8.  Together 2^-6.
    _, allowed = plain.tolerance(plain.orthogonalize, 1.95 * gs[0].double().cpu(), dtype=F32)
    each = 0.1 * 16.0 * allowed / gs[0].numel() ** 0.5
    assert ((a[0].float() - b[0].float()).abs() <= 2.0 ** -6 * a[0].float().abs() + each).all()
    assert torch.equal(a[1], b[1])
