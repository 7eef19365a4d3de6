"""The operators for matrix-shaped parameters on the GPU against plain 64-bit forms
(`muon_plain`, which also says where the tolerances come from)."""

from __future__ import annotations

import math

import pytest
import torch

import muon_plain as plain
import torchopt_amd
from torchopt_amd import dequantize_blocks, orthogonalize, quantize_blocks
from torchopt_amd._C import muon_op

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def randn(*shape, dtype=F32, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=gen)).to(dtype)


def check_forward(cpu, dtype, what='', spread=True, gpu=None, **kw):
    """One matrix; `gpu` where it lies in another way than `cpu.cuda()` does."""
    x = cpu.cuda() if gpu is None else gpu
    y = orthogonalize(x, **kw)
    assert y.dtype == dtype and y.shape == cpu.shape and y.is_contiguous()
    exact, allowed = plain.tolerance(plain.orthogonalize, cpu.double(), dtype=dtype, **kw)
    plain.assert_close(y, exact, allowed, what, spread)
    return y


# one workgroup takes up to 32 x 864 or 64 x 224; tiles are 64, 128 and 256 wide; a row's piece is
# 32 or 64 elements
SIZES = [(1, 1), (1, 2), (2, 1), (1, 33), (1, 1000), (1000, 1), (2, 3), (5, 5), (16, 16), (31, 32),
         (32, 32), (33, 32), (32, 864), (32, 865), (33, 224), (64, 224), (64, 225), (65, 64),
         (63, 223), (64, 64), (65, 65), (7, 129), (127, 128), (128, 128), (129, 127), (100, 900),
         (255, 256), (257, 256), (40, 2000), (300, 520), (513, 130)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n', SIZES)
def test_orthogonalize_sizes(m, n, dtype):
    check_forward(randn(m, n, dtype=dtype, seed=m * n), dtype, f'{m} x {n}')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n', [(1, 5000), (7, 3000), (32, 900), (33, 700), (63, 300), (64, 1111), (2000, 40)])
def test_thin_matrices(m, n, dtype):
    """Too wide for one workgroup, up to 64 rows: what lies between X's own products is one launch."""
    x = randn(3, m, n, dtype=dtype, seed=m + n)
    for kw in (dict(), dict(steps=4), dict(steps=3, coefficients=(1.5, -0.5, 0.0)),
               dict(steps=2, coefficients=(0.5, 1.0, 0.01))):
        y = orthogonalize(x.cuda(), **kw)
        for k in range(3):
            exact, allowed = plain.tolerance(plain.orthogonalize, x[k].double(), dtype=dtype, **kw)
            plain.assert_close(y[k], exact, allowed, str(kw), spread=m > 1)


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 6, 9])
@pytest.mark.parametrize('m,n', [(20, 50), (90, 400), (130, 140), (50, 700)])
def test_numbers_of_steps(m, n, steps):
    """(90 x 400 takes its steps in pairs and an odd one last.)"""
    for dtype in (F32, BF16):
        check_forward(randn(m, n, dtype=dtype, seed=steps), dtype, steps=steps)


@pytest.mark.parametrize('coefficients', [
    (1.5, -0.5, 0.0),           # a cubic: no square to complete
    (1.875, -1.25, 0.375),      # the convergent quintic
    (2.0, -1.5, 0.5),
    (0.5, 1.0, 0.01),           # b over c large: the other form of the polynomial
    (1.0, 0.0, 0.0),            # nothing but the normalisation
    (-1.5, 0.5, 0.0),
    (3.0, -3.0, -0.1),
    (0.0, 0.0, 0.0),
])
@pytest.mark.parametrize('m,n', [(30, 31), (70, 500), (150, 130)])
def test_coefficients(m, n, coefficients):
    x, dy = randn(m, n, seed=5), randn(m, n, seed=6)
    kw = dict(steps=3, coefficients=coefficients)
    check_forward(x, F32, str(coefficients), **kw)
    check_gradient(x, dy, F32, str(coefficients), **kw)


def test_eps_counts():
    check_forward(randn(20, 30, seed=1, scale=1e-3), F32, eps=0.5)
    check_forward(randn(100, 300, seed=1, scale=1e-3), F32, eps=0.5)
    check_forward(randn(100, 300, seed=1), F32, eps=0.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scale', [1e-30, 1e-4, 1e4, 1e30])
@pytest.mark.parametrize('m,n', [(20, 40), (90, 300)])
def test_magnitudes(m, n, scale, dtype):
    """Norms near the ends of the types' ranges: squares overflow or vanish in 32 bits."""
    if dtype == F16 and not 1e-5 < scale < 1e5:
        scale = 1e-6 if scale < 1.0 else 1e4
    x = randn(m, n, seed=3, scale=scale).to(dtype)
    check_forward(x, dtype, eps=0.0)


def low_rank(m, n, rank, seed=0):
    return randn(m, rank, seed=seed) @ randn(rank, n, seed=seed + 1)


@pytest.mark.parametrize('m,n', [(24, 60), (100, 260), (260, 100)])
def test_special_matrices(m, n):
    eye = torch.eye(m, n)
    spread = torch.ones(m, n)
    spread[0, 0] = 1e6      # one element that rules the norm
    uneven = randn(m, n, seed=9) * torch.logspace(0, -6, n)[None, :]
    for what, x in [('rank one', low_rank(m, n, 1)), ('rank three', low_rank(m, n, 3)),
                    ('identity', eye), ('ones', torch.ones(m, n)), ('one element', spread),
                    ('uneven columns', uneven), ('empty rows', randn(m, n) * (torch.arange(m) % 3 == 0)[:, None]),
                    ('empty columns', randn(m, n) * (torch.arange(n) % 2 == 0))]:
        y = check_forward(x, F32, what, spread=False)
        if what == 'empty columns':
            assert not y[:, 1::2].any()
        if what == 'empty rows':
            assert not y[1::3].any()


@pytest.mark.parametrize('dtype', TYPES)
def test_zero_and_not_finite(dtype):
    """A zero matrix stays zero (eps = 0 divides by zero and gives NaN, as the formula does), one
    with a NaN or an infinity becomes NaN, and its neighbours in the list see nothing of it."""
    for m, n in ((20, 30), (100, 300)):
        good = randn(m, n, dtype=dtype, seed=2).cuda()
        nan, inf = good.clone(), good.clone()
        nan[m // 2, 3], inf[0, n - 1] = float('nan'), float('-inf')
        zero = torch.zeros_like(good)
        alone = orthogonalize(good)
        out = orthogonalize([good, nan, zero, inf, good])
        assert torch.equal(out[0], alone) and torch.equal(out[4], alone)
        assert out[1].isnan().all() and out[3].isnan().all()
        assert not out[2].any()
        dx = muon_op.orthogonalize_backward_multi([good] * 5, [good, nan, zero, inf, good])
        assert torch.equal(dx[0], dx[4]) and dx[0].isfinite().all()
        assert dx[1].isnan().all() and dx[3].isnan().all()
        # at zero the map is G / eps times the slope: finite, and large
        if dtype == F32:
            exact = plain.COEFFICIENTS[0] ** 5 * good.double() / 1e-7
            assert ((dx[2].double() - exact).norm() / exact.norm()) < 1e-5


# ---- layouts ---------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n', [(30, 50), (70, 270), (270, 70), (129, 131)])
def test_layouts(m, n, dtype):
    """Strides, orders and alignments: all give what the dense matrix gives, bit for bit (the
    same arithmetic from other places), which is right by the other tests."""
    x = randn(m, n, dtype=dtype, seed=7).cuda()
    want = orthogonalize(x)
    turned = x.t().contiguous().t()
    padded = torch.full((m, n + 3), 7.0, dtype=dtype, device='cuda')[:, 1:n + 1].copy_(x)
    both = torch.full((2 * m, 3 * n), 7.0, dtype=dtype, device='cuda')[::2, ::3].copy_(x)
    odd = torch.empty(m * n + 1, dtype=dtype, device='cuda')[1:].view(m, n).copy_(x)
    for what, v in [('turned', turned), ('padded', padded), ('both', both), ('odd', odd)]:
        assert torch.equal(orthogonalize(v), want), what
    # the tall form of the same matrix is the same computation
    assert torch.equal(orthogonalize(x.t()), want.t())
    flipped = x.flip(1)
    check_forward(flipped.cpu(), dtype, gpu=flipped)
    # one row or one column for all
    row = randn(1, n, dtype=dtype, seed=8).cuda().expand(m, n)
    assert torch.equal(orthogonalize(row), orthogonalize(row.contiguous()))
    # the gradient takes every layout as well
    dy = randn(m, n, dtype=dtype, seed=9).cuda()
    dx, = muon_op.orthogonalize_backward_multi([dy], [x])
    for v in (turned, padded, both, odd):
        for w in (dy, dy.t().contiguous().t()):
            assert torch.equal(muon_op.orthogonalize_backward_multi([w], [v])[0], dx)
    g = torch.ones((), dtype=dtype, device='cuda').expand(m, n)
    assert torch.equal(muon_op.orthogonalize_backward_multi([g], [x])[0],
                       muon_op.orthogonalize_backward_multi([g.contiguous()], [x])[0])


def test_batches_and_lists():
    x = randn(2, 3, 40, 70, seed=1).cuda()
    y = orthogonalize(x)
    assert y.shape == x.shape
    for i in range(2):
        for j in range(3):
            assert torch.equal(y[i, j], orthogonalize(x[i, j]))
    t = x.permute(1, 0, 3, 2)
    assert torch.equal(orthogonalize(t), y.permute(1, 0, 3, 2))
    # more shapes than one launch takes, small and tiled ones mixed, types mixed, some empty
    sizes = [(3 + 5 * k, 200 + 7 * k) for k in range(25)] + [(0, 5), (5, 0), (90, 2), (2, 90)]
    many = [randn(m, n, dtype=TYPES[k % 3], seed=k).cuda() for k, (m, n) in enumerate(sizes)]
    for kind in (list, tuple):
        out = orthogonalize(kind(many))
        assert type(out) is kind
        for x, y in zip(many, out):
            assert y.dtype == x.dtype and y.shape == x.shape
            plain_y, allowed = plain.tolerance(plain.orthogonalize, x.double().cpu(), dtype=x.dtype) \
                if x.numel() else (x.double().cpu(), 0.0)
            plain.assert_close(y, plain_y, allowed, str(tuple(x.shape)))
    # many small ones
    lots = [randn(3, 4, seed=k).cuda() for k in range(300)]
    out = orthogonalize(lots)
    for k in (0, 24, 25, 150, 299):
        assert torch.equal(out[k], orthogonalize(lots[k]))
    batch = randn(5000, 2, 3, seed=4).cuda()  # more matrices than one set of records
    assert torch.equal(orthogonalize(batch)[4321], orthogonalize(batch[4321]))
    for empty in (torch.empty(0, 3, 4), torch.empty(3, 0, 4), torch.empty(2, 3, 0)):
        assert orthogonalize(empty.cuda()).shape == empty.shape


@pytest.mark.parametrize('count,m,n', [(8, 256, 1024), (3, 512, 512), (2, 700, 1500), (40, 128, 384),
                                       (1, 1024, 640)])
def test_larger_batches(count, m, n):
    """Larger tiles and their rules; the first and last matrix against the 64-bit form."""
    x = randn(count, m, n, seed=count).cuda()
    for dtype in TYPES:
        y = orthogonalize(x.to(dtype))
        for k in {0, count - 1}:
            exact, allowed = plain.tolerance(plain.orthogonalize, x[k].to(dtype).double().cpu(),
                                             dtype=dtype)
            plain.assert_close(y[k], exact, allowed, f'{dtype} {k}', spread=True)


@pytest.mark.parametrize('dtype', TYPES)
def test_small_ones_beside_larger_ones(dtype):
    """Few go through the larger ones' launches, many through their own."""
    for few in (3, 60):
        sizes = [(20, 30), (7, 129), (64, 100)] * (few // 3) + [(90, 400), (130, 65)]
        xs = [randn(*s, dtype=dtype, seed=k) for k, s in enumerate(sizes)]
        dys = [randn(*s, dtype=dtype, seed=k + 200) for k, s in enumerate(sizes)]
        leaves = [x.cuda().requires_grad_() for x in xs]
        ys = orthogonalize(leaves)
        grads = torch.autograd.grad(ys, leaves, [d.cuda() for d in dys])
        for k in sorted({0, 1, 2, len(xs) - 3, len(xs) - 2, len(xs) - 1}):
            exact, allowed = plain.tolerance(plain.orthogonalize, xs[k].double(), dtype=dtype)
            plain.assert_close(ys[k], exact, allowed, f'{few} {sizes[k]}')
            exact, allowed = plain.tolerance(plain.gradient, xs[k].double(), dys[k].double(), dtype=dtype)
            plain.assert_close(grads[k], exact, allowed, f'gradient {few} {sizes[k]}')


def test_the_same_call_gives_the_same_bits():
    x, dy = randn(4, 200, 700, seed=1).cuda(), randn(4, 200, 700, seed=2).cuda()
    s, ds = randn(9, 32, 288, seed=3).cuda(), randn(9, 32, 288, seed=4).cuda()
    y, dx = orthogonalize([x, s]), muon_op.orthogonalize_backward_multi([dy, ds], [x, s])
    for _ in range(3):
        assert all(map(torch.equal, orthogonalize([x, s]), y))
        assert all(map(torch.equal, muon_op.orthogonalize_backward_multi([dy, ds], [x, s]), dx))


# ---- the gradient ----------------------------------------------------------------------------


def check_gradient(x, dy, dtype, what='', **kw):
    leaf = x.cuda().requires_grad_()
    y = orthogonalize(leaf, **kw)
    y.backward(dy.cuda())
    assert leaf.grad.dtype == dtype and leaf.grad.shape == x.shape
    exact, allowed = plain.tolerance(plain.gradient, x.double(), dy.double(), dtype=dtype, **kw)
    plain.assert_close(leaf.grad, exact, allowed, what, spread=True)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n', [(1, 2), (2, 2), (5, 3), (31, 33), (32, 288), (32, 865), (64, 224),
                                 (65, 225), (7, 129), (127, 129), (200, 90), (128, 600), (300, 520)])
def test_gradient_sizes(m, n, dtype):
    check_gradient(randn(m, n, dtype=dtype, seed=m), randn(m, n, dtype=dtype, seed=n + 1000), dtype,
                   f'{m} x {n}')


@pytest.mark.parametrize('steps', [1, 2, 4, 7])
def test_gradient_steps(steps):
    for m, n in ((20, 50), (90, 400)):
        check_gradient(randn(m, n, seed=1), randn(m, n, seed=2), F32, steps=steps)
        check_gradient(randn(m, n, seed=1, scale=1e-3), randn(m, n, seed=2), F32, steps=steps,
                       eps=0.25)


@pytest.mark.parametrize('steps,coefficients', [
    (8, plain.COEFFICIENTS), (12, plain.COEFFICIENTS), (20, plain.COEFFICIENTS), (32, (1.5, -0.5, 0.0)),
    (16, (2.0, -1.5, 0.5)), (3, (5.0, -6.0, 2.0))])
@pytest.mark.parametrize('m,n', [(5, 9), (20, 50), (70, 300)])
def test_gradient_of_long_series(m, n, steps, coefficients):
    """The slopes' product runs far ahead of what a cotangent really grows by."""
    for rank in (None, 3):
        x = randn(m, n, seed=1) if rank is None else low_rank(m, n, rank) + 0.05 * randn(m, n, seed=4)
        check_gradient(x, randn(m, n, seed=2), F32, f'rank {rank}', steps=steps,
                       coefficients=coefficients)
    # a cotangent of zeros, and one of a NaN, among others
    x = [randn(m, n, seed=k).cuda() for k in range(3)]
    dy = [torch.zeros_like(x[0]), torch.full_like(x[1], float('nan')), randn(m, n, seed=7).cuda()]
    kw = dict(steps=steps, coefficients=coefficients)
    dx = muon_op.orthogonalize_backward_multi(dy, x, **kw)
    assert not dx[0].any() and dx[1].isnan().all()
    assert torch.equal(dx[2], muon_op.orthogonalize_backward_multi(dy[2:], x[2:], **kw)[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_kept_iterates_give_the_same_gradient(dtype):
    """The gradient from kept iterates is that from iterates made again, bit for bit (both take every
    step by itself with 22-bit operands); the buffer is only read, and serves as often as asked."""
    shapes = [(90, 400), (20, 30), (300, 130), (90, 400), (65, 65), (0, 5)]
    for kw in (dict(steps=9), dict(steps=1), dict(steps=4, coefficients=(1.5, -0.5, 0.0)), dict()):
        xs = [randn(*s, dtype=dtype, seed=k).cuda() for k, s in enumerate(shapes)]
        dys = [randn(*s, dtype=dtype, seed=k + 20).cuda() for k, s in enumerate(shapes)]
        ys, kept = muon_op.orthogonalize_keep_multi(xs, 1 << 30, **kw)
        assert kept is not None
        before = kept.clone()
        want = muon_op.orthogonalize_backward_multi(dys, xs, **kw)
        for _ in range(2):
            got = muon_op.orthogonalize_backward_multi(dys, xs, **kw, kept=kept)
            assert all(map(torch.equal, got, want))
        assert torch.equal(kept, before)
        for x, y in zip(xs, ys):
            if x.numel():
                exact, allowed = plain.tolerance(plain.orthogonalize, x.double().cpu(), dtype=F32, **kw)
                plain.assert_close(y, exact, allowed)
    assert muon_op.orthogonalize_keep_multi(xs, kept.numel() - 1, **kw)[1] is None
    assert muon_op.orthogonalize_keep_multi(xs[1:2], 1 << 30)[1] is None
    for bad in (kept[:-256], kept.float(), kept.cpu()):
        with pytest.raises(RuntimeError, match='not what the forward pass kept'):
            muon_op.orthogonalize_backward_multi(dys, xs, **kw, kept=bad)
    with pytest.raises(RuntimeError, match='not what the forward pass kept'):
        muon_op.orthogonalize_backward_multi(dys[:1], xs[:1], **kw, kept=kept)


@pytest.mark.parametrize('each', [1, 2])
def test_gradients_of_many_shapes(each):
    """More shapes than one launch takes, in few matrices and in more than come with a launch's
    arguments; kept and made again."""
    shapes = [(40 + 9 * k, 230 + 13 * k) for k in range(20)]
    xs = [randn(each, *s, seed=k).cuda() for k, s in enumerate(shapes)]
    dys = [randn(each, *s, seed=k + 50).cuda() for k, s in enumerate(shapes)]
    _, kept = muon_op.orthogonalize_keep_multi(xs, 1 << 30)
    got = muon_op.orthogonalize_backward_multi(dys, xs, kept=kept)
    assert all(map(torch.equal, got, muon_op.orthogonalize_backward_multi(dys, xs)))
    for k in (0, 7, 15, 16, 19):
        exact, allowed = plain.tolerance(plain.gradient, xs[k][-1].double().cpu(),
                                         dys[k][-1].double().cpu(), dtype=F32)
        plain.assert_close(got[k][-1], exact, allowed, str(shapes[k]), spread=True)


@pytest.mark.parametrize('m,n', [(20, 40), (90, 300)])
@pytest.mark.parametrize('of_x,of_dy', [(1e-10, 1e-20), (1e20, 1e25), (1e-20, 1e-25), (1.0, 1e30),
                                        (1.0, 1e-30)])
def test_gradient_magnitudes(m, n, of_x, of_dy):
    check_gradient(randn(m, n, seed=1, scale=of_x), randn(m, n, seed=2, scale=of_dy), F32, eps=0.0)


def test_a_matrix_beyond_32_bits():
    """1100 x 2^20 in float16: its operand has 4.8 GB.  (Reference on the GPU in 64 bits; both
    steps of two are half-step roundings of float16 apart.)"""
    m, n = 1100, 1 << 20
    gen = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(m, n, generator=gen, device='cuda', dtype=torch.float16)
    y = orthogonalize(x, steps=2)
    w = x.double()
    w /= w.square().sum().sqrt() + 1e-7
    a, b, c = plain.COEFFICIENTS
    for _ in range(2):
        s = w @ w.t()
        w = (b * s + c * (s @ s) + a * torch.eye(m, device='cuda', dtype=torch.float64)) @ w
    # rows of the operands at both ends and in the middle, whole columns too
    half = torch.finfo(torch.float16)
    for at in (slice(0, 40), slice(540, 560), slice(1060, 1100)):
        diff = (y[at].double() - w[at]).abs() - half.eps / 2 * w[at].abs() - half.smallest_normal * half.eps / 2
        # 22-bit operands: two steps of few 2^-22 each
        assert float(diff.max()) <= 2.0 ** -18 * float(w[at].abs().max())


def test_gradient_with_and_without_keeping(monkeypatch):
    from torchopt_amd.accelerated_op import muon_op as module
    x, dy = randn(3, 200, 700, seed=1).cuda(), randn(3, 200, 700, seed=2).cuda()
    grads = []
    for limit in (module.KEEP_BYTES, 0):
        monkeypatch.setattr(module, 'KEEP_BYTES', limit)
        leaf = x.clone().requires_grad_()
        y = orthogonalize(leaf)
        grads += [torch.autograd.grad(y, leaf, dy, retain_graph=True)[0],
                  torch.autograd.grad(y, leaf, dy)[0]]
    assert all(torch.equal(g, grads[0]) for g in grads[1:])


def test_plain_gradient_is_autograds():
    x, dy = randn(30, 40).double().requires_grad_(), randn(30, 40, seed=1).double()
    want, = torch.autograd.grad(plain.orthogonalize(x), x, dy)
    assert (plain.gradient(x.detach(), dy) - want).norm() < 1e-12 * want.norm()


@pytest.mark.parametrize('m,n', [(24, 60), (100, 260)])
def test_gradient_against_differences(m, n):
    """<dy, Y(G + hD) - Y(G - hD)> / 2h and <gradient, D> of the operators differ by what the
    products may be off (over h), by the gradient's tolerance, and by the difference quotient's own
    error, which the 64-bit form shows and which is small itself."""
    g, d, dy = randn(m, n, seed=1), randn(m, n, seed=2), randn(m, n, seed=3)
    h = 2.0 ** -7
    up, down = g + h * d, g - h * d
    d = (up.double() - down.double()) / (2.0 * h)  # as the additions rounded
    dy64 = dy.double()
    exact, allowed = [], 0.0
    for x in (up, down):
        y, a = plain.tolerance(plain.orthogonalize, x.double(), dtype=F32)
        exact.append(y)
        allowed += a + 2.0 ** -24 * float(y.norm())
    quotient = float((dy64 * (exact[0] - exact[1])).sum()) / (2.0 * h)
    grad, off = plain.tolerance(plain.gradient, g.double(), dy64, dtype=F32)
    slope = float((grad * d).sum())
    size = float(grad.norm() * d.norm())
    own = orthogonalize([up.cuda(), down.cuda()])
    own_quotient = float((dy64 * (own[0].double() - own[1].double()).cpu()).sum()) / (2.0 * h)
    own_grad, = muon_op.orthogonalize_backward_multi([dy.cuda()], [g.cuda()])
    own_slope = float((own_grad.double().cpu() * d).sum())
    truncation = abs(quotient - slope)
    assert truncation < 0.02 * size
    bound = truncation + float(dy64.norm()) * allowed / (2.0 * h) + float(d.norm()) * (
        off + 2.0 ** -24 * float(grad.norm()))
    assert bound < 0.2 * size
    assert abs(own_quotient - own_slope) <= bound


def test_gradients_of_lists():
    """Outputs without a cotangent, inputs that need no gradient, one tensor given twice, a
    broadcast input, and no second derivative."""
    xs = [randn(40, 50, seed=k).cuda() for k in range(4)]
    a, b, c = (x.clone().requires_grad_() for x in xs[:3])
    ys = orthogonalize([a, b, xs[3], c, a])
    dy = randn(40, 50, seed=9).cuda()
    ga, gc = torch.autograd.grad([ys[0], ys[3], ys[4]], [a, c], [dy, 2 * dy, dy])
    one, = muon_op.orthogonalize_backward_multi([dy], [xs[0]])
    assert torch.equal(ga, one + one)
    assert torch.equal(gc, muon_op.orthogonalize_backward_multi([2 * dy], [xs[2]])[0])
    assert torch.autograd.grad(orthogonalize([a, b])[0].sum(), b, allow_unused=True)[0] is None
    row = randn(1, 50, seed=3).cuda().requires_grad_()
    orthogonalize(row.expand(40, 50)).backward(dy)
    full, = muon_op.orthogonalize_backward_multi([dy], [row.detach().expand(40, 50)])
    assert torch.equal(row.grad, full.sum(0, keepdim=True))
    y = orthogonalize(a)
    g, = torch.autograd.grad(y.square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        x = b * 1.0
        y = orthogonalize(x)
        x.add_(1.0)
        y.sum().backward()
    # mixed types in one list, each with its own gradient
    mixed = [x.to(t).requires_grad_() for x, t in zip(xs, (F32, BF16, F32))]
    sum(y.float().square().sum() for y in orthogonalize(mixed)).backward()
    assert all(x.grad is not None and x.grad.dtype == x.dtype for x in mixed)


# ---- 8-bit blocks ----------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [1, 2, 127, 128, 129, 255, 1000, 70001])
def test_blocks_are_exact(n, dtype):
    """Codes, scales and values are the formula's, ties included."""
    x = randn(n, seed=n).to(dtype)
    x[:128] = torch.arange(n).float()[:128].sub(64).to(dtype)       # ties among them
    if n > 700:
        x[256:384] = 0.0
        x[512:640] = (torch.arange(128).float() * 0.5 - 31.5).to(dtype)
        x[640] = 63.5
        x[400:402] = torch.finfo(dtype).tiny if dtype != F16 else 2.0 ** -20
    for lead in (0, 1):
        v = torch.empty(n + lead, dtype=dtype, device='cuda')[lead:].copy_(x)
        codes, scales = quantize_blocks(v)
        want_codes, want_scales, want = plain.quantize(x.double())
        assert codes.dtype == torch.int8 and scales.dtype == F32
        assert torch.equal(scales.cpu(), want_scales)
        assert torch.equal(codes.double().cpu(), want_codes)
        for t in TYPES:
            assert torch.equal(dequantize_blocks(codes, scales, t).cpu(), want.float().to(t)), t
    assert (want - x.double()).abs().max() <= want_scales.max() * 0.5 * (1 + 1e-6)


def test_blocks_lists_and_layouts():
    xs = [randn(30, 40, seed=1).cuda(), randn(5, seed=2, dtype=BF16).cuda(), torch.empty(0, device='cuda'),
          randn(6, 7, 8, seed=3).cuda().transpose(0, 2), torch.tensor(-3.0).cuda()]
    codes, scales = quantize_blocks(xs)
    back = dequantize_blocks(codes, scales)
    for x, c, s, b in zip(xs, codes, scales, back):
        assert c.shape == x.shape == b.shape and s.numel() == -(-x.numel() // 128)
        if x.numel():
            assert c.stride() == x.stride()
            assert ((b - x).abs().max() <= s.max() * 0.5 * (1 + 1e-6))
    assert float(back[4]) == -3.0
    x = randn(400, seed=1).cuda()
    x[5], x[300] = float('nan'), float('inf')
    b = dequantize_blocks(*quantize_blocks(x))
    assert b[:128].isnan().all() and b[256:384].isnan().all() and b[384:].isfinite().all()
    assert b[128:256].isfinite().all()
    many = [randn(50 + k, seed=k).cuda() for k in range(150)]
    for x, b in zip(many, dequantize_blocks(*quantize_blocks(many))):
        assert torch.equal(b.cpu(), plain.quantize(x.double().cpu())[2].float())


# ---- the step --------------------------------------------------------------------------------

LEAVES = [(4, 6), (32, 288), (5, 800), (70, 300), (300, 70), (1, 9), (129, 131), (6, 3, 3, 2), (0, 4)]


def leaf(shape, dtype, seed, order):
    t = randn(*shape, dtype=dtype, seed=seed).cuda()
    if order == 'column-major' and t.dim() == 2:
        return t.t().contiguous().t()
    if order == 'channels-last' and t.dim() == 4:
        return t.contiguous(memory_format=torch.channels_last)
    return t


def plain_step(p, g, m, scales, lr, momentum, nesterov, wd, maximize, adjust, apply, kw):
    """The step of one leaf in 64 bits (CPU tensors): new parameter or update, its allowed
    deviation before rounding, new momentum, new scales."""
    kind, dtype = m.dtype, p.dtype
    g = (-g if maximize else g).double()
    if kind == torch.int8:
        flat = m.permute(order_of(m)).reshape(-1).double()
        old = (flat * scales.double().repeat_interleave(plain.BLOCK)[:flat.numel()])
        new = momentum * old + g.permute(order_of(m)).reshape(-1)
        codes, new_scales, values = plain.quantize(new)
        back = [order_of(m).index(d) for d in range(m.dim())]
        unflat = lambda v: v.view([m.shape[d] for d in order_of(m)]).permute(back)  # noqa: E731
        kept, new_m = unflat(values.float().double()), unflat(codes)
    else:
        new_m = (momentum * m.double() + g).to(kind)
        kept, new_scales = new_m.double(), None
    u = (g + momentum * kept if nesterov else kept).flatten(1)
    o, allowed = plain.tolerance(plain.orthogonalize, u, dtype=dtype, **kw)
    r = plain.rate(*u.shape, adjust)
    # the look-ahead is held in 32 bits (a relative 2^-24 more, within the model's margin)
    if not apply:
        return r * o.view(g.shape), r * allowed, new_m, new_scales
    return ((1.0 - lr * wd) * p.double() - lr * r * o.view(g.shape), lr * r * allowed, new_m,
            new_scales)


def order_of(t):
    """Dimensions from the slowest to the fastest in memory."""
    return sorted(range(t.dim()), key=lambda d: -t.stride(d))


VARIANTS = [
    dict(), dict(nesterov=False), dict(weight_decay=0.1), dict(maximize=True, weight_decay=0.3),
    dict(adjust_lr_fn='match_rms_adamw'), dict(adjust_lr_fn='none', nesterov=False),
    dict(momentum=0.0), dict(steps=2, eps=0.1), dict(coefficients=(1.5, -0.5, 0.0), steps=3),
]


@pytest.mark.parametrize('apply', [True, False])
@pytest.mark.parametrize('order', ['dense', 'column-major', 'channels-last'])
@pytest.mark.parametrize('kept', ['own', 'float32', 'int8'])
@pytest.mark.parametrize('dtype', TYPES)
def test_step(dtype, kept, order, apply):
    kind = {'own': dtype, 'float32': F32, 'int8': torch.int8}[kept]
    variants = VARIANTS if order == 'dense' else VARIANTS[:1] + VARIANTS[3:4]
    for v, variant in enumerate(variants):
        variant = dict(variant)
        momentum = variant.pop('momentum', 0.95)
        nesterov, wd = variant.pop('nesterov', True), variant.pop('weight_decay', 0.0)
        maximize, adjust = variant.pop('maximize', False), variant.pop('adjust_lr_fn', None)
        if not apply and (wd or maximize):
            continue
        ps = [leaf(s, dtype, 3 * k, order) for k, s in enumerate(LEAVES)]
        gs = [leaf(s, dtype, 3 * k + 1, order) for k, s in enumerate(LEAVES)]
        ms, scales = [], None
        for k, s in enumerate(LEAVES):
            m = leaf(s, F32, 3 * k + 2, order)
            ms.append(m if kind == torch.int8 else m.to(kind))
        if kind == torch.int8:
            ms, scales = quantize_blocks(ms)
        old = [[t.cpu() if t is not None else None for t in ts]
               for ts in (ps, gs, ms, scales or [None] * len(ms))]
        versions = [t._version for t in ps + ms]
        if apply:
            muon_op.fused_step_multi_(ps, gs, ms, scales, momentum, 0.25, nesterov=nesterov,
                                      weight_decay=wd, maximize=maximize, adjust_lr_fn=adjust,
                                      **variant)
            out = ps
            assert all(torch.equal(g.cpu(), o) for g, o in zip(gs, old[1]))
            assert all(t._version > b for t, b in zip(ps + ms, versions))
        else:
            out = gs
            muon_op.forward_multi_(gs, ms, scales, momentum, nesterov=nesterov,
                                   adjust_lr_fn=adjust, **variant)
        for k, s in enumerate(LEAVES):
            if 0 in s:
                continue
            p, g, m, sc = (o[k] for o in old)
            want, allowed, new_m, new_s = plain_step(p, g, m, sc, 0.25, momentum, nesterov, wd,
                                                     maximize, adjust, apply, variant)
            what = f'variant {v} leaf {s}'
            assert out[k].stride() == p.stride()
            plain.assert_close(out[k], want, allowed, what)
            if kind == torch.int8:
                assert torch.equal(scales[k].cpu(), new_s), what
                assert torch.equal(ms[k].cpu().double(), new_m), what
            else:
                assert torch.equal(ms[k].cpu(), new_m), what


def test_one_gradient_for_two_parameters():
    g = randn(40, 70, seed=1).cuda()
    ps = [randn(40, 70, seed=k).cuda() for k in (2, 3)]
    qs, ms = [p.clone() for p in ps], [torch.zeros_like(p) for p in ps]
    muon_op.fused_step_multi_(ps, [g, g], ms, None, 0.9, 0.1)
    for q, p in zip(qs, ps):
        muon_op.fused_step_multi_([q], [g], [torch.zeros_like(q)], None, 0.9, 0.1)
        assert torch.equal(p, q)
    assert torch.equal(ms[0], ms[1])


def test_step_of_zero_gradients_decays_only():
    p = randn(70, 300, seed=1).cuda()
    want = p * (1.0 - 0.5 * 0.1)
    m, g = torch.zeros_like(p), torch.zeros_like(p)
    muon_op.fused_step_multi_([p], [g], [m], None, 0.95, 0.5, weight_decay=0.1)
    assert torch.allclose(p, want, rtol=2.0 ** -23, atol=0.0) and not m.any()


# ---- refusals --------------------------------------------------------------------------------


def test_refusals():
    x = torch.ones(3, 4, device='cuda')
    v, d = torch.ones(5, device='cuda'), torch.ones(3, 4, device='cuda', dtype=torch.float64)
    scale = torch.ones(1, device='cuda')
    q = torch.zeros(3, 4, device='cuda', dtype=torch.int8)

    def step(out=None, grads=None, mu=None, scales=None, momentum=0.9, lr=0.1, **kw):
        muon_op.fused_step_multi_(out or [x.clone()], grads or [x], mu or [x.clone()], scales,
                                  momentum, lr, **kw)

    base = x.clone()
    wide = torch.ones(3, 8, device='cuda')
    refused = [
        lambda: orthogonalize(v), lambda: orthogonalize(d), lambda: orthogonalize([x, v]),
        lambda: orthogonalize(x.to(torch.int32)), lambda: orthogonalize(torch._neg_view(x)),
        lambda: orthogonalize(x, steps=2.5), lambda: orthogonalize(x, steps=0),
        lambda: orthogonalize(x, steps=33), lambda: orthogonalize(x, eps=-1.0),
        lambda: orthogonalize(x, eps=float('nan')),
        lambda: orthogonalize(x, coefficients=(50.0, 1.0, 1.0)),
        lambda: orthogonalize(x, steps=3, coefficients=(6.0, -9.0, 4.0)),  # may reach 68
        lambda: orthogonalize(x, coefficients=(float('nan'), 1.0, 1.0)),
        lambda: muon_op.orthogonalize_multi([x, x.half()]),
        lambda: muon_op.orthogonalize_multi([x, x.cpu()]),
        lambda: muon_op.orthogonalize_backward_multi([x], [x, x]),
        lambda: muon_op.orthogonalize_backward_multi([x.t()], [x]),
        lambda: muon_op.orthogonalize_backward_multi([x.half()], [x]),
        lambda: step(grads=[x, x]), lambda: step(grads=[x.half()]), lambda: step(grads=[x.t()]),
        lambda: step(mu=[x.half()]), lambda: step(mu=[x.cpu()]), lambda: step(grads=[x.cpu()]),
        lambda: step(out=[v], grads=[v], mu=[v]), lambda: step(mu=[q]),       # blocks, no scales
        lambda: step(scales=[scale]),                                         # scales, no blocks
        lambda: step(mu=[q], scales=[]), lambda: step(mu=[q], scales=[scale.half()]),
        lambda: step(mu=[q], scales=[torch.ones(2, device='cuda')]),
        lambda: step(mu=[q], scales=[scale.cpu()]),
        lambda: step(momentum=1.0), lambda: step(momentum=-0.1), lambda: step(lr=float('nan')),
        lambda: step(adjust_lr_fn='unheard of'), lambda: step(steps=0),
        # other memory orders than the parameter's, gaps, and memory used twice
        lambda: step(mu=[torch.ones(4, 3, device='cuda').t()]),
        lambda: step(out=[wide[:, ::2]], mu=[x.clone()]),
        lambda: step(mu=[torch.ones(1, 4, device='cuda').expand(3, 4)]),
        lambda: step(out=[base], mu=[base]),
        lambda: step(out=[base], grads=[base]),
        lambda: step(mu=[x]),
        lambda: step(out=[base, base], grads=[x, x], mu=[x.clone(), x.clone()]),
        lambda: step(out=[x.clone(), x.clone()], grads=[x, x], mu=[base, base]),
        lambda: quantize_blocks(d), lambda: quantize_blocks(wide[:, ::2]),
        lambda: dequantize_blocks(q, scale, torch.float64),
        lambda: dequantize_blocks(q, torch.ones(2, device='cuda')),
        lambda: dequantize_blocks(x, scale),
    ]
    for k, call in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()
            pytest.fail(f'call {k} was not refused')
    assert torch.equal(x, torch.ones_like(x)) and torch.equal(base, x)


# ---- streams, captured graphs, threads -------------------------------------------------------


def test_on_another_stream():
    x, dy = randn(3, 300, 700, seed=1).cuda(), randn(3, 300, 700, seed=2).cuda()
    want = orthogonalize(x), muon_op.orthogonalize_backward_multi([dy], [x])[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 2:   # in flight side by side, each with its own workspace
        with torch.cuda.stream(s):
            got.append((orthogonalize(x), muon_op.orthogonalize_backward_multi([dy], [x])[0]))
    torch.cuda.synchronize()
    for y, dx in got:
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])


def test_captured_forward_and_backward():
    xs = [randn(90, 400, seed=1).cuda(), randn(32, 288, seed=2).cuda()]
    dys = [randn(90, 400, seed=3).cuda(), randn(32, 288, seed=4).cuda()]

    def both():
        leaves = [x.detach().requires_grad_() for x in xs]
        ys = orthogonalize(leaves)
        return [y.detach() for y in ys], list(torch.autograd.grad(ys, leaves, dys))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):   # two graphs: each has a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = both()
        graphs.append((graph, kept))
    for k in range(4):
        for x in xs:
            x.copy_(randn(*x.shape, seed=50 + k))
        graphs[0][0].replay()
        graphs[1][0].replay()
        eager = both()
        torch.cuda.synchronize()
        for _, kept in graphs:
            for a, b in zip(kept[0] + kept[1], eager[0] + eager[1]):
                assert torch.equal(a, b)


@pytest.mark.parametrize('kind', [None, torch.int8])
def test_captured_step(kind):
    def make():
        ps = [randn(90, 400, seed=1, dtype=BF16).cuda(), randn(32, 9, 4, seed=2, dtype=BF16).cuda()]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, torchopt_amd.FusedMuon(ps, lr=0.1, momentum_dtype=kind)

    (ps, opt), (qs, other) = make(), make()
    with pytest.raises(RuntimeError, match='init_state'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.init_state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for p, q in zip(ps, qs):
            p.grad.copy_(randn(*p.shape, seed=k + 7, dtype=BF16))
            q.grad.copy_(p.grad)
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        assert all(map(torch.equal, ps, qs))
    scheduled = torchopt_amd.FusedMuon(ps, lr=lambda n: 0.1)
    scheduled.init_state()
    with pytest.raises(RuntimeError, match='schedule'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            scheduled.step()


def test_two_threads():
    import threading
    x = randn(2, 200, 300, seed=1).cuda()
    want, wrong = orthogonalize(x), []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                if not torch.equal(orthogonalize(x), want):
                    wrong.append(1)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
