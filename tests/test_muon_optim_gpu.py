"""The optimizers on the operators for matrix-shaped parameters: `FusedMuon`, the functional
`muon` and `scale_by_muon`, `MetaMuon`, and a run of them together."""

from __future__ import annotations

import math

import pytest
import torch
from torch import nn

import muon_plain as plain
import torchopt_amd
from torchopt_amd import FusedMuon, MetaMuon, muon, orthogonalize
from torchopt_amd.transform import scale_by_muon

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def randn(*shape, dtype=F32, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=gen)).to(dtype).cuda()


SHAPES = [(40, 60), (16, 3, 3, 3), (100, 30)]


def params(dtype=F32, seed=0):
    return [nn.Parameter(randn(*s, dtype=dtype, seed=seed + k)) for k, s in enumerate(SHAPES)]


def give_grads(ps, step):
    for k, p in enumerate(ps):
        p.grad = randn(*p.shape, dtype=p.dtype, seed=100 * step + k)


def test_optimizer_follows_the_formula():
    """Three steps with a schedule, a missing gradient and a closure."""
    ps = params()
    opt = FusedMuon(ps, lr=lambda n: 0.1 / (1 + n), weight_decay=0.2)
    want = [p.detach().double().cpu() for p in ps]
    ms = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(ps)
    for n in range(3):
        give_grads(ps, n)
        if n == 1:
            ps[2].grad = None
        loss = opt.step(lambda: torch.ones(()))
        assert float(loss) == 1.0
        lr = 0.1 / (1 + n)
        for k, p in enumerate(ps):
            if p.grad is None:
                continue
            g = p.grad.double().cpu()
            ms[k] = (0.95 * ms[k] + g).float().double()
            u = (g + 0.95 * ms[k]).flatten(1)
            o, allowed = plain.tolerance(plain.orthogonalize, u, dtype=F32)
            r = lr * plain.rate(*u.shape, None)
            want[k] = (1.0 - lr * 0.2) * want[k] - r * o.view(g.shape)
            slack[k] += r * allowed + 2.0 ** -24 * float(want[k].norm())
        for k, p in enumerate(ps):
            plain.assert_close(p, want[k], slack[k], f'step {n} leaf {k}')
    (taken, state), = opt.state_dict()
    assert taken == 3 and all(torch.equal(m.double().cpu(), w) for m, w in zip(state.momentum, ms))


@pytest.mark.parametrize('source,target', [(None, torch.int8), (torch.int8, None), (torch.int8, torch.int8),
                                           (None, F32), (F32, None)])
def test_state_moves_between_momentum_types(source, target):
    ps, qs = params(BF16), params(BF16)
    qs[1].data = qs[1].data.contiguous(memory_format=torch.channels_last)
    first = FusedMuon(ps, lr=0.1, momentum_dtype=source)
    give_grads(ps, 1)
    first.step()
    second = FusedMuon(qs, lr=0.1, momentum_dtype=target)
    second.load_state_dict(first.state_dict())
    (n, a), = first.state_dict()
    (m, b), = second.state_dict()
    assert n == m == 1
    for k, q in enumerate(qs):
        assert b.momentum[k].dtype == (target or BF16) and b.momentum[k].stride() == q.stride()
        values = [torchopt_amd.dequantize_blocks(s.momentum[k], s.scales[k])
                  if s.scales[k] is not None else s.momentum[k].float() for s in (a, b)]
        # blocks: half a scale; bfloat16: half a step
        worst = values[0].abs().max() * (0.5 / 127 + 2.0 ** -8) * 1.001
        assert (values[0] - values[1]).abs().max() <= worst
        q.data.copy_(ps[k].data)
        q.grad = ps[k].grad.clone(memory_format=torch.preserve_format)
    if source == target and source is not None:
        assert torch.equal(a.momentum[0], b.momentum[0]) and torch.equal(a.scales[0], b.scales[0])
    for p, q in zip(ps, qs):
        q.grad = torch.empty_like(q).copy_(p.grad)
    second.step()
    assert all(torch.isfinite(q).all() for q in qs)


def test_groups_devices_and_types_in_one_optimizer():
    a, b = params(), params(BF16, seed=9)
    opt = FusedMuon(a + b, lr=0.1)
    opt.add_param_group([nn.Parameter(randn(5, 7, seed=3))])
    last = opt.param_groups[1][0]
    before = [p.detach().clone() for p in a + b + [last]]
    give_grads(a + b + [last], 2)
    opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(a + b + [last], before))
    alone = [p.detach().clone() for p in before[3:6]]
    single = [nn.Parameter(p) for p in alone]
    for p, q in zip(single, b):
        p.grad = q.grad
    FusedMuon(single, lr=0.1).step()
    assert all(torch.equal(p, q) for p, q in zip(single, b))
    opt.zero_grad()
    assert all(not p.grad.any() for p in a + b)
    opt.zero_grad(set_to_none=True)
    assert all(p.grad is None for p in a + b)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('adjust', [None, 'match_rms_adamw', 'none'])
def test_transform_in_and_out_of_place(dtype, adjust):
    ps = [p.detach() for p in params(dtype)] + [None]
    gs = [randn(*s, dtype=dtype, seed=70 + k) for k, s in enumerate(SHAPES)] + [None]
    t = scale_by_muon(adjust_lr_fn=adjust)
    s_in, s_out = t.init(ps), t.init(ps)
    for n in range(2):
        out, s_out = t.update(gs, s_out, inplace=False)
        mine = [None if g is None else g.clone() for g in gs]
        ret, s_in = t.update(mine, s_in, inplace=True)
        assert ret[3] is None and out[3] is None
        for k, g in enumerate(gs[:3]):
            assert ret[k] is mine[k]
            # in place forms the sums in 64 bits and rounds once, out of place rounds each
            # operation to the type: a few half steps of the update that goes into the series
            u = torch.finfo(dtype).eps / 2
            exact, allowed = plain.tolerance(
                plain.orthogonalize, _look_ahead(gs[k], s_in.momentum[k]), dtype=dtype)
            r = plain.rate(g.shape[0], g.numel() // g.shape[0], adjust)
            shift = _moved(_look_ahead(gs[k], s_in.momentum[k]), exact, 8 * u)
            plain.assert_close(ret[k], r * exact.view(g.shape), r * allowed, f'{n} {k}')
            plain.assert_close(out[k], r * exact.view(g.shape),
                               r * (allowed + shift + u * float(exact.norm())), f'{n} {k}')
            assert (s_in.momentum[k].float() - s_out.momentum[k].float()).abs().max() <= \
                8 * u * s_in.momentum[k].float().abs().max()


def _look_ahead(g, m):
    return (g.double() + 0.95 * m.double()).flatten(1).cpu()


def _moved(u, exact, relative):
    """Four times the largest move of the result under random relative changes of its input."""
    worst = 0.0
    for seed in (1, 2, 3):
        gen = torch.Generator().manual_seed(seed)
        noise = 1.0 + relative * (2.0 * torch.rand(u.shape, generator=gen, dtype=u.dtype) - 1.0)
        worst = max(worst, float((plain.orthogonalize(u * noise) - exact).norm()))
    return 4.0 * worst


def test_transform_with_blocks_is_the_steps():
    """`scale_by_muon` with 8-bit blocks, applied by hand, is `FusedMuon`'s step."""
    ps, qs = params(), params()
    opt = FusedMuon(ps, lr=0.5, weight_decay=0.0, momentum_dtype=torch.int8)
    t = scale_by_muon(momentum_dtype=torch.int8)
    state = t.init([q.detach() for q in qs])
    for n in range(3):
        give_grads(ps, n)
        gs = [p.grad.clone() for p in ps]
        opt.step()
        gs, state = t.update(gs, state)
        (_, kept), = opt.state_dict()
        for k, q in enumerate(qs):
            assert torch.equal(kept.momentum[k], state.momentum[k])
            assert torch.equal(kept.scales[k], state.scales[k])
            q.data.sub_(0.5 * gs[k])
            # (one rounding against two)
            assert torch.allclose(ps[k], q, rtol=0.0, atol=2.0 ** -22 * float(q.abs().max()))


def test_functional_partition():
    """Matrices go through Muon, the rest through Adam; dicts may change their order."""
    tree = {'w': randn(20, 30, seed=1), 'b': randn(30, seed=2), 's': randn(seed=3), 'n': None}
    grads = {k: None if v is None else randn(*v.shape, seed=9) for k, v in tree.items()}
    both = muon(0.1, weight_decay=0.0)
    updates, state = both.update({k: None if g is None else g.clone() for k, g in grads.items()},
                                 both.init(tree), params=tree)
    alone = scale_by_muon()
    w, _ = alone.update([grads['w'].clone()], alone.init([tree['w']]))
    assert torch.equal(updates['w'], w[0] * -0.1)
    adam = torchopt_amd.adam(0.1, (0.9, 0.95))
    rest = [tree['b'], tree['s']]
    want, _ = adam.update([grads['b'].clone(), grads['s'].clone()], adam.init(rest))
    assert torch.equal(updates['b'], want[0]) and torch.equal(updates['s'], want[1])
    assert updates['n'] is None
    turned = {k: None if grads[k] is None else grads[k].clone() for k in reversed(list(grads))}
    again, _ = both.update(turned, both.init(tree), params=tree)
    assert torch.equal(again['w'], updates['w']) and torch.equal(again['b'], updates['b'])
    out, _ = both.update(grads, both.init(tree), params=tree, inplace=False)
    assert (out['w'] - updates['w']).abs().max() < 1e-4


def test_outer_gradient_through_two_steps():
    """d/d(initial weights, gradients) of a loss after two differentiable steps, against the same
    in 64 bits with autograd through the plain form."""
    w0, g0, g1 = randn(24, 40, seed=1), randn(24, 40, seed=2), randn(24, 40, seed=3)

    def run(w, a, b, series):
        m = torch.zeros_like(w)
        for g in (a, b):
            g = g * w  # the second gradient depends on the first step
            m = 0.95 * m + g
            w = w - 0.1 * series(g + 0.95 * m)
        return w.pow(3).sum()

    leaves = [x.double().cpu().requires_grad_() for x in (w0, g0, g1)]
    want = torch.autograd.grad(run(*leaves, plain.orthogonalize), leaves)

    t = scale_by_muon(moment_requires_grad=False)
    mine = [x.clone().requires_grad_() for x in (w0, g0, g1)]
    w, state = mine[0], t.init([w0])
    for g in mine[1:]:
        (u,), state = t.update([g * w], state, inplace=False)
        w = w - 0.1 * u
    got = torch.autograd.grad(w.pow(3).sum(), mine)
    # both forms of every step are conditioned alike: the deviation under the rounding model
    noisy = [torch.autograd.grad(run(*leaves, lambda u, s=s: plain.orthogonalize(
        u, r=plain.Noisy(s, F32))), leaves) for s in (1, 2, 3)]
    for k, (a, b) in enumerate(zip(got, want)):
        allowed = 4.0 * max(float((n[k] - b).norm()) for n in noisy)
        plain.assert_close(a, b, allowed, f'argument {k}')


def test_meta_muon():
    torch.manual_seed(0)
    net = nn.Sequential(nn.Conv2d(1, 8, 3), nn.ReLU(), nn.Flatten(), nn.Linear(8 * 36, 5)).cuda()
    x, y = randn(16, 1, 8, 8, seed=1), torch.arange(16).cuda() % 5
    scale = torch.ones((), device='cuda', requires_grad=True)
    inner = MetaMuon(net, lr=0.05, adam_eps_root=1e-8)
    meta = list(net.parameters())
    before = [p.detach().clone() for p in meta]
    for _ in range(2):
        inner.step(nn.functional.cross_entropy(net(scale * x), y))
    loss = nn.functional.cross_entropy(net(x), y)
    grads = torch.autograd.grad(loss, meta + [scale])
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)
    assert all(torch.equal(p, b) for p, b in zip(meta, before))


def test_compiled():
    x = randn(3, 40, 70, seed=1)

    def f(x, w):
        return (orthogonalize(x * 2.0, steps=3) * w).sum()

    w = randn(3, 40, 70, seed=2)
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    torch.compile(f, fullgraph=True, backend='aot_eager')(leaf, w).backward()
    f(other, w).backward()
    assert torch.equal(leaf.grad, other.grad)


def test_registered_operators_pass_opcheck():
    x, dy = randn(2, 20, 30, seed=1), randn(2, 20, 30, seed=2)
    p, g, m = (randn(20, 30, seed=k) for k in (3, 4, 5))
    q, s = torchopt_amd.quantize_blocks(m)
    series, ops = (3, list(plain.COEFFICIENTS), 1e-7), torch.ops.torchopt_amd
    torch.library.opcheck(ops.orthogonalize_multi.default, ([x, x[0]], *series))
    torch.library.opcheck(ops.orthogonalize_multi.default, ([x.clone().requires_grad_()], *series))
    torch.library.opcheck(ops.orthogonalize_backward_multi.default, ([dy], [x], *series))
    torch.library.opcheck(ops.muon_forward_multi_.default, ([g.clone()], [q.clone()], [s.clone()], 0.9,
                                                            True, *series, None))
    torch.library.opcheck(ops.muon_fused_step_multi_.default, (
        [p.clone()], [g], [m.clone()], [], 0.9, 0.1, True, 0.0, False, *series, 'none'))


@pytest.mark.parametrize('kind', [None, torch.int8])
def test_compiled_transform(kind):
    t = scale_by_muon(momentum_dtype=kind)
    gs = [randn(20, 30, seed=1), randn(40, 300, seed=2)]
    state, other = t.init(gs), t.init(gs)

    def step(gs, state):
        return t.update(gs, state)

    mine = torch.compile(step, fullgraph=True, backend='aot_eager')
    for _ in range(2):
        out, state = mine([g.clone() for g in gs], state)
        want, other = t.update([g.clone() for g in gs], other)
        assert all(map(torch.equal, out, want))
        assert all(map(torch.equal, state.momentum, other.momentum))


def test_a_run_of_them_together():
    """A small network: matrices by FusedMuon with 8-bit blocks, the rest by FusedAdam, in
    bfloat16, saved and restored half way; the restored run repeats the first bit for bit."""
    def net():
        torch.manual_seed(3)
        return nn.Sequential(nn.Linear(64, 128), nn.Tanh(), nn.Linear(128, 128), nn.Tanh(),
                             nn.Linear(128, 8)).cuda().to(BF16)

    def optimizers(model):
        matrices = [p for p in model.parameters() if p.dim() >= 2]
        rest = [p for p in model.parameters() if p.dim() < 2]
        return [FusedMuon(matrices, lr=0.02, momentum_dtype=torch.int8),
                torchopt_amd.FusedAdam(rest, lr=0.01, betas=(0.9, 0.95))]

    x, y = randn(256, 64, dtype=BF16, seed=4), randn(256, 8, dtype=BF16, seed=5)

    def train(model, opts, steps):
        for _ in range(steps):
            for o in opts:
                o.zero_grad(set_to_none=True)
            (model(x) - y).float().square().mean().backward()
            for o in opts:
                o.step()

    model = net()
    opts = optimizers(model)
    train(model, opts, 4)
    saved = {k: v.clone() for k, v in model.state_dict().items()}
    copy = lambda s: torch.utils._pytree.tree_map(  # noqa: E731
        lambda t: t.clone() if isinstance(t, torch.Tensor) else t, s)
    states = [copy(o.state_dict()) for o in opts]
    train(model, opts, 4)
    again = net()
    again.load_state_dict(saved)
    fresh = optimizers(again)
    for o, s in zip(fresh, states):
        o.load_state_dict(s)
    train(again, fresh, 4)
    for p, q in zip(model.parameters(), again.parameters()):
        assert torch.equal(p, q) and torch.isfinite(p).all()
    for p in model.parameters():
        if p.dim() >= 2:
            o = orthogonalize(p.detach())
            assert o.float().norm() / math.sqrt(min(p.shape)) < 1.3
