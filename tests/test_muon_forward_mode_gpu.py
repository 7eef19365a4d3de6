"""Forward-mode derivatives are refused by the operators for matrix-shaped parameters: a result without
a tangent would count as a constant in whatever it enters."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import torchopt_amd
from torchopt_amd import orthogonalize, quantize_blocks
from torchopt_amd._C import muon_op
from torchopt_amd.transform import scale_by_muon

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('m,n', [(20, 30), (90, 300)])
def test_dual_tensors_are_refused(m, n, grad):
    x, tangent = randn(m, n, seed=1), randn(m, n, seed=2)
    want = orthogonalize(x)
    codes, scales = quantize_blocks(x)
    t = scale_by_muon()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        d = forward_ad.make_dual(x.clone(), tangent)
        dual_scales = forward_ad.make_dual(scales.clone(), torch.ones_like(scales))
        new = torch.empty_like
        refused = [
            lambda: orthogonalize(d), lambda: orthogonalize([x, d]), lambda: orthogonalize(d.t()),
            lambda: orthogonalize(d[1:]), lambda: orthogonalize(d.clone().requires_grad_()),
            lambda: muon_op.orthogonalize_multi([d]), lambda: muon_op.orthogonalize_keep_multi([d], 1 << 30),
            lambda: muon_op.orthogonalize_backward_multi([d], [x]),
            lambda: muon_op.orthogonalize_backward_multi([x], [d]),
            lambda: t.update([d], t.init([x]), inplace=False),
            lambda: t.update([d], t.init([x])),
            lambda: t.update([x.clone()], t.init([x])._replace(momentum=[d]), inplace=False),
            lambda: t.update([x.clone()], t.init([x])._replace(momentum=[d])),
            lambda: torchopt_amd.muon().update([d], torchopt_amd.muon().init([x]), params=[x]),
            lambda: muon_op.fused_step_multi_([d], [x], [x.clone()], None, 0.9, 0.1),
            lambda: muon_op.fused_step_multi_([x.clone()], [d], [x.clone()], None, 0.9, 0.1),
            lambda: muon_op.fused_step_multi_([x.clone()], [x], [d], None, 0.9, 0.1),
            lambda: muon_op.fused_step_multi_([x.clone()], [x], [codes.clone()], [dual_scales], 0.9, 0.1),
            lambda: quantize_blocks(d),
            lambda: muon_op.dequantize_multi_([new(x)], [codes], [dual_scales]),
        ]
        for k, call in enumerate(refused):
            with pytest.raises(NotImplementedError):
                call()
                pytest.fail(f'call {k} was not refused')
        assert torch.equal(forward_ad.unpack_dual(d).primal, x)
        # what is no dual tensor is served beside one
        assert torch.equal(orthogonalize(x), want)
        assert torch.equal(orthogonalize(forward_ad.unpack_dual(d).primal), want)


def test_function_transforms_are_refused():
    x = randn(20, 30, seed=1)
    for call in (lambda: torch.func.jvp(orthogonalize, (x,), (x,)),
                 lambda: torch.func.vmap(orthogonalize)(x[None])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
