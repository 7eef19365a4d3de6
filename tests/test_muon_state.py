"""`FusedMuon.load_state_dict` takes a copy: steps leave the state that was loaded as it is."""

from __future__ import annotations

import pytest
import torch

from torchopt_amd import FusedMuon

KINDS = [None, torch.float32, torch.int8]


def params(device, dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    shapes = [(6, 40), (4, 3, 3, 3), (50, 7)]
    ps = [torch.randn(s, generator=gen).to(device, dtype) for s in shapes]
    ps[1] = ps[1].contiguous(memory_format=torch.channels_last)
    ps[2] = ps[2].t().contiguous().t()
    return ps


def tensors(state_dict):
    (_, state), = state_dict
    return [t for part in state for t in part if t is not None]


@pytest.mark.parametrize('kind', KINDS)
def test_loaded_state_lies_in_its_own_memory(kind):
    first, second = (FusedMuon(params('cpu'), momentum_dtype=kind) for _ in range(2))
    first.init_state()
    second.load_state_dict(first.state_dict())
    mine, theirs = tensors(first.state_dict()), tensors(second.state_dict())
    assert len(mine) == len(theirs) == (6 if kind == torch.int8 else 3)
    for a, b in zip(mine, theirs):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a, b) and a.data_ptr() != b.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_snapshot_serves_more_than_once(dtype, kind):
    def step(opt, seed):
        gen = torch.Generator().manual_seed(seed)
        for p in opt.param_groups[0]:
            p.grad = torch.randn(p.shape, generator=gen).to(p)
        opt.step()

    first = FusedMuon(params('cuda', dtype), lr=0.1, momentum_dtype=kind)
    step(first, 1)
    snapshot = first.state_dict()
    before = [t.clone() for t in tensors(snapshot)]
    ends = []
    for _ in range(2):
        again = FusedMuon(params('cuda', dtype), lr=0.1, momentum_dtype=kind)
        again.load_state_dict(snapshot)
        step(again, 2)
        step(again, 3)
        ends.append(again.param_groups[0])
        assert all(map(torch.equal, tensors(snapshot), before))
    assert all(map(torch.equal, *ends))
