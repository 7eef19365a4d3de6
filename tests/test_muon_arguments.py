"""Hyper-parameters that the optimizers on matrices would otherwise change silently are refused."""

from __future__ import annotations

import pytest
import torch

from torchopt_amd import FusedMuon, MetaMuon, muon
from torchopt_amd.transform import scale_by_muon

MAKERS = [lambda **kw: FusedMuon([torch.ones(3, 4)], **kw), lambda **kw: scale_by_muon(**kw),
          lambda **kw: muon(**kw), lambda **kw: MetaMuon(torch.nn.Linear(3, 4), **kw)]


@pytest.mark.parametrize('make', MAKERS)
def test_fractional_steps_and_infinite_eps(make):
    for bad in (dict(ns_steps=2.5), dict(ns_steps=float('nan')), dict(ns_steps=0.5), dict(eps=float('inf')),
                dict(eps=float('nan'))):
        with pytest.raises(ValueError):
            make(**bad)


def test_whole_steps_of_other_types():
    for good in (5, 5.0, torch.tensor(5)):
        assert FusedMuon([torch.ones(3, 4)], ns_steps=good).ns_steps == 5
        scale_by_muon(ns_steps=good)
