"""Hyper-parameters that the optimizers on matrices would otherwise change silently are refused."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from conftest import REPO
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


def test_coefficients_beyond_what_operands_hold():
    """Products of 1e30 and more leave the range of the operands' scales: they gave NaN."""
    class Series(ctypes.Structure):
        _fields_ = [('steps', ctypes.c_int)] + [(k, ctypes.c_double) for k in ('a', 'b', 'c', 'eps')]

    lib = ctypes.CDLL(os.path.join(REPO, 'torchopt_amd', 'libtoa_muon.so'))
    lib.toa_muon_orthogonalize_workspace.restype = ctypes.c_size_t
    side, status = (ctypes.c_int64 * 1)(100), ctypes.c_int(0)

    def refused(steps, a, b, c):
        status.value = 99
        lib.toa_muon_orthogonalize_workspace(0, ctypes.c_size_t(1), side, side,
                                             ctypes.byref(Series(steps, a, b, c, 1e-7)), 0,
                                             ctypes.byref(status))
        return status.value

    for series in ((1, 1e31, 0.0, 0.0), (1, 0.0, 1e31, 0.0), (1, 0.0, 0.0, 1e30), (1, 1e300, 1e300, 1e300),
                   (2, 1.0, 1e38, 0.0)):
        assert refused(*series) == -5, series
    for series in ((1, 1e29, 0.0, 0.0), (1, 100.0, -3.0, 0.0), (5, 3.4445, -4.775, 2.0315), (3, 0.0, 0.0, 0.0)):
        assert refused(*series) == 0, series
