"""Gradient transformations that sit directly on the native operators."""

from torchopt_amd.transform.scale_by_adam import ScaleByAdamState, scale_by_accelerated_adam
from torchopt_amd.transform.scale_by_muon import ScaleByMuonState, scale_by_muon

__all__ = ['ScaleByAdamState', 'ScaleByMuonState', 'scale_by_accelerated_adam', 'scale_by_muon']
