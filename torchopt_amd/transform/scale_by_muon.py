"""The Muon transformation: momentum, then orthogonalisation of every matrix-shaped update.

The reference has no counterpart; the transformation follows its protocol
(/root/reference/torchopt/base.py:118-151), so it chains with the others.  Per leaf

    ``M <- momentum * M + g``,   ``U = g + momentum * M`` (``nesterov``; else ``U = M``),
    ``update = r * orthogonalize(U)``

where ``r`` follows `adjust_lr_fn`: ``sqrt(max(1, rows / columns))`` for None or ``'original'``,
``0.2 * sqrt(max(rows, columns))`` for ``'match_rms_adamw'`` (updates as large as AdamW's, so
that one learning rate serves both), 1 for ``'none'``.

A leaf of more than two dimensions is the matrix of its first dimension times all the others.
In place the whole tree is one call per device and dtype, which overwrites updates and momentum.
Out of place everything is differentiable with respect to updates and momentum.  Both ways a 16-bit
momentum is the 64-bit sum rounded once, and the look-ahead and the result are held in 32 bits until the
update is rounded to its type; the series may round differently, as `orthogonalize` takes the other way
through its steps where a gradient is needed.
"""

from __future__ import annotations

import math
from typing import Any, NamedTuple

import torch

from torchopt_amd import _tree
from torchopt_amd.accelerated_op.library import dispatch
from torchopt_amd.accelerated_op.muon_op import COEFFICIENTS, orthogonalize
from torchopt_amd.base import GradientTransformation


__all__ = ['ScaleByMuonState', 'scale_by_muon']

ADJUST = (None, 'original', 'match_rms_adamw', 'none')
BLOCK = 128  # elements that share a scale in an 8-bit momentum
_HALVES = (torch.float16, torch.bfloat16)


class ScaleByMuonState(NamedTuple):
    """Momentum per leaf and, for a momentum in 8-bit blocks, its scales (None otherwise)."""

    momentum: Any
    scales: Any


def check_muon(momentum: float, ns_steps: int, ns_coefficients: tuple, eps: float,
               adjust_lr_fn: str | None, momentum_dtype: torch.dtype | None) -> None:
    """Refuses hyper-parameters that the operator does not take."""
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f'Invalid momentum value: {momentum}')
    if int(ns_steps) != ns_steps or not 1 <= ns_steps <= 32:
        raise ValueError(f'Invalid ns_steps value: {ns_steps} (a whole number, 1 to 32)')
    if len(ns_coefficients) != 3 or not all(math.isfinite(c) for c in ns_coefficients):
        raise ValueError(f'Invalid ns_coefficients: {ns_coefficients} (three finite numbers)')
    if not 0.0 <= eps < math.inf:
        raise ValueError(f'Invalid epsilon value: {eps}')
    if adjust_lr_fn not in ADJUST:
        raise ValueError(f'Invalid adjust_lr_fn: {adjust_lr_fn!r}')
    if momentum_dtype not in (None, torch.float32, torch.int8):
        raise ValueError(f'Invalid momentum_dtype: {momentum_dtype} (None for the parameters\' '
                         'own, torch.float32, or torch.int8 for 8-bit blocks)')


def require_matrix(t: torch.Tensor, who: str) -> None:
    if t.dim() < 2:
        raise ValueError(f'{who}: takes matrices (2 dimensions or more), got a tensor of shape '
                         f'{tuple(t.shape)}; step vectors and scalars with Adam')
    if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f'{who}: takes float32, float16 and bfloat16, got {t.dtype}')


def zero_momentum(t: torch.Tensor, momentum_dtype: torch.dtype | None,
                  requires_grad: bool = False):
    """``(momentum, scales)`` of a parameter before its first step, in its memory layout."""
    kind = t.dtype if momentum_dtype is None else momentum_dtype
    m = torch.zeros_like(t, dtype=kind, requires_grad=requires_grad and kind != torch.int8)
    scales = None
    if kind == torch.int8:
        scales = torch.zeros(-(-t.numel() // BLOCK), dtype=torch.float32, device=t.device)
    return m, scales


def shape_rate(t: torch.Tensor, adjust_lr_fn: str | None) -> float:
    rows, cols = t.shape[0], t.numel() // max(1, t.shape[0])
    if adjust_lr_fn in (None, 'original'):
        return math.sqrt(max(1.0, rows / max(1, cols)))
    return 0.2 * math.sqrt(max(rows, cols)) if adjust_lr_fn == 'match_rms_adamw' else 1.0


def scale_by_muon(
    momentum: float = 0.95,
    nesterov: bool = True,
    ns_steps: int = 5,
    ns_coefficients: tuple[float, float, float] = COEFFICIENTS,
    eps: float = 1e-7,
    adjust_lr_fn: str | None = None,
    moment_requires_grad: bool = False,
    momentum_dtype: torch.dtype | None = None,
) -> GradientTransformation:
    """Rescale updates according to Muon.

    Args:
        momentum: decay rate of the momentum.
        nesterov: look one step of the momentum ahead.
        ns_steps, ns_coefficients, eps: the Newton-Schulz series, see `orthogonalize`.
        adjust_lr_fn: how the update's length follows the matrix's shape.
        moment_requires_grad: create the momentum with ``requires_grad=True``.
        momentum_dtype: what the momentum is kept in: None (the parameters' type),
            ``torch.float32``, or ``torch.int8``: 8-bit blocks of 128 elements with a float32
            scale each, in place only.

    Returns:
        An ``(init, update)`` pair.
    """
    check_muon(momentum, ns_steps, ns_coefficients, eps, adjust_lr_fn, momentum_dtype)
    series = dict(steps=int(ns_steps), coefficients=tuple(ns_coefficients), eps=float(eps))

    def init_fn(params):
        leaves, spec = _tree.flatten(params)
        kept = []
        for t in leaves:
            if t is None:
                kept.append((None, None))
                continue
            require_matrix(t, 'scale_by_muon')
            kept.append(zero_momentum(t, momentum_dtype, moment_requires_grad))
        return ScaleByMuonState(momentum=_tree.rebuild([m for m, _ in kept], params, spec),
                                scales=_tree.rebuild([s for _, s in kept], params, spec))

    def update_fn(updates, state, *, params=None, inplace=True):  # noqa: ARG001
        g_leaves, g_spec = _tree.flatten(updates)
        m_leaves, m_spec = _tree.flatten(state.momentum)
        s_leaves = _tree.leaves_like(state.scales, m_spec)
        if (type(g_spec) is _tree.DictSpec and type(m_spec) is _tree.DictSpec
                and g_spec.keys != m_spec.keys):
            # the same names in another order: line the gradients up with the state
            g_leaves = _tree.leaves_like(updates, m_spec)
            g_spec = _tree.DictSpec(g_spec.kind, m_spec.keys)
        if len(g_leaves) != len(m_leaves):
            raise ValueError('updates and optimizer state have different tree structures; '
                             'make sure `init` was called on matching parameters')
        # no state for a leaf: nothing comes out of it; no gradient: its state stays
        new_g = [None if m is None else g for g, m in zip(g_leaves, m_leaves)]
        new_m = list(m_leaves)
        live = [k for k, g in enumerate(new_g) if g is not None]
        if inplace:
            groups: dict[tuple, list[int]] = {}
            for k in live:
                groups.setdefault((new_g[k].device, new_g[k].dtype), []).append(k)
            for ks in groups.values():
                scales = None
                if s_leaves[ks[0]] is not None:
                    scales = [s_leaves[k] for k in ks]
                dispatch.muon_forward_multi_(
                    [new_g[k] for k in ks], [m_leaves[k] for k in ks], scales, momentum,
                    nesterov=nesterov, adjust_lr_fn=adjust_lr_fn, **series)
        elif live:
            if any(m_leaves[k].dtype == torch.int8 for k in live):
                raise ValueError('scale_by_muon: a momentum in 8-bit blocks is updated in place '
                                 'only')
            looked = []
            for k in live:
                g, m = new_g[k], m_leaves[k]
                halves = m.dtype in _HALVES and g.dtype == m.dtype
                if halves:
                    # (a sum in 16 bits would round twice, and one in 32 with the decay rate as a
                    # float breaks the ties of short binary fractions)
                    new_m[k] = m.double().mul(momentum).add(g).to(m.dtype)
                else:
                    new_m[k] = m.mul(momentum).add(g)
                u = new_m[k].float() if halves else new_m[k]
                looked.append((u.mul(momentum).add(g) if nesterov else u).flatten(1))
            for k, o in zip(live, orthogonalize(looked, **series)):
                g, r = new_g[k], shape_rate(new_g[k], adjust_lr_fn)
                new_g[k] = (o if r == 1.0 else o.mul(r)).view(g.shape).to(g.dtype)
        return (_tree.rebuild(new_g, updates, g_spec),
                ScaleByMuonState(momentum=_tree.rebuild(new_m, state.momentum, m_spec),
                                 scales=state.scales))

    return GradientTransformation(init_fn, update_fn)
