"""`FusedMuon`: the classic Muon optimizer with its whole step -- momentum, look-ahead,
orthogonalisation, weight decay and the addition to the parameters -- on the operators of
`torchopt_amd._C.muon_op`, one call per device and dtype for any number of parameters.

The reference has no counterpart.  Constructor arguments are those of ``torch.optim.Muon``; parameters come as
tensors (dicts of groups are refused, `add_param_group` takes another list), with the same settings for all
groups.  The step:

    ``M <- momentum * M + g``,   ``U = g + momentum * M`` (``nesterov``; else ``U = M``),
    ``P <- (1 - lr * weight_decay) * P - lr * r * orthogonalize(U)``

with ``r`` after `adjust_lr_fn` (see `scale_by_muon`).  Beside ``torch.optim.Muon``:

  * the momentum is the plain sum, not the mean of the gradients, which is ``1 - momentum`` times it;
    the normalisation takes the factor out again (but for `eps`);
  * the series runs on operands of 22 significant bits with float32 sums, not in bfloat16, whatever the
    parameters' type;
  * `ns_steps` is at most 32 (there 99), and coefficients under which an iterate could grow beyond 64 are
    refused by the first step;
  * parameters of more than two dimensions are taken too, as the matrix of their first dimension
    times all the others (a convolution's kernel); vectors and scalars are refused;
  * `momentum_dtype=torch.int8` keeps the momentum in 8-bit blocks: a quarter of float32's
    memory.  Each step reads the blocks, updates and writes them again, rounded to the nearest of
    255 multiples of a block's scale; the update is computed from what is kept;
  * nothing of the step depends on a step number, so it can be captured in a HIP graph (with a
    constant learning rate, which the graph then holds); `init_state()` or one step has to come
    before, so that the momentum exists outside the graph.
"""

from __future__ import annotations

from typing import Any, Callable, Iterable, Sequence

import torch

from torchopt_amd.accelerated_op.library import dispatch
from torchopt_amd.accelerated_op.muon_op import (COEFFICIENTS, dequantize_blocks,
                                                 quantize_blocks)
from torchopt_amd.transform.scale_by_muon import (ScaleByMuonState, check_muon, require_matrix,
                                                  zero_momentum)


__all__ = ['FusedMuon', 'Muon']


class FusedMuon:
    """Muon for matrix-shaped GPU parameters (float32, float16, bfloat16)."""

    def __init__(
        self,
        params: Iterable[torch.Tensor],
        lr: float | Callable[[int], float] = 1e-3,
        weight_decay: float = 0.1,
        momentum: float = 0.95,
        nesterov: bool = True,
        ns_coefficients: tuple[float, float, float] = COEFFICIENTS,
        eps: float = 1e-7,
        ns_steps: int = 5,
        adjust_lr_fn: str | None = None,
        *,
        maximize: bool = False,
        momentum_dtype: torch.dtype | None = None,
    ) -> None:
        if not callable(lr) and not lr >= 0.0:
            raise ValueError(f'Invalid learning rate: {lr}')
        if not weight_decay >= 0.0:
            raise ValueError(f'Invalid weight_decay value: {weight_decay}')
        check_muon(momentum, ns_steps, ns_coefficients, eps, adjust_lr_fn, momentum_dtype)
        self.lr, self.weight_decay, self.momentum, self.nesterov = lr, weight_decay, momentum, nesterov
        self.ns_coefficients, self.eps, self.ns_steps = tuple(ns_coefficients), eps, int(ns_steps)
        self.adjust_lr_fn, self.maximize, self.momentum_dtype = adjust_lr_fn, maximize, momentum_dtype
        self.param_groups: list[tuple[torch.Tensor, ...]] = []
        self.state_groups: list[ScaleByMuonState | None] = []
        self._taken: list[int] = []  # steps taken, for a learning-rate schedule
        self.add_param_group(params)

    def add_param_group(self, params: Iterable[torch.Tensor]) -> None:
        group = tuple(params)
        for p in group:
            if not isinstance(p, torch.Tensor):
                raise TypeError(f'expected tensors, got {type(p).__name__}')
            require_matrix(p, type(self).__name__)
        self.param_groups.append(group)
        self.state_groups.append(None)  # built on the first step, like the reference's
        self._taken.append(0)

    def zero_grad(self, set_to_none: bool = False) -> None:
        for group in self.param_groups:
            for p in group:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    if p.grad.grad_fn is not None:
                        p.grad.detach_()
                    else:
                        p.grad.requires_grad_(False)
                    p.grad.zero_()

    def init_state(self) -> None:
        """Create the momentum now (the first `step()` does otherwise), e.g. before capturing
        `step()` in a graph."""
        for i, group in enumerate(self.param_groups):
            if self.state_groups[i] is None:
                kept = [zero_momentum(p, self.momentum_dtype) for p in group]
                self.state_groups[i] = ScaleByMuonState(momentum=tuple(m for m, _ in kept),
                                                        scales=tuple(s for _, s in kept))

    def state_dict(self) -> tuple:
        """Per group ``(steps taken, ScaleByMuonState)`` with the tensors that steps go on to change, or
        None before the first step."""
        return tuple(None if s is None else (n, s) for n, s in zip(self._taken, self.state_groups))

    def load_state_dict(self, state_dict: Sequence[Any]) -> None:
        """Takes a copy of the state of `state_dict()`, which steps then leave as it is.  A momentum
        kept in another type (one in 8-bit blocks into an optimizer that keeps float32, or the other
        way round) is converted."""
        if len(state_dict) != len(self.param_groups):
            raise ValueError(f'expected the state of {len(self.param_groups)} groups, got '
                             f'{len(state_dict)}')
        taken, groups = [], []
        for group, entry in zip(self.param_groups, state_dict):
            if entry is None:
                taken.append(0)
                groups.append(None)
                continue
            n, state = entry
            momentum, scales = list(state.momentum), list(state.scales)
            if len(momentum) != len(group) or len(scales) != len(group):
                raise ValueError('state and parameters differ in length')
            for k, p in enumerate(group):
                if momentum[k].shape != p.shape:
                    raise ValueError(f'state of shape {tuple(momentum[k].shape)} for a parameter '
                                     f'of shape {tuple(p.shape)}')
                momentum[k], scales[k] = self._kept(p, momentum[k], scales[k])
            taken.append(int(n))
            groups.append(ScaleByMuonState(momentum=tuple(momentum), scales=tuple(scales)))
        self._taken[:], self.state_groups[:] = taken, groups

    def _kept(self, p: torch.Tensor, m: torch.Tensor, scales: torch.Tensor | None):
        """A momentum and its scales in the type, place and memory layout this optimizer keeps for
        `p`, from any other, in memory of their own."""
        kind = p.dtype if self.momentum_dtype is None else self.momentum_dtype
        same_layout = m.stride() == torch.empty_like(p, device='meta').stride()
        m = m.detach().to(p.device, copy=True)
        if scales is not None:
            scales = scales.detach().to(p.device, copy=True)
            if kind == torch.int8 and same_layout:
                return m, scales
            m = dequantize_blocks(m, scales, torch.float32)
        if kind == torch.int8:
            # (blocks follow the memory order, so the layout comes first)
            return quantize_blocks(torch.empty_like(p, dtype=torch.float32).copy_(m))
        if m.dtype == kind and same_layout:
            return m, None
        return torch.empty_like(p, dtype=kind).copy_(m), None

    @torch.no_grad()
    def step(self, closure: Callable[[], torch.Tensor] | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            if callable(self.lr):
                raise RuntimeError('FusedMuon.step(): a schedule is evaluated on the host, which '
                                   'a captured graph would freeze; use a constant learning rate')
            if any(s is None for s in self.state_groups):
                raise RuntimeError('FusedMuon: take one step (or call init_state()) before '
                                   'capturing, so that the state exists outside the graph')
        self.init_state()
        for i, (group, state) in enumerate(zip(self.param_groups, self.state_groups)):
            lr = float(self.lr(self._taken[i])) if callable(self.lr) else self.lr
            buckets: dict[tuple, list[int]] = {}
            for k, p in enumerate(group):
                if p.grad is not None:
                    buckets.setdefault((p.device, p.dtype), []).append(k)
            if not buckets:
                continue
            self._taken[i] += 1
            for ks in buckets.values():
                scales = None
                if state.scales[ks[0]] is not None:
                    scales = [state.scales[k] for k in ks]
                dispatch.muon_fused_step_multi_(
                    [group[k] for k in ks], [group[k].grad for k in ks],
                    [state.momentum[k] for k in ks], scales, self.momentum, lr,
                    nesterov=self.nesterov, weight_decay=self.weight_decay,
                    maximize=self.maximize, steps=self.ns_steps,
                    coefficients=self.ns_coefficients, eps=self.eps,
                    adjust_lr_fn=self.adjust_lr_fn)
        return loss


# the name torch.optim has
Muon = FusedMuon
