"""`orthogonalize`: Newton-Schulz orthogonalisation of matrices, differentiable, and the 8-bit
blocks an optimizer can keep its momentum in.

The reference has no counterpart; the manners are those of `AdamOp`: `torchopt_amd._C.muon_op`
(hand-written gfx950 kernels) and nothing else behind it, GPU tensors only, work on the current
stream, whole lists in one call.

For a matrix ``G`` with ``X = G / (|G|_F + eps)``, each of `steps` times

    ``X <- a X + b (X X^T) X + c (X X^T)^2 X``

takes the singular values of ``X`` through the polynomial ``a t + b t^3 + c t^5`` and leaves its
singular vectors: with the default coefficients every singular value that is not tiny ends between
0.7 and 1.2, so the result is close to the nearest matrix with orthonormal rows (or columns).

The gradient is the formula's own (through every step and the norm), not that of an ideal
orthogonalisation.  It needs every iterate.  Autograd keeps them between the passes where a call's take
no more than `KEEP_BYTES`; for more (and for small matrices, whose iterates are made again faster than
they are read) it keeps the input alone and the gradient makes them again: eight 1024 x 1024 float32
matrices and their gradient take 2.7 ms that way and 2.1 with 0.6 GiB kept.  The gradient is not
differentiable a second time, and forward-mode derivatives are refused.
"""

from __future__ import annotations

import operator
from typing import Any, Sequence

import torch

try:
    from torchopt_amd._C import muon_op
except ImportError as exc:  # no fallback module: the op is the compiled extension or nothing
    raise ImportError(
        'torchopt_amd._C, the compiled extension in front of libtoa_muon.so, cannot be '
        f'imported ({exc}); build it with `python torchopt_amd/build.py`. There is no '
        'pure-Python or CPU fallback.') from exc

from torch.autograd.function import once_differentiable

# the same functions, visible to torch.compile while it traces
from torchopt_amd.accelerated_op import library  # noqa: E402, F401


__all__ = ['COEFFICIENTS', 'KEEP_BYTES', 'dequantize_blocks', 'orthogonalize', 'quantize_blocks']

# the quintic whose slope at zero is steep (small singular values grow 3.4-fold a step) at the
# price of ending near one instead of at it
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

# Iterates that autograd may keep for one call, in bytes: five steps of a square matrix keep 80 for each
# of its elements, so this is 13 million elements (an update of 50 MB in float32).
KEEP_BYTES = 1 << 30


class _Orthogonalize(torch.autograd.Function):
    """All matrices of a list as one node."""

    @staticmethod
    def forward(ctx: Any, series: tuple, *inputs: torch.Tensor):
        ctx.series = series
        ctx.set_materialize_grads(False)
        outputs, kept = muon_op.orthogonalize_keep_multi(inputs, KEEP_BYTES, *series)
        ctx.save_for_backward(kept, *inputs)
        return tuple(outputs)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, *grads: torch.Tensor | None):
        kept, *inputs = ctx.saved_tensors
        live = [k for k, g in enumerate(grads) if g is not None and ctx.needs_input_grad[1 + k]]
        out: list[torch.Tensor | None] = [None] * len(inputs)
        if live:
            # (the iterates of the whole list are of no use for a part of it)
            fresh = muon_op.orthogonalize_backward_multi(
                [grads[k] for k in live], [inputs[k] for k in live], *ctx.series,
                kept if len(live) == len(inputs) else None)
            for k, g in zip(live, fresh):
                out[k] = g
        return (None, *out)


def _by_kind(tensors: Sequence[torch.Tensor]) -> list[list[int]]:
    """Positions of the tensors of each device and dtype."""
    if _one_kind(tensors):
        return [list(range(len(tensors)))]
    kinds: dict[tuple, list[int]] = {}
    for k, t in enumerate(tensors):
        kinds.setdefault((t.device, t.dtype), []).append(k)
    return list(kinds.values())


def _one_kind(tensors: Sequence[torch.Tensor]) -> bool:
    first = tensors[0]
    return all(t.dtype is first.dtype and t.device == first.device for t in tensors)


def orthogonalize(
    matrices: torch.Tensor | Sequence[torch.Tensor],
    *,
    steps: int = 5,
    coefficients: tuple[float, float, float] = COEFFICIENTS,
    eps: float = 1e-7,
):
    """Orthogonalise a tensor of matrices (its last two dimensions), or every tensor of a list or
    tuple, whose shapes, dtypes and devices may differ.

    Args:
        matrices: GPU tensors of float32, float16 or bfloat16, any strides.
        steps: how often the polynomial is applied, 1 to 32.
        coefficients: ``(a, b, c)``.  Coefficients under which an iterate but the last could grow
            beyond 64 are refused.
        eps: added to the Frobenius norm.

    Returns:
        A tensor like `matrices` (a list or tuple of them for a list or tuple), differentiable
        with respect to it.  Results come from products with 22-bit operands and float32 sums;
        for bfloat16 the operands of the last step may carry 11 bits, where the coefficients keep
        what that adds within half a step of the type (the default ones do not).
    """
    single = isinstance(matrices, torch.Tensor)
    tensors = [matrices] if single else list(matrices)
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'orthogonalize: expected tensors, got {type(t).__name__}')
    series = (operator.index(steps), tuple(float(c) for c in coefficients), float(eps))
    out: list[torch.Tensor | None] = [None] * len(tensors)
    grad = torch.is_grad_enabled()
    for ks in _by_kind(tensors) if tensors else []:
        group = [tensors[k] for k in ks]
        if torch.compiler.is_compiling():
            fresh = torch.ops.torchopt_amd.orthogonalize_multi(group, series[0], list(series[1]),
                                                               series[2])
        elif grad and any(t.requires_grad for t in group):
            fresh = _Orthogonalize.apply(series, *group)
        else:
            fresh = muon_op.orthogonalize_multi(group, *series)
        for k, y in zip(ks, fresh):
            out[k] = y
    if single:
        return out[0]
    return out if isinstance(matrices, list) else tuple(out)


def quantize_blocks(tensors: torch.Tensor | Sequence[torch.Tensor]):
    """8-bit blocks of a dense tensor, or of every tensor of a list: ``(codes, scales)``.

    Each 128 consecutive elements in memory order (the last ones may be fewer) share one float32
    scale, the largest magnitude among them over 127; the int8 code of an element is its multiple
    of the scale, rounded half to even.  So an element is off by half a scale at most, and a block
    of zeros stays one.  A block with a NaN or an infinity stands for NaN throughout.  Neither this nor
    `dequantize_blocks` is differentiable."""
    if isinstance(tensors, torch.Tensor):
        codes, scales = muon_op.quantize_multi([tensors])
        return codes[0], scales[0]
    codes: list = [None] * len(tensors)
    scales: list = [None] * len(tensors)
    for ks in _by_kind(tensors) if len(tensors) else []:
        for k, c, s in zip(ks, *muon_op.quantize_multi([tensors[k] for k in ks])):
            codes[k], scales[k] = c, s
    return codes, scales


def dequantize_blocks(codes, scales, dtype: torch.dtype = torch.float32):
    """What `quantize_blocks` made, as a tensor (or list of tensors) of `dtype`."""
    if isinstance(codes, torch.Tensor):
        out = torch.empty_like(codes, dtype=dtype)
        return muon_op.dequantize_multi_([out], [codes], [scales])[0]
    out = [torch.empty_like(c, dtype=dtype) for c in codes]
    by_device: dict[torch.device, list[int]] = {}
    for k, c in enumerate(codes):
        by_device.setdefault(c.device, []).append(k)
    for ks in by_device.values():
        muon_op.dequantize_multi_([out[k] for k in ks], [codes[k] for k in ks],
                                  [scales[k] for k in ks])
    return out
