"""MI355X-native fused Adam operator: a drop-in for TorchOpt's accelerated Adam op.

    from torchopt_amd._C import adam_op                    # the 7-function native surface
    from torchopt_amd.accelerated_op import AdamOp         # the per-leaf callable
    from torchopt_amd import accelerated_op_available
    from torchopt_amd import orthogonalize, Muon, muon     # matrix-shaped parameters
"""

import sys as _sys

from torchopt_amd import accelerated_op
from torchopt_amd.accelerated_op import (AdamOp, MultiAdamOp, dequantize_blocks, orthogonalize,
                                         quantize_blocks)
from torchopt_amd.accelerated_op import is_available as accelerated_op_available
from torchopt_amd.alias import adam, adamw, apply_updates, chain, muon
from torchopt_amd.func import FuncOptimizer
from torchopt_amd.meta import MetaAdam, MetaAdamW, MetaMuon
from torchopt_amd.optim import Adam, AdamW, FusedAdam, FusedAdamW
from torchopt_amd.optim_muon import FusedMuon, Muon
from torchopt_amd.placement import (placed_like_tree, state_empty_like, state_zeros_like,
                                    state_zeros_like_tree, unshared)

# `import torchopt_amd._C.adam_op` should work like `from torchopt_amd._C import adam_op`
from torchopt_amd import _C  # noqa: E402

_sys.modules.setdefault('torchopt_amd._C.adam_op', _C.adam_op)
_sys.modules.setdefault('torchopt_amd._C.muon_op', _C.muon_op)

__version__ = '0.1.0'

__all__ = ['Adam', 'AdamOp', 'AdamW', 'FuncOptimizer', 'FusedAdam', 'FusedAdamW', 'FusedMuon', 'MetaAdam', 'MetaAdamW',
           'MetaMuon', 'MultiAdamOp', 'Muon', 'accelerated_op',
           'accelerated_op_available', 'adam', 'adamw', 'apply_updates', 'chain', 'dequantize_blocks',
           'muon', 'orthogonalize', 'placed_like_tree', 'quantize_blocks', 'state_empty_like', 'state_zeros_like', 'state_zeros_like_tree', 'unshared']
