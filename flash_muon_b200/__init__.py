"""B200-native (sm_100a) Muon hot path: drop-in for the operator interface of nil0x9/flash-muon.

Exports the reference's four names (flash_muon/__init__.py:1-4) and, for the parameters Muon does
not take, AdamW and the clipping of gradients.  Everything runs through the
C-ABI library ``libflash_muon_b200.so``; importing the package fails if it has not been built.
"""
from .ops import (fast_newtonschulz, matmul_transpose, matmul_transpose_assign,
                  newtonschulz_workspace_bytes)
from .muon import Muon
from .adamw import (AdamW, adamw8_encode, adamw8_step, adamw8_values, adamw_step, clip_grad_norm_,
                    grad_norm)

__all__ = ["matmul_transpose", "matmul_transpose_assign", "fast_newtonschulz", "Muon",
           "newtonschulz_workspace_bytes", "AdamW", "adamw_step", "adamw8_step", "adamw8_values",
           "adamw8_encode", "grad_norm", "clip_grad_norm_"]
