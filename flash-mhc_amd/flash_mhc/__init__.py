"""flash-mHC for MI355X: the mHC-lite K1/K3/K4 fused path on gfx950 HIP kernels.

Importing the package registers the ``torch.ops.flash_mhc.*`` custom ops.
Beyond the reference's names it has ``LayerNorm`` / ``layer_norm`` and, for
activations kept in 8 bits, ``pack8`` / ``unpack8``.
The HIP extension itself is loaded on first use (see ``flash_mhc._abi``).
"""

from .block import MHCLiteBlock, build_permutation_matrices
from . import ops as _ops  # noqa: F401  # registers the torch.library ops
from .activation8 import pack8, unpack8  # noqa: F401
from .norm import LayerNorm, layer_norm  # noqa: F401

# What `from flash_mhc import *` gives: the reference's names.
__all__ = ["MHCLiteBlock", "build_permutation_matrices"]
