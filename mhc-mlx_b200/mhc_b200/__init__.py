"""mhc_b200: the mHC (manifold-constrained hyper-connections) hot path of
svdrecbd/mhc-mlx, rebuilt for NVIDIA B200 (sm_100a).

Public API mirrors mhc_mlx: MHCLayer, MHCRewire, AutoPatcher,
residual_add_agg, diagnostics; the launcher-level entry points live in
mhc_b200.metal under the reference's names.
"""

from .diagnostics import diagnostics
from .layer import MHCLayer, MHCRewire
from .linear import FusedLinear, linear_act
from .losses import (policy_loss, policy_loss_grad, preference_loss, preference_loss_grad,
                     token_logprobs)
from .optim import AdamW
from .patching import AutoPatcher
from .quantized import QuantizedLinear
from .utils import residual_add_agg

__version__ = "1.0.0"

__all__ = ["MHCLayer", "MHCRewire", "diagnostics", "residual_add_agg", "AutoPatcher",
           "QuantizedLinear", "token_logprobs", "preference_loss", "preference_loss_grad",
           "policy_loss", "policy_loss_grad", "AdamW", "linear_act", "FusedLinear",
           "__version__"]
