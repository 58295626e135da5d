"""ThetaScan on MI355X: the public API of the reference package with a
hand-written gfx950 ``hip`` scan backend underneath."""
from .api import ThetaScan
from .state import ThetaScanState
from .decode import DecodeGraph
from .delta import GatedDelta, GatedDeltaConfig
from ._core.ops.delta import gated_delta_rule
from ._core.ops.policy import policy_loss, token_log_probs
from .config import (
    Backend,
    BankMode,
    BlendMode,
    Family,
    GNConfig,
    GNNonlinearity,
    GNReadNormalization,
    KernelBSplineScaleMode,
    KernelConfig,
    KernelFeatureMap,
    KernelReLU2ThresholdMode,
    KernelReadNormalization,
    KernelSharpnessMode,
    KernelSparsity,
    KernelValueRepresentation,
    RegularizationConfig,
    RoPEConfig,
    RoPEMode,
    RoPEPlacement,
    RuntimeConfig,
    TemporalConfig,
    TemporalMode,
    ThetaScanConfig,
)

__version__ = "0.1.0"

__all__ = [
    "Backend", "BankMode", "BlendMode", "Family", "GNConfig", "GNNonlinearity", "GNReadNormalization",
    "GatedDelta", "GatedDeltaConfig",
    "DecodeGraph", "KernelBSplineScaleMode", "KernelConfig", "KernelFeatureMap", "KernelReLU2ThresholdMode",
    "KernelReadNormalization", "KernelSharpnessMode", "KernelSparsity", "KernelValueRepresentation",
    "RegularizationConfig", "RoPEConfig", "RoPEMode", "RoPEPlacement", "RuntimeConfig", "TemporalConfig",
    "TemporalMode", "ThetaScan", "ThetaScanConfig", "ThetaScanState", "gated_delta_rule", "policy_loss",
    "token_log_probs",
]
