"""Model-side adapter of the ALUT path: the cached MoE layer forward on the ALUT kernels."""
from .fp8_moe import Fp8SharedExpert
from .fused_moe import ALUTCachedMoE

__all__ = ["ALUTCachedMoE", "Fp8SharedExpert"]
