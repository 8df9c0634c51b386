"""Ops of the TableMoE layers on sm_100a: the router (``qwen_topk_softmax``, drop-in for the
reference's ``table_moe/ops``; ``route_experts`` with sigmoid scores, a balance bias and expert
groups) and products in 8-bit floating point (``Fp8Linear``, ``Fp8Experts``, ``quantize_fp8``).
The fp16 fused expert MLP of the reference's package is not provided."""
from .expert_routing import route_experts
from .fp8 import Fp8Experts, Fp8Linear, quantize_fp8
from .qwen_topk_softmax import qwen_topk_softmax, route_for_lookup

__all__ = ["qwen_topk_softmax", "route_for_lookup", "route_experts", "Fp8Experts", "Fp8Linear", "quantize_fp8"]
