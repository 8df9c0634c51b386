"""A shared expert in 8-bit floating point: the experts of a layer that every token passes
(``deepseek_vl2/deepseek_layers.py:600-729`` adds them beside the routed ones; they never take
part in the lookup). The routed experts are ``table_moe.ops.Fp8Experts``."""
from __future__ import annotations

import torch

from ..ops.fp8 import Fp8Linear


class Fp8SharedExpert:
    """down(silu(gate x) * (up x)) on two ``Fp8Linear``: ``gate_up`` [2 I, H] (gate rows, then up
    rows) and ``down`` [H, I]."""

    def __init__(self, gate_up: Fp8Linear, down: Fp8Linear):
        if gate_up.n != 2 * down.k or gate_up.k != down.n:
            raise ValueError(f"gate_up [{gate_up.n}, {gate_up.k}] and down [{down.n}, {down.k}] do not fit")
        self.gate_up, self.down = gate_up, down

    @classmethod
    def quantize(cls, gate_up, down):
        return cls(Fp8Linear.quantize(gate_up), Fp8Linear.quantize(down))

    def __call__(self, x, *, out_dtype=None):
        gate, up = self.gate_up(x, out_dtype=torch.float32).chunk(2, dim=-1)
        return self.down(torch.nn.functional.silu(gate) * up, out_dtype=out_dtype or x.dtype)
