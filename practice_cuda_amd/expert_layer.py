"""Layers of experts: trained on the package's products, and served in int8.

``ExpertMLP`` sends each token to its experts' gated two-product networks,

    y[t] = sum_j weights[t, j] down_e(silu(gate_e(x[t])) * up_e(x[t])),  e = ids[t, j]

with ``expert_sort``, ``expert_dispatch`` and ``expert_combine`` around one
``BMMLinear`` pair an expert, so ``convert_to_float8_bmm_training`` makes it an
fp8 layer and gradients reach tokens, weights and the router's weights.
``Int8Experts`` is the served form: int8 codes of all experts in two tensors,
and both products grouped by expert in one launch each, the tokens' rows found
within the first. The reference has the batched layer that the experts are made
of (fp8_training/fp8_bench/modules/bmm_linear.py), not the routing.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .impls._common import without_gradient
from .impls.hip_expert import hip_expert_bmm, hip_expert_combine, hip_expert_dispatch, hip_expert_sort
from .impls.hip_int8 import hip_int8_quant
from .modules import BMMLinear
from .registry import QuantResult


class ExpertMLP(nn.Module):
    """experts x (hidden -> 2 inner gates and others -> hidden), without biases.

    ``forward(x, ids, weights)``: x [T, hidden], ids [T, k] the experts of each
    token (negative: none), weights [T, k]. Reads the group sizes back to the
    host, as each expert's products are calls of their own."""

    def __init__(self, hidden: int, inner: int, experts: int, *, device=None, dtype=None) -> None:
        super().__init__()
        if experts <= 0:
            raise ValueError(f"experts must be positive, got {experts}")
        self.hidden, self.inner, self.experts = hidden, inner, experts
        kw = {"bias": False, "device": device, "dtype": dtype}
        self.gate_up = nn.ModuleList([BMMLinear(1, hidden, 2 * inner, **kw) for _ in range(experts)])
        self.down = nn.ModuleList([BMMLinear(1, inner, hidden, **kw) for _ in range(experts)])

    def forward(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        plan = hip_expert_sort(ids, self.experts)
        rows = hip_expert_dispatch(x, plan)
        starts = plan.starts.tolist()
        parts = []
        for e in range(self.experts):
            if starts[e + 1] > starts[e]:
                gate, up = self.gate_up[e](rows[None, starts[e]:starts[e + 1]]).chunk(2, -1)
                parts.append(self.down[e](F.silu(gate) * up)[0])
        parts.append(rows[starts[-1]:])  # pairs without an expert: zeros
        return hip_expert_combine(torch.cat(parts), plan, weights)

    def served(self) -> "Int8Experts":
        """The int8 form of the weights as they are now."""
        with torch.no_grad():
            return Int8Experts(torch.cat([m.weight for m in self.gate_up]), torch.cat([m.weight for m in self.down]))


class Int8Experts(nn.Module):
    """Experts served in int8: codes of gate_up [E, 2 inner, hidden] and down [E, hidden, inner].

    Weights have a scale for each output channel, activations one for each
    token. hidden and inner are multiples of 16. ``forward(x, ids, weights)``
    takes bfloat16 or float16 [T, hidden]; nothing is read back to the host."""

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor) -> None:
        super().__init__()
        if gate_up.ndim != 3 or down.ndim != 3 or down.shape[0] != gate_up.shape[0] or (
                gate_up.shape[1:] != (2 * down.shape[2], down.shape[1])):
            raise ValueError("gate_up must be [E, 2 inner, hidden] and down [E, hidden, inner], got "
                             f"{tuple(gate_up.shape)} and {tuple(down.shape)}")
        if down.shape[1] % 16 or down.shape[2] % 16:
            raise ValueError(f"hidden and inner must be multiples of 16, got {tuple(down.shape[1:])}")
        self.experts, self.hidden, self.inner = down.shape
        for name, w in (("gate_up", gate_up), ("down", down)):
            q = hip_int8_quant(w.detach().transpose(1, 2), channel_axis=-1)
            self.register_buffer(name, q.tensor.transpose(1, 2))  # [E, out, in]
            self.register_buffer(f"{name}_scale", q.dequant_scale)

    def _apply(self, fn, recurse=True):
        """Type changes leave the scales in 32 bits."""
        kept = {n: getattr(self, n) for n in ("gate_up_scale", "down_scale")}
        super()._apply(fn, recurse)
        for name, old in kept.items():
            new = getattr(self, name)
            if new.dtype != torch.float32:
                setattr(self, name, old.to(new.device))
        return self

    def _weight(self, name: str) -> QuantResult:
        return QuantResult(getattr(self, name).transpose(1, 2), getattr(self, f"{name}_scale"), "hip_int8", "channel",
                           {"channel_axis": -1})

    def forward(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        if torch.is_grad_enabled() and (x.requires_grad or weights.requires_grad):
            with torch.no_grad():
                y = self._serve(x, ids, weights)
            return without_gradient(type(self).__name__, (x, weights), y)[0]
        return self._serve(x, ids, weights)

    def _serve(self, x, ids, weights):
        plan = hip_expert_sort(ids, self.experts)
        h = hip_expert_bmm(hip_int8_quant(x), self._weight("gate_up"), plan, gather=True, out_dtype=x.dtype,
                           activation="swiglu")
        y = hip_expert_bmm(hip_int8_quant(h), self._weight("down"), plan, out_dtype=x.dtype)
        return hip_expert_combine(y, plan, weights)


__all__ = ["ExpertMLP", "Int8Experts"]
