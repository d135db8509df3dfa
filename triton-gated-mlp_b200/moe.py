"""FusedMoEGatedMLP: a mixture of gated MLPs for inference on sm_100a kernels.

The layer that stands in FusedGatedMLP's place in a mixture-of-experts block:
  y[t] = sum_j weights[t, j] * MLP_{ids[t, j]}(x[t]) (+ residual[t])
with ids and weights from a linear router (softmax over all experts, the top_k largest, optionally divided by their
sum) and MLP_e the gated MLP of FusedGatedMLP without biases. Three launches for up to 64 tokens (router, gate/up of
the chosen experts, their down projections), five on 4-bit experts from 5 tokens on (before each of the two a kernel
that makes the activations' terms); only the experts that some token chose are read. There is no counterpart
in the reference, whose module has one MLP (src/triton_gated_mlp/gated_mlp.py:203-237).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from .ops import kernels
from .ops.fwd import SUPPORTED_ACTS


class FusedMoEGatedMLP(nn.Module):
    """Inference-only mixture of gated MLPs in bfloat16 or float16; see the module docstring.

    Parameters: router.weight [num_experts, hidden], gate_proj and up_proj [num_experts, intermediate, hidden],
    down_proj [num_experts, hidden, intermediate]. forward takes any number of leading dimensions and any number of
    tokens; the kernels work on 64 tokens at a time, so that a call of more tokens reads the experts once per 64
    of them. There is no backward pass: forward raises where a gradient would be needed. No host synchronisation:
    a call can be captured into a CUDA graph."""

    def __init__(self, hidden_size: int, intermediate_size: int, num_experts: int, top_k: int,
                 hidden_act: str = "silu", *, renormalize: bool = True):
        super().__init__()
        if hidden_act not in SUPPORTED_ACTS:
            raise NotImplementedError(f"gate activation {hidden_act!r}: supported are {sorted(SUPPORTED_ACTS)}")
        if not 1 <= num_experts <= kernels.MOE_MAX_EXPERTS:
            raise ValueError(f"{num_experts} experts: 1 to {kernels.MOE_MAX_EXPERTS} are supported")
        if not 1 <= top_k <= min(num_experts, kernels.MOE_MAX_TOP_K):
            raise ValueError(f"top_k={top_k}: 1 to {min(num_experts, kernels.MOE_MAX_TOP_K)} are supported for "
                             f"{num_experts} experts")
        if hidden_size <= 0 or intermediate_size <= 0 or hidden_size % 64 or intermediate_size % 64:
            raise ValueError("mixtures of experts need hidden_size and intermediate_size multiples of 64; got "
                             f"{hidden_size} and {intermediate_size}")
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.num_experts, self.top_k = num_experts, top_k
        self.act_fn = hidden_act
        self.renormalize = bool(renormalize)
        self.router = nn.Linear(hidden_size, num_experts, bias=False)
        self.gate_proj = nn.Parameter(torch.empty(num_experts, intermediate_size, hidden_size))
        self.up_proj = nn.Parameter(torch.empty(num_experts, intermediate_size, hidden_size))
        self.down_proj = nn.Parameter(torch.empty(num_experts, hidden_size, intermediate_size))
        for p in (self.gate_proj, self.up_proj, self.down_proj):   # nn.Linear's range, expert by expert
            nn.init.uniform_(p, -p.shape[-1] ** -0.5, p.shape[-1] ** -0.5)
        self._w4 = None

    def quantize_decode_weights(self, enable: bool = True, bits: int = 4, group_size: int = 128) -> None:
        """Prepare (or drop) 4-bit copies of the experts with one scale and zero point per `group_size` (32, 64 or
        128) columns; forward then streams a quarter of the weight bytes. Call again after the weights change.
        Needs hidden and intermediate sizes that are multiples of the group size."""
        if not enable:
            self._w4 = None
            return
        if bits != 4:
            raise NotImplementedError(f"{bits}-bit experts: 4 bits are supported")
        if group_size not in kernels.INT4_GROUPS or self.hidden_size % group_size or self.intermediate_size % group_size:
            raise ValueError(f"4-bit experts need a group size in {kernels.INT4_GROUPS} that divides hidden_size and "
                             f"intermediate_size; got {group_size}")
        self._w4 = tuple(_quantize_experts(p, group_size) for p in (self.gate_proj, self.up_proj, self.down_proj))

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters())
                                        or (residual is not None and residual.requires_grad)):
            raise NotImplementedError("FusedMoEGatedMLP has no backward pass: call it under torch.no_grad()")
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != input shape {tuple(x.shape)}")
        rows = x.reshape(-1, x.shape[-1])
        res = None if residual is None else residual.reshape(-1, x.shape[-1])
        ids, weights = kernels.moe_route(rows, self.router.weight, self.top_k, self.renormalize)
        out = []
        step = kernels.DECODE_MAX_TOKENS
        for t in range(0, max(rows.shape[0], 1), step):
            part = slice(t, t + step)
            args = (rows[part], ids[part], weights[part])
            kw = dict(act=self.act_fn, residual=None if res is None else res[part])
            if self._w4 is not None:
                out.append(kernels.moe_decode_fwd_w4(*args, *self._w4, **kw))
            else:
                out.append(kernels.moe_decode_fwd(*args, self.gate_proj, self.up_proj, self.down_proj, **kw))
        return (out[0] if len(out) == 1 else torch.cat(out)).view(x.shape)


def _quantize_experts(p: Tensor, group: int) -> kernels.Int4Weight:
    """quantize_weight_int4 expert by expert: its float32 copies are then those of one expert."""
    w4, scale, zero = zip(*(kernels.quantize_weight_int4(w, group) for w in p.detach()))
    return kernels.Int4Weight(torch.stack(w4), torch.stack(scale), torch.stack(zero))
