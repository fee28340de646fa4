"""Group normalisation with an activation, for channels-last maps (csrc/groupnorm.hip).

The counterpart of the fused BatchNorm+activation (ops/bnrelu.py) for networks
without batch statistics: small batches, accumulated gradients, evaluation that
is the same function as training.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import require_ext_for

ACTS = {"none": 0, "relu": 1, "swish": 2}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, num_groups, weight, bias, eps, act):
    if act not in ACTS:
        raise ValueError(f"group_norm_act: act={act!r} is none of {sorted(ACTS)}")
    if x.dim() < 2:
        raise ValueError("group_norm_act: x is [N, C, ...]")
    if x.dtype not in DTYPES:
        raise TypeError(f"group_norm_act: x is fp32, bf16 or fp16, not {x.dtype}")
    c = x.size(1)
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"group_norm_act: {c} channels cannot be {num_groups} groups")
    if not eps >= 0.0:
        raise ValueError("group_norm_act: eps >= 0 is needed")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (c,):
            raise ValueError(f"group_norm_act: {name} is [{c}], not {list(p.shape)}")
        if p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"group_norm_act: {name} is of x's type or fp32, not {p.dtype}")
        if p.device != x.device:
            raise ValueError(f"group_norm_act: {name} is on {p.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("group_norm_act: weight and bias are of one type")


def _composed(x, num_groups, weight, bias, eps, act):
    """The CPU path, which also defines the kernels' semantics."""
    z = x.float()
    if x.numel():
        z = z.reshape(x.size(0), num_groups, -1)
        z = z - z.mean(2, keepdim=True)
        z = (z * (z.square().mean(2, keepdim=True) + eps).rsqrt()).reshape(x.shape)
    column = (1, -1) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * weight.float().view(column)
    if bias is not None:
        z = z + bias.float().view(column)
    z = F.relu(z) if act == "relu" else F.silu(z) if act == "swish" else z
    return z.to(x.dtype)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                   act: str = "none") -> torch.Tensor:
    """act(weight * (x - mean) / sqrt(var + eps) + bias), statistics over groups of channels.

    x: [N, C, ...] in fp32, bf16 or fp16; mean and variance (biased) are taken
    for each sample over the C / num_groups channels of a group and all pixels.
    ``weight`` and ``bias`` are [C] or None, in x's type or fp32. ``act`` is
    "none", "relu" or "swish". Everything is computed in fp32 and rounded once.
    On the GPU the result is channels last (a map of another order is copied
    into it first), and gradients go to x, weight and bias, once. There a sample
    has fewer than 2^31 values, a group at most 16384 channels, and N times the
    groups, or the workgroups they are cut into, stay below 2^24; more is refused.
    """
    _check(x, num_groups, weight, bias, eps, act)
    if not x.is_cuda:
        return _composed(x, num_groups, weight, bias, eps, act)
    return require_ext_for(x).group_norm_act(x, num_groups, weight, bias, eps, ACTS[act])


class GroupNormAct(torch.nn.GroupNorm):
    """nn.GroupNorm on ``group_norm_act`` where that has x's type; ``ops.modules`` fuses the activation that follows it."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dtype not in DTYPES:
            return super().forward(x)
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps)
