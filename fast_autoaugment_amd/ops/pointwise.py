"""Matrix product with bias, residual and activation in one kernel (csrc/pointwise.hip).

``linear_act`` takes rows of features, ``conv1x1_act`` channels-last maps: a 1x1
convolution of stride 1 is the same product over pixels.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import require_ext_for

ACTS = {"none": 0, "relu": 1, "swish": 2, "sigmoid": 3}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, residual, act):
    if act not in ACTS:
        raise ValueError(f"linear_act: act={act!r} is none of {sorted(ACTS)}")
    if x.dtype not in DTYPES:
        raise TypeError(f"linear_act: x is fp32, bf16 or fp16, not {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.size(-1) != weight.size(1):
        raise ValueError(f"linear_act: x [..., K] and weight [N, K], not {list(x.shape)} and {list(weight.shape)}")
    if weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError("linear_act: weight is empty")
    if bias is not None and bias.shape != (weight.size(0),):
        raise ValueError(f"linear_act: bias is [{weight.size(0)}], not {list(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.size(0)):
        raise ValueError(f"linear_act: residual is shaped like the result, not {list(residual.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"linear_act: {name} is {t.dtype}, x {x.dtype}")
        if t is not None and t.device != x.device:
            raise ValueError(f"linear_act: {name} is on {t.device}, x on {x.device}")


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, act: str = "none") -> torch.Tensor:
    """act(x @ weight.T + bias + residual).

    x is [..., K], weight [N, K], bias [N] and residual [..., N], all of one type
    (fp32, bf16 or fp16). ``act`` is "none", "relu", "swish" or "sigmoid". Sums
    are in fp32 and the result is rounded once. Gradients go to all four, once;
    for swish and sigmoid the slopes are kept for them in fp32, and for 16-bit
    types the backward products take the gradient behind the activation as a sum
    of two numbers of that type, which holds 16 (bf16) or 22 (fp16) bits of it.
    On the GPU x has fewer than 2^31 - 256 rows, K and N are 2^23 at most, and a
    result has fewer than 2^24 tiles; more is refused.
    """
    _check(x, weight, bias, residual, act)
    C = require_ext_for(x)
    if C is None:
        z = x.float() @ weight.float().t()
        if bias is not None:
            z = z + bias.float()
        if residual is not None:
            z = z + residual.float()
        z = {"none": lambda v: v, "relu": torch.relu, "swish": torch.nn.functional.silu,
             "sigmoid": torch.sigmoid}[act](z)
        return z.to(x.dtype)
    n, k = weight.shape
    if x.dim() == 2 and x.is_contiguous() and weight.is_contiguous() and (residual is None or residual.is_contiguous()):
        return C.linear_act(x, weight, bias if bias is None else bias.contiguous(), residual, ACTS[act])
    y = C.linear_act(x.reshape(x.numel() // k, k).contiguous(), weight.contiguous(),
                     None if bias is None else bias.contiguous(),
                     None if residual is None else residual.reshape(x.numel() // k, n).contiguous(), ACTS[act])
    return y.view(*x.shape[:-1], n)


def conv1x1_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, act: str = "none") -> torch.Tensor:
    """``linear_act`` over the pixels of a map: a 1x1 convolution of stride 1.

    x [B, K, H, W], weight [N, K, 1, 1] or [N, K], residual [B, N, H, W]; the
    result is channels last (maps of another order are copied into it first).
    """
    if x.dim() != 4 or (residual is not None and residual.dim() != 4):
        raise ValueError("conv1x1_act: maps are [B, C, H, W]")
    if weight.dim() == 4:
        if weight.shape[2:] != (1, 1):
            raise ValueError(f"conv1x1_act: a kernel of {tuple(weight.shape[2:])} is not 1x1")
        weight = weight.flatten(1)
    last = lambda t: None if t is None else t.permute(0, 2, 3, 1)  # noqa: E731
    return linear_act(last(x), weight, bias, last(residual), act).permute(0, 3, 1, 2)


class LinearAct(torch.nn.Linear):
    """nn.Linear on ``linear_act`` where x has the weights' type (under autocast it may not: torch's product then)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dtype != self.weight.dtype or x.dtype not in DTYPES:
            return torch.nn.functional.linear(x, self.weight, self.bias)
        return linear_act(x, self.weight, self.bias)


def fuse_pointwise(model: torch.nn.Module) -> int:
    """Put a model's linear heads and squeeze-and-excitation products on ``linear_act``. Returns how many."""
    n = 0
    for m in model.modules():
        if type(m) is torch.nn.Linear:
            m.__class__ = LinearAct
            n += 1
        elif getattr(m, "has_se", False) and hasattr(m, "fused_se"):
            m.fused_se = True
            n += 2
    return n
