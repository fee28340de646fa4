"""Small fused building blocks shared by the model zoo.

``bn_relu(x, bn)`` is the pre-activation hot path of WideResNet/PyramidNet:
on GPU it dispatches to the fused NHWC BatchNorm+ReLU HIP kernel
(fwd + bwd as one custom Function); on CPU it composes torch ops. The BN
module keeps standard nn.BatchNorm2d parameters/buffers so state_dicts stay
checkpoint-compatible with the reference layout.

A GroupNorm in the place of the BatchNorm (models built with ``norm: group``)
goes to the fused group norm instead, on either device.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import has_ext
from .groupnorm import DTYPES, group_norm_act


import os


def _group_norm(x: torch.Tensor, gn: torch.nn.GroupNorm, act: str) -> torch.Tensor:
    if x.dtype not in DTYPES:       # fp64, where gradients are checked
        z = F.group_norm(x, gn.num_groups, gn.weight, gn.bias, gn.eps)
        return F.relu(z) if act == "relu" else F.silu(z) if act == "swish" else z
    return group_norm_act(x, gn.num_groups, gn.weight, gn.bias, gn.eps, act)


def bn_relu(x: torch.Tensor, bn: torch.nn.BatchNorm2d) -> torch.Tensor:
    """BatchNorm2d followed by ReLU, fused on GPU."""
    if isinstance(bn, torch.nn.GroupNorm):
        return _group_norm(x, bn, "relu")
    if (x.is_cuda and has_ext()
            and os.environ.get("FAA_NO_FUSED_BN") != "1"):
        from .bnrelu import fused_bn_relu
        return fused_bn_relu(x, bn)
    return F.relu(bn(x))


def bn_only(x: torch.Tensor, bn: torch.nn.BatchNorm2d) -> torch.Tensor:
    """BatchNorm2d without activation, fused on GPU."""
    if isinstance(bn, torch.nn.GroupNorm):
        return _group_norm(x, bn, "none")
    if (x.is_cuda and has_ext()
            and os.environ.get("FAA_NO_FUSED_BN") != "1"):
        from .bnrelu import fused_bn
        return fused_bn(x, bn)
    return bn(x)


def bn_swish(x: torch.Tensor, bn: torch.nn.BatchNorm2d) -> torch.Tensor:
    """BatchNorm2d followed by swish, fused on GPU (EfficientNet)."""
    if isinstance(bn, torch.nn.GroupNorm):
        return _group_norm(x, bn, "swish")
    if (x.is_cuda and has_ext()
            and os.environ.get("FAA_NO_FUSED_BN") != "1"):
        from .bnrelu import fused_bn_swish
        return fused_bn_swish(x, bn)
    from .functional import swish
    return swish(bn(x))


def res_add(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Residual join; on GPU it also pre-computes the next BN's fwd-reduce
    partials in the same pass (consumed by the following bn_relu call)."""
    if (a.is_cuda and has_ext()
            and os.environ.get("FAA_NO_FUSED_BN") != "1"):
        from .bnrelu import residual_add
        return residual_add(a, b)
    return a + b
