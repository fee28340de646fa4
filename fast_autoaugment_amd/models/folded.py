"""Frozen networks with their BatchNorm folded into the 1x1 convolutions.

The policy search scores hundreds of augmentation policies on child networks
that do not change any more (search/density_match.py). In evaluation a
BatchNorm is a scale and a shift a channel, so a 1x1 convolution with the
BatchNorm behind it (before it too, where nothing lies between), the skip
connection and the activation are one matrix product with an epilogue
(ops/pointwise.py). ``fold_for_inference`` rebuilds the bottleneck blocks of
ResNet and PyramidNet and the MBConv blocks of EfficientNet that way.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from ..ops.modules import bn_relu, bn_swish
from ..ops.pointwise import conv1x1_act, linear_act
from . import efficientnet, pyramidnet, resnet


def _affine(bn: nn.BatchNorm2d):
    """Scale and shift of a BatchNorm in evaluation, in 64 bits."""
    scale = bn.weight.double() / torch.sqrt(bn.running_var.double() + bn.eps)
    return scale, bn.bias.double() - bn.running_mean.double() * scale


class Pointwise(nn.Module):
    """A 1x1 convolution with the affine maps around it: out * (conv(inp(x))), in ``dtype``."""

    def __init__(self, conv: nn.Conv2d, dtype, inp=None, out=None, factor: float = 1.0):
        super().__init__()
        weight = conv.weight.detach().double().flatten(1)
        bias = conv.bias.detach().double() if conv.bias is not None else torch.zeros_like(weight[:, 0])
        if inp is not None:
            scale, shift = _affine(inp)
            bias = bias + weight @ shift
            weight = weight * scale
        if out is not None:
            scale, shift = _affine(out)
            weight, bias = weight * scale[:, None], bias * scale + shift
        self.stride = conv.stride[0]
        self.register_buffer("weight", (weight * factor).to(dtype).contiguous())
        self.register_buffer("bias", (bias * factor).to(dtype).contiguous())

    def forward(self, x, residual=None, act: str = "none"):
        if self.stride != 1:
            x = x[:, :, ::self.stride, ::self.stride]
        return conv1x1_act(x.to(self.weight.dtype), self.weight, self.bias,
                           None if residual is None else residual.to(self.weight.dtype), act)


class FoldedBottleneck(nn.Module):
    """resnet.Bottleneck: 1x1 -> 3x3 -> 1x1, skip and relu."""

    def __init__(self, block: resnet.Bottleneck, dtype):
        super().__init__()
        self.first = Pointwise(block.conv1, dtype, out=block.bn1)
        self.conv2, self.bn2 = block.conv2, block.bn2
        self.last = Pointwise(block.conv3, dtype, out=block.bn3)
        self.skip = None if block.downsample is None else Pointwise(block.downsample[0], dtype, out=block.downsample[1])

    def forward(self, x):
        out = bn_relu(self.conv2(self.first(x, act="relu")), self.bn2)
        return self.last(out, residual=x if self.skip is None else self.skip(x), act="relu")


class FoldedPyramidBottleneck(nn.Module):
    """pyramidnet.Bottleneck: BN -> 1x1 -> 3x3 -> 1x1 -> BN, ShakeDrop's expectation, zero-padded skip."""

    def __init__(self, block: pyramidnet.Bottleneck, dtype):
        super().__init__()
        self.first = Pointwise(block.conv1, dtype, inp=block.bn1, out=block.bn2)
        self.conv2, self.bn3 = block.conv2, block.bn3
        self.last = Pointwise(block.conv3, dtype, out=block.bn4, factor=1.0 - block.shake_drop.p_drop)
        self.downsample = block.downsample

    def forward(self, x):
        out = bn_relu(self.conv2(self.first(x, act="relu")), self.bn3)
        skip = self.downsample(x) if self.downsample is not None else x
        if skip.size(1) == self.last.weight.size(0):
            return self.last(out, residual=skip)
        out = self.last(out)
        return pyramidnet._pad_add(out, skip.to(out.dtype))


class FoldedMBConv(nn.Module):
    """efficientnet.MBConvBlock without experts: expand -> depthwise -> squeeze and excite -> project, skip."""

    def __init__(self, block: efficientnet.MBConvBlock, dtype, drop_connect_rate: float):
        super().__init__()
        args = block._block_args
        self.expand = Pointwise(block._expand_conv, dtype, out=block._bn0) if args.expand_ratio != 1 else None
        self.depthwise, self.bn1 = block._depthwise_conv, block._bn1
        self.reduce = Pointwise(block._se_reduce, dtype) if block.has_se else None
        self.excite = Pointwise(block._se_expand, dtype) if block.has_se else None
        self.skips = args.id_skip and args.stride == 1 and args.input_filters == args.output_filters
        # evaluation scales the branch by its chance to be there
        self.project = Pointwise(block._project_conv, dtype, out=block._bn2,
                                 factor=1.0 - drop_connect_rate if self.skips else 1.0)

    def forward(self, inputs, drop_connect_rate=None):
        x = inputs if self.expand is None else self.expand(inputs, act="swish")
        x = bn_swish(self.depthwise(x), self.bn1)
        if self.reduce is not None:
            gate = F.adaptive_avg_pool2d(x, 1).flatten(1).to(self.reduce.weight.dtype)
            gate = linear_act(gate, self.reduce.weight, self.reduce.bias, act="swish")
            gate = linear_act(gate, self.excite.weight, self.excite.bias, act="sigmoid")
            x = gate[:, :, None, None] * x
        return self.project(x, residual=inputs if self.skips else None)


def fold_for_inference(model: nn.Module, dtype: torch.dtype = torch.float32) -> int:
    """Fold a frozen model's blocks in place; ``dtype`` is what they compute in. Returns how many were folded.

    The model has to be in evaluation, and stays there: a folded block has no statistics to go back to.
    """
    if model.training:
        raise ValueError("fold_for_inference: the model is in training")

    def has_batch_norms(m):
        norms = [b for b in m.modules() if isinstance(b, (nn.modules.batchnorm._BatchNorm, nn.GroupNorm))]
        return bool(norms) and all(type(b) is nn.BatchNorm2d for b in norms)

    def folded(m, rate):
        if type(m) is resnet.Bottleneck and has_batch_norms(m):
            return FoldedBottleneck(m, dtype)
        if type(m) is pyramidnet.Bottleneck and has_batch_norms(m):
            return FoldedPyramidBottleneck(m, dtype)
        if type(m) is efficientnet.MBConvBlock and has_batch_norms(m) and not m._is_condconv():
            return FoldedMBConv(m, dtype, rate)
        return None

    count = 0

    def walk(parent):
        nonlocal count
        for name, child in list(parent.named_children()):
            rate = 0.0
            if isinstance(model, efficientnet.EfficientNet) and parent is model._blocks:
                rate = (model._global_params.drop_connect_rate or 0.0) * int(name) / len(model._blocks)
            new = folded(child, rate)
            if new is None:
                walk(child)
            else:
                new.eval()
                parent._modules[name] = new
                count += 1

    with torch.no_grad():
        walk(model)
    return count
