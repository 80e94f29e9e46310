"""4-bit storage for the weights of frozen layers, and products with it.

A trained classifier that no longer changes -- a teacher -- keeps the weight of its Linear head (`ResNet.fc`, or heads of
the user's own behind the encoder's features) in 4.25 bits an element instead of 16 or 32.  A layer with few
rows is bound by reading its weight, one with many by the matrix rate, and 4-bit operands help both:

    w = quantize_mx4(linear.weight)                    # once per checkpoint
    y = mx4_linear(x, w, linear.bias.detach())         # x is quantised the same way on its way in; fp32 sums
    model.fc = MX4Linear.from_linear(model.fc)         # the same as a module, in a models.resnet.ResNet

Format: 32 consecutive elements of a row share a power-of-two scale 2^(E - 127) and are rounded to
{0, .5, 1, 1.5, 2, 3, 4, 6} with a sign (to nearest, ties to the even code, saturating).  E is the exponent of the block's largest
magnitude less two; a block that holds an infinity or a NaN becomes NaN as a whole.

The projector, predictor and fuser MLPs of the pre-train model (src/models/backbone.py:12-31) are trained by the engine, which
takes nn.Linear alone there and refuses other layers with an error.

The gradient runs through to x (`dx = dy W`, the rounding of x passed straight through); the weight is frozen and has none.
All arithmetic is in csrc/mx4.hip; there is no CPU path."""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import kernels as kn


class MX4Tensor:
    """A [rows, cols] matrix in 4-bit storage: codes uint8 [G, rows, 128] and scales uint8 [G, rows, 8], G = ceil(cols / 256)
    (element 2i of a group in the low half of byte i; codes behind the last column must be zero)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        rows = kn._mx4(codes, scales, int(cols), "MX4Tensor", kn._gpu(codes, "MX4Tensor"))[0]
        self.codes, self.scales, self.shape = codes, scales, torch.Size((rows, int(cols)))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """the values the codes stand for; exact in float32 and (but for subnormals) bfloat16, in float16 where they fit"""
        y = torch.empty(self.shape, dtype=dtype, device=self.device)
        kn.mx4_dequantize(self.codes, self.scales, y)
        return y

    def __repr__(self) -> str:
        return f"MX4Tensor({tuple(self.shape)}, device={self.device})"


def _matrix(x: torch.Tensor, name: str) -> torch.Tensor:
    """[..., cols] as [rows, cols] with adjacent elements in a row, copied only where its strides need it"""
    kn._gpu(x, name)
    kn._float(x, name)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: expected [..., cols] with at least one column, got {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if not x.is_contiguous() and ((x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1])):
        x = x.contiguous()
    return x


def quantize_mx4(x: torch.Tensor) -> MX4Tensor:
    """[..., cols] float32 / bfloat16 / float16 -> MX4Tensor [rows, cols]; not differentiable"""
    x = _matrix(x.detach(), "quantize_mx4")
    G = (x.shape[1] + kn.MX4_GROUP - 1) // kn.MX4_GROUP
    codes = torch.empty(G, x.shape[0], kn.MX4_GROUP // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(G, x.shape[0], kn.MX4_GROUP // 32, dtype=torch.uint8, device=x.device)
    kn.mx4_quantize(x, codes, scales)
    return MX4Tensor(codes, scales, x.shape[1])


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, out_dtype):
        ctx.save_for_backward(weight.codes, weight.scales)
        ctx.like = (x.shape, x.dtype)
        rows = _matrix(x, "mx4_linear")
        y = torch.empty(rows.shape[0], weight.shape[0], dtype=out_dtype, device=x.device)
        kn.mx4_linear(rows, weight.codes, weight.scales, y, bias)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        shape, dtype = ctx.like
        dy = _matrix(dy, "mx4_linear backward")
        dx = torch.empty(dy.shape[0], shape[-1], dtype=dtype, device=dy.device)
        kn.mx4_dgrad(dy, codes, scales, dx)
        return dx if len(shape) == 2 else dx.view(shape), None, None, None


def mx4_linear(x: Union[torch.Tensor, MX4Tensor], weight: MX4Tensor, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = Q(x) weight^T + bias: x [..., cols] float32 / bfloat16 / float16 (quantised here) or an MX4Tensor [rows, cols];
    weight MX4Tensor [out, cols]; bias float32 [out], frozen like the weight.  y [..., out] in out_dtype (default: x's type,
    float32 for an MX4Tensor), summed in float32.  Differentiable in x when it is a tensor."""
    if not isinstance(weight, MX4Tensor):
        raise TypeError("mx4_linear: weight must be an MX4Tensor (quantize_mx4)")
    if x.shape[-1:] != weight.shape[-1:]:
        raise ValueError(f"mx4_linear: x has shape {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if weight.shape[0] == 0:
        raise ValueError("mx4_linear: weight has no rows")
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("mx4_linear: the layer is frozen; pass bias.detach()")
    if isinstance(x, MX4Tensor):
        y = torch.empty(x.shape[0], weight.shape[0], dtype=out_dtype or torch.float32, device=x.device)
        return kn.mx4_gemm(x.codes, x.scales, weight.codes, weight.scales, x.shape[1], y, bias)
    kn._gpu(x, "mx4_linear")
    return _LinearFn.apply(x, weight, bias, out_dtype or x.dtype)


class MX4Linear(torch.nn.Module):
    """nn.Linear with a frozen 4-bit weight; state: codes, scales, bias as buffers"""

    def __init__(self, weight: MX4Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear) -> "MX4Linear":
        b = None if linear.bias is None else linear.bias.detach().float().clone()
        return cls(quantize_mx4(linear.weight), b)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        bias = None if self.bias is None else self.bias.float()  # a module cast to 16 bits takes its buffers along
        return mx4_linear(x, MX4Tensor(self.codes, self.scales, self.in_features), bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
