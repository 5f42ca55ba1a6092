"""RMS norm with the residual's addition, in one pass each way: ``h = x + residual``,
``y = relu?(h / sqrt(mean(h^2) + eps) * weight)`` -- next to ``sage.dropout_layernorm_relu``, for layers that carry a
residual stream -- and the same with ``y`` leaving in the 8-bit format that ``fp8.product`` reads.  Widths of 1 to 16384,
fp32 or bf16 rows, the weight in fp32 or the rows' type.  In a row with an infinity ``1 / sqrt(mean(h^2) + eps)`` is zero: its
finite values give zero, its infinite ones NaN; a NaN makes its whole row NaN, and either spoils no other row."""
from typing import Optional, Tuple

import torch

from . import ext
from .fp8 import QuantizedRows


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             relu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)`` of x [..., width]: ``h = x + residual`` (rounded to x's type; ``x`` itself without a residual) and
    ``y`` its RMS norm times ``weight``, through a ReLU where asked for.  Differentiable in x, the residual and the
    weight; the gradient of ``h``, where it is used further, is added inside the backward pass."""
    return ext.train_ops().rms_norm(x, weight, eps, residual, relu)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                 relu: bool = False) -> Tuple[QuantizedRows, torch.Tensor]:
    """``rms_norm`` with ``y`` in the 8-bit format (``fp8.QuantizedRows``; leading dimensions become rows), quantised
    from its fp32 value.  No gradient: ``fp8.norm_linear`` is the differentiable norm in front of a product."""
    codes, scales, h = ext.train_ops().rms_norm_fp8(x, weight, eps, residual, relu)
    return QuantizedRows(codes, scales, x.size(-1)), (x if h is None else h)


class RmsNorm(torch.nn.Module):
    """``rms_norm`` with its weight as a parameter: ``(y, h)`` of x and the residual stream so far."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(width))

    def reset_parameters(self):
        with torch.no_grad():
            self.weight.fill_(1.0)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                relu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
        return rms_norm(x, self.weight, self.eps, residual, relu)
