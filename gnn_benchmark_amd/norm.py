"""RMS norm with the residual's addition, in one pass each way: ``h = x + residual``,
``y = relu?(h / sqrt(mean(h^2) + eps) * weight)`` -- next to ``sage.dropout_layernorm_relu``, for layers that carry a
residual stream -- and the same with ``y`` leaving in the 8-bit format that ``fp8.product`` reads.  Widths of 1 to 16384,
fp32 or bf16 rows, the weight in fp32 or the rows' type."""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ext
from .fp8 import QuantizedRows, address, as_rows, dtype_code, row_stride


def _forward(x, weight, eps, residual, relu, y=None):
    """(y, h or None)"""
    return ext.train_ops().rms_norm(x, weight, eps, residual, relu, y)


def _forward_fp8(x, weight, eps, residual, relu):
    codes, scales, h = ext.train_ops().rms_norm_fp8_forward(x, weight, eps, residual, relu)
    return QuantizedRows(codes, scales, x.size(-1)), (x if h is None else h)


def _backward(grad_y, grad_h, h, weight, eps, relu):
    """(gradient of x and of the residual, gradient of the weight in its type)."""
    shape = h.shape
    h, gy = as_rows(h), as_rows(grad_y)
    gh = None if grad_h is None else as_rows(grad_h)
    w = weight.detach().contiguous()
    rows, width = h.shape
    L = _lib.lib()
    nbytes = int(L.gnnagg_rms_norm_backward_workspace_bytes(rows, width))
    grad_x = torch.empty(shape, dtype=h.dtype, device=h.device)
    grad_w = torch.empty(width, dtype=torch.float32, device=h.device)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    with _lib.on_device(h.device):
        _lib.check(L.gnnagg_rms_norm_backward(
            address(gy), row_stride(gy), address(gh), 0 if gh is None else row_stride(gh), address(h), row_stride(h),
            address(w), dtype_code(w.dtype, "the norm's weight"), float(eps), 1 if relu else 0, address(grad_x), width,
            address(grad_w), address(workspace), nbytes, rows, width, dtype_code(h.dtype, "x"),
            _lib.raw_stream(h.device)))
    return grad_x, grad_w.to(weight.dtype)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, relu):
        y, h = _forward(x, weight, eps, residual, relu)
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps, ctx.relu = eps, relu
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_h=None):
        h, weight = ctx.saved_tensors
        if grad_y is None:  # only the residual stream was used
            grad_x, grad_w = grad_h, None
        else:
            grad_x, grad_w = _backward(grad_y, grad_h, h, weight, ctx.eps, ctx.relu)
        want = ctx.needs_input_grad
        return (grad_x if want[0] else None, grad_x if want[1] else None, grad_w if want[2] else None, None, None)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             relu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)`` of x [..., width]: ``h = x + residual`` (rounded to x's type; ``x`` itself without a residual) and
    ``y`` its RMS norm times ``weight``, through a ReLU where asked for.  Differentiable in x, the residual and the
    weight; the gradient of ``h``, where it is used further, is added inside the backward pass."""
    if not torch.is_grad_enabled():
        y, h = _forward(x, weight, eps, residual, relu)
        return y, (x if h is None else h)
    if residual is None:
        return _RmsNorm.apply(x, None, weight, float(eps), bool(relu)), x
    return _RmsNorm.apply(x, residual, weight, float(eps), bool(relu))


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
