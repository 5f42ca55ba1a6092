"""RMS norm with the residual's addition, in one pass each way: ``h = x + residual``,
``y = relu?(h / sqrt(mean(h^2) + eps) * weight)`` -- next to ``sage.dropout_layernorm_relu``, for layers that carry a
residual stream -- and the same with ``y`` leaving in the 8-bit format that ``fp8.product`` reads.  Widths of 1 to 16384,
fp32 or bf16 rows, the weight in fp32 or the rows' type."""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .fp8 import QuantizedRows, _refuse_grad, address, as_rows, check_gpu, dtype_code, row_stride


def check_norm(x, weight, residual) -> None:
    check_gpu(x, "x")
    check_gpu(weight, "the norm's weight", x.device)
    dtype_code(x.dtype, "x")
    if x.dim() < 1 or weight.dim() != 1 or weight.numel() != x.size(-1):
        raise RuntimeError("Input mismatch: the norm's weight must hold one value per column of x")
    if weight.dtype != torch.float32 and weight.dtype != x.dtype:
        raise RuntimeError("Input mismatch: the norm's weight must be float32 or of x's type")
    if residual is not None:
        check_gpu(residual, "the residual", x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise RuntimeError("Input mismatch: the residual must have x's shape and type")


def _operands(x, weight, residual):
    """What both forward forms pass: rows of x and of the residual, the weight, a fresh h (x's shape) or None."""
    rows = as_rows(x)
    res = None if residual is None else as_rows(residual)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return rows, res, weight.detach().contiguous(), h


def _forward(x, weight, eps, residual, relu, y=None):
    rows, res, w, h = _operands(x, weight, residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if y is None else y
    yr = y.view(-1, x.size(-1)) if y.dim() != 2 else y
    with _lib.on_device(x.device):
        _lib.check(_lib.lib().gnnagg_rms_norm(
            address(rows), row_stride(rows), address(res), 0 if res is None else row_stride(res), address(w),
            dtype_code(w.dtype, "the norm's weight"), float(eps), 1 if relu else 0, address(h),
            0 if h is None else x.size(-1), address(yr), row_stride(yr), rows.size(0), rows.size(1),
            dtype_code(x.dtype, "x"), _lib.raw_stream(x.device)))
    return y, h


def _forward_fp8(x, weight, eps, residual, relu):
    rows, res, w, h = _operands(x, weight, residual)
    q = QuantizedRows.empty(rows.size(0), rows.size(1), x.device)
    with _lib.on_device(x.device):
        _lib.check(_lib.lib().gnnagg_rms_norm_fp8(
            address(rows), row_stride(rows), address(res), 0 if res is None else row_stride(res), address(w),
            dtype_code(w.dtype, "the norm's weight"), float(eps), 1 if relu else 0, address(h),
            0 if h is None else x.size(-1), address(q.codes), address(q.scales), rows.size(0), rows.size(1),
            dtype_code(x.dtype, "x"), _lib.raw_stream(x.device)))
    return q, (x if h is None else h)


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
    check_norm(x, weight, residual)
    if residual is None:
        return _RmsNorm.apply(x, None, weight, float(eps), bool(relu)), x
    return _RmsNorm.apply(x, residual, weight, float(eps), bool(relu))


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                 relu: bool = False) -> Tuple[QuantizedRows, torch.Tensor]:
    """``rms_norm`` with ``y`` in the 8-bit format (``fp8.QuantizedRows``; leading dimensions become rows), quantised
    from its fp32 value.  No gradient: ``fp8.norm_linear`` is the differentiable norm in front of a product."""
    check_norm(x, weight, residual)
    _refuse_grad(x, weight, residual)
    return _forward_fp8(x, weight, eps, residual, relu)


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
