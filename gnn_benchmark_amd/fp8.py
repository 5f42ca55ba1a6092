"""Dense products in 8-bit floating point with one scale per block of 128, and the layer around them.

The format (``include/gnn_train.h``): e4m3 codes in blocks of 128 values, a block's scale a power of two in one byte
(``float8_e8m0fnu``), the smallest for which the block's largest finite magnitude stays at or below 448.  Rows
(activations, gradients) have blocks of 1 x 128 along them, weights of 128 x 128.  An infinity or NaN becomes the NaN code
and leaves its block's scale alone, so it spoils its own row's results and no other.

``linear`` is the differentiable layer: the product and the input gradient multiply codes on the matrix units' 8-bit path,
the weight gradient takes the saved codes (one byte a value is all the backward pass needs of the input) against the
gradient rounded to bf16.  ``norm_linear`` puts the RMS norm in front, whose output then exists in 8 bits only.
"""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ext

BLOCK = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def padded(width: int) -> int:
    return -(-width // BLOCK) * BLOCK


def dtype_code(dtype: torch.dtype, what: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"Input mismatch: {what} must be float32 or bfloat16, not {dtype}")
    return code


def check_gpu(t: torch.Tensor, what: str, device=None) -> None:
    if t.is_cuda and (device is None or t.device == device):
        return
    if not t.is_cuda:
        raise RuntimeError(f"Input mismatch: {what} must be a GPU (HIP) tensor")
    raise RuntimeError(f"Input mismatch: {what} is on {t.device}, the other operands on {device}")


def address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def as_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, width] with contiguous rows and a row stride of at least the width (a copy where it has none)."""
    t = t if t.dim() == 2 else t.reshape(-1, t.size(-1))
    if t.numel() == 0 or (t.stride(1) == 1 or t.size(1) == 1) and (t.stride(0) >= t.size(1) or t.size(0) == 1):
        return t
    return t.contiguous()


def row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 and t.size(1) > 0 else max(t.size(1), 1)


class QuantizedRows:
    """Rows in the 8-bit format: ``codes`` float8_e4m3fn [rows, cols rounded up to 128] (the padding zero), ``scales``
    float8_e8m0fnu [rows, blocks], ``cols`` the width they stand for."""
    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        self.codes, self.scales, self.cols = codes, scales, int(cols)

    @staticmethod
    def empty(rows: int, cols: int, device) -> "QuantizedRows":
        wide = padded(cols)
        return QuantizedRows(torch.empty(rows, wide, dtype=torch.float8_e4m3fn, device=device),
                             torch.empty(rows, wide // BLOCK, dtype=torch.float8_e8m0fnu, device=device), cols)

    def dequantize(self) -> torch.Tensor:
        """The fp32 values [rows, cols] the codes stand for (for looking at them)."""
        values = self.codes.float().view(self.codes.size(0), -1, BLOCK) * self.scales.float().unsqueeze(2)
        return values.view(self.codes.size(0), -1)[:, :self.cols]

    def check(self, what: str) -> None:
        codes, scales = self.codes, self.scales
        check_gpu(codes, what)
        check_gpu(scales, what + "' scales", codes.device)
        if (codes.dtype != torch.float8_e4m3fn or codes.dim() != 2 or self.cols < 1 or codes.size(1) != padded(self.cols)
                or not codes.is_contiguous() or codes.data_ptr() % 16 != 0):
            raise RuntimeError(f"Input mismatch: {what} must hold contiguous, 16-byte aligned float8_e4m3fn codes "
                               "[rows, cols rounded up to 128]")
        if (scales.dtype != torch.float8_e8m0fnu or tuple(scales.shape) != (codes.size(0), codes.size(1) // BLOCK)
                or not scales.is_contiguous()):
            raise RuntimeError(f"Input mismatch: {what} must hold contiguous float8_e8m0fnu scales [rows, blocks of 128]")


class QuantizedWeight:
    """A weight [k, n] in the 8-bit format: ``codes`` float8_e4m3fn [n, k rounded up to 128] for the product,
    ``codes_by_input`` [k, n rounded up to 128] for the input gradient (None where that is not wanted), ``scales``
    float8_e8m0fnu [k blocks, n blocks] (any strides) of its 128 x 128 blocks."""
    __slots__ = ("k", "n", "codes", "scales", "codes_by_input")

    def __init__(self, k: int, n: int, codes: Optional[torch.Tensor], scales: torch.Tensor,
                 codes_by_input: Optional[torch.Tensor] = None):
        self.k, self.n, self.codes, self.scales, self.codes_by_input = int(k), int(n), codes, scales, codes_by_input


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """fp32 or bf16 [rows, width] -> the 8-bit format.  No gradient (``linear`` has one)."""
    return QuantizedRows(*ext.train_ops().quantize_rows(x), x.size(1))


def _quantize_rows(x: torch.Tensor) -> QuantizedRows:
    return QuantizedRows(*ext.train_ops().quantize_rows_forward(x), x.size(1))


def quantize_weight(w: torch.Tensor, for_gradient: bool = False) -> QuantizedWeight:
    """fp32 or bf16 [k, n] -> the 8-bit format; a transposed view (``torch.nn.Linear``'s ``weight.t()``) is read where it
    lies.  ``for_gradient``: also the codes by input.  No gradient."""
    _refuse_grad(w)
    return _quantize_weight(w, True, for_gradient)


def _quantize_weight(w: torch.Tensor, by_output: bool, by_input: bool) -> QuantizedWeight:
    check_gpu(w, "the weight")
    code = dtype_code(w.dtype, "the weight")
    if w.dim() != 2 or w.numel() == 0:
        raise RuntimeError("Input mismatch: the weight must be [k, n], neither zero")
    k, n = w.shape
    if w.stride(1) != 1 and w.stride(0) == 1 and w.stride(1) >= k:  # stored by output: its transpose with the roles exchanged
        t = _quantize_weight(w.t(), by_input, by_output)
        return QuantizedWeight(k, n, t.codes_by_input, t.scales.t(), t.codes)
    w = as_rows(w)
    dev = w.device
    codes = torch.empty(n, padded(k), dtype=torch.float8_e4m3fn, device=dev) if by_output else None
    codes_by_input = torch.empty(k, padded(n), dtype=torch.float8_e4m3fn, device=dev) if by_input else None
    scales = torch.empty(padded(k) // BLOCK, padded(n) // BLOCK, dtype=torch.float8_e8m0fnu, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().gnnagg_fp8_quantize_weight(address(w), row_stride(w), address(codes), address(codes_by_input),
                                                         address(scales), k, n, code, _lib.raw_stream(dev)))
    return QuantizedWeight(k, n, codes, scales, codes_by_input)


def _refuse_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("this operator has no gradient: use fp8.linear or fp8.norm_linear, or torch.no_grad()")


def product(x: QuantizedRows, weight: QuantizedWeight, bias: Optional[torch.Tensor] = None,
            out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
            input_gradient: bool = False) -> torch.Tensor:
    """``x @ weight (+ bias)`` of 8-bit operands, [rows, n] in ``out_dtype`` (fp32 accumulation, one rounding).
    ``input_gradient``: ``x @ weight^T``, [rows, k], from the codes by input.  ``out``: an array of that shape with
    contiguous rows (a column block of a wider one is fine) to write into.  No gradient (``linear`` has one)."""
    return ext.train_ops().product(x.codes, x.scales, x.cols, weight.codes_by_input if input_gradient else weight.codes,
                                   weight.scales, weight.k, weight.n, bias, out_dtype, out, input_gradient)


def _product(x, weight, bias, out_dtype, input_gradient=False):
    return ext.train_ops().product_forward(
        x.codes, x.scales, x.cols, weight.codes_by_input if input_gradient else weight.codes, weight.scales, weight.k,
        weight.n, bias, out_dtype, None, input_gradient)


def weight_gradient(x: QuantizedRows, g: torch.Tensor, with_bias: bool = False):
    """``x^T @ bf16(g)``, fp32 [x.cols, n]; with ``with_bias`` the pair of it and ``g``'s column sums (fp32)."""
    grad_w, grad_b, _ = _weight_gradient(x, g, with_bias, False)
    return (grad_w, grad_b) if with_bias else grad_w


def _weight_gradient(x: QuantizedRows, g: torch.Tensor, with_bias: bool, with_rows: bool):
    """(weight gradient, column sums or None, g in the 8-bit format or None)"""
    x.check("x")
    check_gpu(g, "g", x.codes.device)
    code = dtype_code(g.dtype, "g")
    if g.dim() != 2 or g.size(0) != x.codes.size(0) or g.size(1) == 0:
        raise RuntimeError("Input mismatch: g must be [rows of x, outputs]")
    g = as_rows(g)
    rows, k, n, device = g.size(0), x.cols, g.size(1), g.device
    L = _lib.lib()
    nbytes = int(L.gnnagg_fp8_weight_gradient_workspace_bytes(rows, k, n))
    grad_w = torch.empty(k, n, dtype=torch.float32, device=device)
    grad_b = torch.empty(n, dtype=torch.float32, device=device) if with_bias else None
    g_rows = QuantizedRows.empty(rows, n, device) if with_rows else None
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    with _lib.on_device(device):
        _lib.check(L.gnnagg_fp8_weight_gradient_and_rows(
            address(x.codes), address(x.scales), address(g), row_stride(g), code, address(grad_w), address(grad_b),
            address(g_rows.codes) if with_rows else None, address(g_rows.scales) if with_rows else None,
            address(workspace), nbytes, rows, k, n, _lib.raw_stream(device)))
    return grad_w, grad_b, g_rows


def _product_gradients(rows: QuantizedRows, weight: QuantizedWeight, g: torch.Tensor, want_x: bool, want_w: bool,
                       want_b: bool, x_dtype, w_dtype, b_dtype):
    """(grad of the rows, of the weight, of the bias) of ``rows @ weight + bias``, each None where it is not wanted."""
    grad_x = grad_w = grad_b = g_rows = None
    g = as_rows(g)
    if want_w or want_b:  # (the bias's sums come with the weight gradient's pass, beside a frozen weight too)
        grad_w, grad_b, g_rows = _weight_gradient(rows, g, want_b, want_x)
        grad_w = grad_w.to(w_dtype) if want_w else None
        grad_b = grad_b.to(b_dtype) if want_b else None
    if want_x:
        grad_x = _product(g_rows or _quantize_rows(g), weight, None, x_dtype, input_gradient=True)
    return grad_x, grad_w, grad_b


def _check_linear(x, w, bias):
    check_gpu(x, "x")
    check_gpu(w, "the weight", x.device)
    dtype_code(x.dtype, "x")
    dtype_code(w.dtype, "the weight")
    if x.dim() < 1 or w.dim() != 2 or x.size(-1) != w.size(0) or w.numel() == 0:
        raise RuntimeError(f"Input mismatch: x {tuple(x.shape)} against a weight {tuple(w.shape)}")
    if bias is not None:
        check_gpu(bias, "the bias", x.device)
        dtype_code(bias.dtype, "the bias")
        if bias.dim() != 1 or bias.numel() != w.size(1):
            raise RuntimeError("Input mismatch: the bias must hold one value per output")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        flat = as_rows(x)
        rows = _quantize_rows(flat)
        weight = _quantize_weight(w, True, ctx.needs_input_grad[0])
        out = _product(rows, weight, bias, x.dtype)
        ctx.save_for_backward(rows.codes, rows.scales, weight.codes_by_input, weight.scales)
        ctx.shapes = x.shape, tuple(w.shape)
        ctx.dtypes = x.dtype, w.dtype, None if bias is None else bias.dtype
        return out.view(x.shape[:-1] + (w.size(1),))

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        codes, scales, by_input, w_scales = ctx.saved_tensors
        x_shape, (k, n) = ctx.shapes
        want_x, want_w, want_b = ctx.needs_input_grad
        grad_x, grad_w, grad_b = _product_gradients(
            QuantizedRows(codes, scales, k), QuantizedWeight(k, n, None, w_scales, by_input), g, want_x, want_w, want_b,
            *ctx.dtypes)
        return None if grad_x is None else grad_x.view(x_shape), grad_w, grad_b


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w (+ bias)`` with both operands in the 8-bit format, x [..., k], w [k, n] (``lin.weight.t()`` of a
    ``torch.nn.Linear`` is read where it lies), result in x's type.  The gradients are those of the product of the
    quantised operands with the quantisation passed through: ``grad x = q(g) q(w)^T``, ``grad w = q(x)^T bf16(g)``."""
    _check_linear(x, w, bias)
    return _Linear.apply(x, w, bias)


class _NormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, norm_weight, eps, relu, w, bias):
        from . import norm

        rows, h = norm._forward_fp8(x, norm_weight, eps, residual, relu)
        need = any(ctx.needs_input_grad[i] for i in (0, 1, 2))
        weight = _quantize_weight(w, True, need)
        out = _product(rows, weight, bias, x.dtype)
        ctx.save_for_backward(h, norm_weight, rows.codes, rows.scales, weight.codes_by_input, weight.scales)
        ctx.norm = eps, relu
        ctx.has_residual = residual is not None
        ctx.shapes = x.shape, tuple(w.shape)
        ctx.dtypes = x.dtype, w.dtype, None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        out = out.view(x.shape[:-1] + (w.size(1),))
        return (out, h) if residual is not None else out

    @staticmethod
    @once_differentiable
    def backward(ctx, g, grad_h=None):
        from . import norm

        h, norm_weight, codes, scales, by_input, w_scales = ctx.saved_tensors
        eps, relu = ctx.norm
        x_shape, (k, n) = ctx.shapes
        want_rows = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        grad_rows = grad_x = grad_norm = grad_w = grad_b = None
        if g is not None:
            grad_rows, grad_w, grad_b = _product_gradients(
                QuantizedRows(codes, scales, k), QuantizedWeight(k, n, None, w_scales, by_input), g, want_rows,
                ctx.needs_input_grad[5], ctx.needs_input_grad[6], *ctx.dtypes)
        if want_rows and grad_rows is not None:
            grad_x, grad_norm = norm._backward(grad_rows, grad_h, h, norm_weight, eps, relu)
        elif grad_h is not None:
            grad_x = grad_h
        grad_x = None if grad_x is None else grad_x.view(x_shape)
        return (grad_x if ctx.needs_input_grad[0] else None, grad_x if ctx.needs_input_grad[1] else None,
                grad_norm if ctx.needs_input_grad[2] else None, None, None, grad_w, grad_b)


def norm_linear(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, w: torch.Tensor,
                bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                relu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``linear(norm.rms_norm(x + residual), w, bias)`` with the normalised rows written in 8 bits by the norm itself:
    (result, h) with ``h = x + residual`` the residual stream (``x`` itself without a residual)."""
    _check_linear(x, w, bias)
    if residual is None:
        return _NormLinear.apply(x, None, norm_weight, float(eps), bool(relu), w, bias), x
    return _NormLinear.apply(x, residual, norm_weight, float(eps), bool(relu), w, bias)
