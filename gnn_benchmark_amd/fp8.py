"""Dense products in 8-bit floating point with one scale per block of 128, and the layer around them.

The format (``include/gnn_train.h``): e4m3 codes in blocks of 128 values, a block's scale a power of two in one byte
(``float8_e8m0fnu``), the smallest for which the block's largest finite magnitude stays at or below 448.  Rows
(activations, gradients) have blocks of 1 x 128 along them, weights of 128 x 128.  An infinity or NaN becomes the NaN code
and leaves its block's scale alone, so it spoils its own row's results and no other.

``linear`` is the differentiable layer: the product and the input gradient multiply codes on the matrix units' 8-bit path,
the weight gradient takes the saved codes (one byte a value is all the backward pass needs of the input) against the
gradient rounded to bf16.  ``norm_linear`` puts the RMS norm in front, whose output then exists in 8 bits only.

What a product rounds.  To fp32: products are exact, sums fp32 (codes are decoded to bf16, exactly where the scale lies in
[2^-124, 2^119]; smaller scales leave bf16's subnormals to the smallest codes, and 2^128, what fp32 values from 1.9375 * 2^127
on round to, is infinite).  To bf16: the codes go through the matrix unit's 8-bit instruction, which accumulates in fp32 but
cuts each of the products of eight neighbouring codes to a multiple of 2^-13 of the largest one's power of two.  On random
operands that is 1.5e-5 of the result, far below what storing bf16 rounds away; where large products cancel it is what remains
of them, and a program that needs those sums takes the fp32 result.
"""
from typing import Optional, Tuple

import torch

from . import ext

BLOCK = 128


def padded(width: int) -> int:
    return -(-width // BLOCK) * BLOCK


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


def quantize_weight(w: torch.Tensor, for_gradient: bool = False) -> QuantizedWeight:
    """fp32 or bf16 [k, n] -> the 8-bit format; a transposed view (``torch.nn.Linear``'s ``weight.t()``) is read where it
    lies.  ``for_gradient``: also the codes by input.  No gradient."""
    codes, by_input, scales = ext.train_ops().quantize_weight(w, for_gradient)
    return QuantizedWeight(w.size(0), w.size(1), codes, scales, by_input)


def product(x: QuantizedRows, weight: QuantizedWeight, bias: Optional[torch.Tensor] = None,
            out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
            input_gradient: bool = False) -> torch.Tensor:
    """``x @ weight (+ bias)`` of 8-bit operands, [rows, n] in ``out_dtype``: float32, products exact and sums in
    fp32; or bfloat16, through the 8-bit instruction, whose cut of neighbouring products is described above.
    ``input_gradient``: ``x @ weight^T``, [rows, k], from the codes by input.  ``out``: an array of that shape with
    contiguous rows (a column block of a wider one is fine) to write into, apart from the operands' memory.  No gradient
    (``linear`` has one)."""
    return ext.train_ops().product(x.codes, x.scales, x.cols, weight.codes_by_input if input_gradient else weight.codes,
                                   weight.scales, weight.k, weight.n, bias, out_dtype, out, input_gradient)


def weight_gradient(x: QuantizedRows, g: torch.Tensor, with_bias: bool = False):
    """``x^T @ bf16(g)``, fp32 [x.cols, n]; with ``with_bias`` the pair of it and ``g``'s column sums (fp32).
    No gradient."""
    grad_w, grad_b = ext.train_ops().weight_gradient(x.codes, x.scales, x.cols, g, with_bias)
    return (grad_w, grad_b) if with_bias else grad_w


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w (+ bias)`` with both operands in the 8-bit format, x [..., k], w [k, n] (``lin.weight.t()`` of a
    ``torch.nn.Linear`` is read where it lies), result in x's type (rounded as ``product``'s of that type).
    The gradients are those of the product of the
    quantised operands with the quantisation passed through: ``grad x = q(g) q(w)^T``, ``grad w = q(x)^T bf16(g)``."""
    return ext.train_ops().linear(x, w, bias)


def norm_linear(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, w: torch.Tensor,
                bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                relu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``linear(norm.rms_norm(x + residual), w, bias)`` with the normalised rows written in 8 bits by the norm itself:
    (result, h) with ``h = x + residual`` the residual stream (``x`` itself without a residual)."""
    return ext.train_ops().norm_linear(x, norm_weight, eps, w, bias, residual, relu)
