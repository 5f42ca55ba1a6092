"""The 8-bit format of include/gnn_train.h and the training operators' formulas in 64 bits, on the CPU, written from the
definitions (not collected by pytest)."""
import torch

BLOCK = 128
HALF32, HALF16 = 2.0 ** -24, 2.0 ** -8  # half a step of fp32 / bf16, relative
STEP8 = 2.0 ** -4                       # half a step of e4m3, relative


def padded(n):
    return -(-n // BLOCK) * BLOCK


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def block_exponent(top):
    """Smallest e in [-126, 120] with top * 2^-e <= 448, for fp64 tops >= 0."""
    e = torch.full_like(top, -126.0)
    for _ in range(2):  # the estimate, then one step for its rounding
        guess = torch.where(top > 0, torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448.0)), -126.0)
        e = torch.where(top * torch.exp2(-guess) > 448.0, guess + 1, guess)
        e = torch.where(top * torch.exp2(1 - e) <= 448.0, e - 1, e)
    return e.clamp(-126, 120)


def e4m3_nearest(y):
    """Nearest e4m3 value, ties to even, of fp64 |y| <= 448 (NaN stays)."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().nan_to_num().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def quantize_blocks(x):
    """fp64 [..., 128] blocks -> (code values, exponents)."""
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
    e = block_exponent(finite.amax(-1, keepdim=True))
    y = torch.where(torch.isfinite(x), x, torch.nan) * torch.exp2(-e)
    return e4m3_nearest(y), e


def quantize_rows(x):
    """fp64 [M, K] -> (code values [M, padded], exponents [M, blocks], dequantised [M, K])."""
    rows, width = x.shape
    full = torch.zeros(rows, padded(width), dtype=torch.float64)
    full[:, :width] = x
    codes, e = quantize_blocks(full.view(rows, -1, BLOCK))
    values = (codes * torch.exp2(e)).view(rows, -1)[:, :width]
    return codes.view(rows, -1), e.squeeze(-1), values


def quantize_weight(w):
    """fp64 [K, N] -> (code values [K, N], exponents [K blocks, N blocks], dequantised [K, N])."""
    k, n = w.shape
    kb, nb = padded(k) // BLOCK, padded(n) // BLOCK
    full = torch.zeros(kb * BLOCK, nb * BLOCK, dtype=torch.float64)
    full[:k, :n] = w
    grid = full.view(kb, BLOCK, nb, BLOCK)
    finite = torch.where(torch.isfinite(grid), grid.abs(), 0.0)
    e = block_exponent(finite.amax((1, 3), keepdim=True))
    codes = e4m3_nearest(torch.where(torch.isfinite(grid), grid, torch.nan) * torch.exp2(-e))
    values = (codes * torch.exp2(e)).view(kb * BLOCK, nb * BLOCK)[:k, :n]
    return codes.view(kb * BLOCK, nb * BLOCK)[:k, :n], e.view(kb, nb), values


def rms_norm(h, w, eps, relu):
    """(y, h / rms, 1 / rms) of fp64 rows."""
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    z = h * r
    y = z * w
    return (torch.where(y < 0, 0.0, y) if relu else y), z, r


def same(got, want):
    """Equal values, NaN in the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    return got.shape == want.shape and bool(((got == want) | (got.isnan() & want.isnan())).all())


def assert_within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    excess = (got - want).abs() - bound
    at = int(excess.argmax())
    assert float(excess.max()) <= 0.0, (f"{what}: off by {float((got - want).abs().flatten()[at]):.3e}, allowed "
                                        f"{float((bound + 0 * want).flatten()[at]):.3e}, at {at} of {tuple(want.shape)}")
