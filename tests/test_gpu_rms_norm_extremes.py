"""RMS norm of rows with infinities: 1 / rms is zero there, so by the formula the finite values give zero and the infinite
ones NaN (infinity times zero).  And the gradient of rows near the lower end of fp32's range."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import norm

pytestmark = pytest.mark.gpu
EPS = 1e-6
WIDTHS = [1, 7, 47, 64, 256, 300, 1000, 2048, 5120, 6148, 16384]  # every kernel shape, aligned and not


def rows_of(width, dtype):
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(6, width, generator=gen).to(dtype)
    x[1, width // 2] = float("inf")
    x[3, 0] = -float("inf")
    x[3, width - 1] = float("inf")
    x[4, width // 3] = float("nan")
    w = (torch.rand(width, generator=gen) + 0.5).to(dtype)
    return x, w


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
def test_a_row_with_an_infinity(dtype, relu):
    for width in WIDTHS:
        x, w = rows_of(width, dtype)
        xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        y, _ = norm.rms_norm(xg, wg, EPS, relu=relu)
        want, z, r = o.rms_norm(x.double(), w.double(), EPS, relu)
        got = y.detach().double().cpu()
        assert torch.equal(got.isnan(), want.isnan()), width
        for i in (1, 3):                                    # zero beside the infinity, NaN in its place
            finite = x[i].isfinite()
            assert bool((got[i][finite] == 0).all()) and bool(got[i][~finite].isnan().all()), width
        assert bool(got[4].isnan().all())
        q, _ = norm.rms_norm_fp8(x.cuda(), w.cuda(), EPS, relu=relu)
        codes = q.codes.double().cpu()[:, :width]
        assert torch.equal(codes.isnan(), want.isnan()), width
        assert bool((codes[1][x[1].isfinite()] == 0).all()) and bool(torch.isfinite(q.scales.float()).all())
        # the weight's gradient: a spoiled row reaches the columns of its NaN and no other
        g = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype)
        g[4] = 0.0
        keep = [0, 1, 2, 3, 5]
        _, gw = torch.autograd.grad((y,), (xg, wg), (g.cuda(),))
        clean = x[keep].cuda().requires_grad_()
        wc = w.cuda().requires_grad_()
        yc, _ = norm.rms_norm(clean, wc, EPS, relu=relu)
        gx, gwc = torch.autograd.grad((yc,), (clean, wc), (g[keep].cuda(),))
        gn = torch.where(want[keep] > 0, g[keep].double(), 0.0) if relu else g[keep].double()
        wanted = (gn * z[keep]).sum(0)
        assert torch.equal(gwc.cpu().isnan(), wanted.isnan()), width
        assert bool(gw.isnan().all())
        fine = ~wanted.isnan()
        bound = (77 * o.HALF32) * (gn * z[keep]).abs().sum(0) + o.half_step(dtype) * 1.01 * wanted.abs()
        if bool(fine.any()):
            o.assert_within(gwc.cpu()[fine], wanted[fine], bound[fine], f"grad w {width}")
        assert bool(gx[[1, 3]].isnan().all()) and bool(gx[[0, 2, 4]].isfinite().all())


def test_gradient_of_rows_near_the_lower_end():
    """Rows of 1e-30: 1 / rms is 1e30, and the gradient is of that size: no term on the way leaves fp32's range."""
    for width in (47, 260, 5120):
        gen = torch.Generator().manual_seed(width)
        x = torch.randn(5, width, generator=gen) * 1e-30
        w = torch.rand(width, generator=gen) + 0.5
        g = torch.randn(5, width, generator=gen)
        xg = x.cuda().requires_grad_()
        y, _ = norm.rms_norm(xg, w.cuda(), 1e-70)
        (got,) = torch.autograd.grad((y,), (xg,), (g.cuda(),))
        y64, z, r = o.rms_norm(x.double(), w.double(), 1e-70, False)
        o.assert_within(y, y64, 4 * o.HALF32 * y64.abs(), "y")
        gw = g.double() * w.double()
        c = (gw * z).mean(-1, keepdim=True)
        terms = (gw.abs() + z.abs() * c.abs()) * r
        bound = 8 * o.HALF32 * terms + 2 * o.HALF32 * z.abs() * r * (gw * z).abs().mean(-1, keepdim=True)
        o.assert_within(got, (gw - z * c) * r, bound, "grad x")
