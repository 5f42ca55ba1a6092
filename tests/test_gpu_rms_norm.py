"""RMS norm with the residual's addition: forward, 8-bit output and gradient against the formula in 64 bits.

Tolerances count roundings (half a step of fp32 is 2^-24, of bf16 2^-8, relative).  h is one rounded addition: equal.
y = h r w: r is rounded once (its 64-bit value is exact beside that), two products: 3 half steps of fp32 and the store's;
4 are allowed for second-order terms.  The gradient, per element, with z = h r and c = mean(gn w z):
  grad = (gn w - z c) r + grad_h:  at most 8 roundings on each of its terms, plus c's own error, where gn w was rounded
  before the sum (64 bits) was taken: a half step of mean|gn w z|.
grad w: a chain of at most rows + 70 fp32 additions of gn z with 2 roundings each."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import norm

pytestmark = pytest.mark.gpu
EPS = 1e-6

SHAPES = [(1, 1), (3, 1), (5, 7), (64, 16), (37, 32), (4, 47), (257, 64), (33, 100), (7, 128), (9, 129), (65, 256),
          (13, 300), (5, 512), (3, 1000), (2, 1024), (3, 1025), (2, 2048), (3, 4097), (2, 5120), (3, 6148), (1, 8192),
          (2, 10007), (2, 16384), (2100, 8), (700, 260)]


def data(rows, width, dtype, residual, seed=0):
    gen = torch.Generator().manual_seed(seed + 1000 * rows + width)
    x = torch.randn(rows, width, generator=gen).to(dtype)
    res = torch.randn(rows, width, generator=gen).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=gen)).to(dtype)
    gy = torch.randn(rows, width, generator=gen).to(dtype)
    gh = torch.randn(rows, width, generator=gen).to(dtype) if residual else None
    return x, res, w, gy, gh


def cuda(t):
    return None if t is None else t.cuda()


def stream_of(x, res):
    return x if res is None else (x.float() + res.float()).to(x.dtype)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_gradient(dtype, residual, relu):
    for rows, width in SHAPES:
        print(f"rms_norm rows={rows} width={width} {dtype} residual={residual} relu={relu}", flush=True)
        x, res, w, gy, gh = data(rows, width, dtype, residual)
        xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        rg = res.cuda().requires_grad_() if residual else None
        y, h = norm.rms_norm(xg, wg, EPS, residual=rg, relu=relu)
        want_h = stream_of(x, res)
        assert o.same(h.detach(), want_h)
        h64, w64 = want_h.double(), w.double()
        y64, z, r = o.rms_norm(h64, w64, EPS, relu)
        store = 0.0 if dtype == torch.float32 else o.HALF16 * 1.01
        o.assert_within(y, y64, (4 * o.HALF32 + store) * y64.abs(), "y")
        outs, grads = ((y, h), (gy.cuda(), gh.cuda())) if residual else ((y,), (gy.cuda(),))
        got = torch.autograd.grad(outs, (xg, wg) + ((rg,) if residual else ()), grads)
        gn = torch.where(y64 > 0, gy.double(), 0.0) if relu else gy.double()
        gw = gn * w64
        c = (gw * z).mean(-1, keepdim=True)
        dx = (gw - z * c) * r + (gh.double() if residual else 0.0)
        terms = (gw.abs() + z.abs() * c.abs()) * r + (gh.double().abs() if residual else 0.0)
        bound = 8 * o.HALF32 * terms + 2 * o.HALF32 * z.abs() * r * (gw * z).abs().mean(-1, keepdim=True)
        o.assert_within(got[0], dx, bound + store * dx.abs(), "grad x")
        dw = (gn * z).sum(0)
        o.assert_within(got[1], dw, (rows + 72) * o.HALF32 * (gn * z).abs().sum(0) + store * dw.abs(), "grad w")
        if residual:
            assert torch.equal(got[0], got[2])


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_output_in_8_bits(dtype, relu):
    """A code is the nearest to a y that is 4 half steps of fp32 off at most: half a step of e4m3, or of its
    subnormals (2^-10 of the scale), and those 4 on top; a scale is the smallest that holds the block, to the same 4."""
    for residual in (False, True):
        for rows, width in SHAPES:
            print(f"rms_norm_fp8 rows={rows} width={width} {dtype} residual={residual} relu={relu}", flush=True)
            x, res, w, _, _ = data(rows, width, dtype, residual, seed=5)
            q, h = norm.rms_norm_fp8(x.cuda(), w.cuda(), EPS, residual=cuda(res), relu=relu)
            want_h = stream_of(x, res)
            assert o.same(h, want_h) and q.cols == width
            y, _, _ = o.rms_norm(want_h.double(), w.double(), EPS, relu)
            full = torch.zeros(rows, o.padded(width), dtype=torch.float64)
            full[:, :width] = y
            codes, scale = q.codes.double().cpu(), q.scales.double().cpu()
            assert codes.shape == full.shape and bool((codes[:, width:] == 0).all())
            top = full.view(rows, -1, 128).abs().amax(2)
            slack = 1 + 8 * o.HALF32
            assert bool((top <= 448 * scale * slack).all())
            assert bool(((top * slack > 224 * scale) | (scale == 2.0 ** -126)).all())
            s = scale.repeat_interleave(128, 1)
            bound = torch.maximum(o.STEP8 * full.abs(), s * 2.0 ** -10) * slack + 8 * o.HALF32 * full.abs()
            o.assert_within(codes * s, full, bound, "codes")


def test_forward_and_8_bit_output_agree():
    """fp32 rows: the codes are those of the fp32 y that the plain form returns, bit for bit."""
    from gnn_benchmark_amd import fp8

    for rows, width in [(65, 256), (9, 129), (4, 47), (3, 4097), (2, 5120)]:
        x, res, w, _, _ = data(rows, width, torch.float32, True, seed=9)
        y, h = norm.rms_norm(x.cuda(), w.cuda(), EPS, residual=res.cuda())
        q, h8 = norm.rms_norm_fp8(x.cuda(), w.cuda(), EPS, residual=res.cuda())
        want = fp8.quantize_rows(y)
        assert torch.equal(h, h8)
        assert torch.equal(q.codes.view(torch.uint8), want.codes.view(torch.uint8))
        assert torch.equal(q.scales.view(torch.uint8), want.scales.view(torch.uint8))


def test_rows_of_other_strides_and_places():
    """Column blocks of wider arrays, rows that start off a 16-byte boundary, a transposed view, leading dimensions,
    a broadcast residual: the bits of the contiguous call."""
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(40, 203, generator=gen).cuda()
    w = torch.randn(64, generator=gen).cuda()
    for x in (wide[:, 1:65], wide[:, 4:68], wide[:, 139:203], wide.t()[3:50, :].t()[:, :47][:, :47].repeat(1, 2)[:, :64]):
        y, _ = norm.rms_norm(x, w, EPS)
        want, _ = norm.rms_norm(x.clone(memory_format=torch.contiguous_format), w, EPS)
        assert torch.equal(y, want)
    t = torch.randn(64, 33, generator=gen).cuda().t()          # [33, 64] stored by column
    assert torch.equal(norm.rms_norm(t, w, EPS)[0], norm.rms_norm(t.contiguous(), w, EPS)[0])
    x3 = torch.randn(3, 5, 64, generator=gen).cuda()
    y3, h3 = norm.rms_norm(x3, w, EPS, residual=x3[:1, :1].expand(3, 5, 64))
    want, hw = norm.rms_norm(x3.view(15, 64), w, EPS, residual=x3[0, 0].repeat(15, 1))
    assert y3.shape == (3, 5, 64) and torch.equal(y3.view(15, 64), want) and torch.equal(h3.view(15, 64), hw)
    off = torch.randn(33 * 64 + 1, generator=gen).cuda()[1:].view(33, 64)  # 4 bytes off
    assert torch.equal(norm.rms_norm(off, w, EPS)[0], norm.rms_norm(off.clone(), w, EPS)[0])
    q, _ = norm.rms_norm_fp8(off, w, EPS)
    assert torch.equal(q.codes.view(torch.uint8), norm.rms_norm_fp8(off.clone(), w, EPS)[0].codes.view(torch.uint8))


def test_broadcast_residual_gets_its_summed_gradient():
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(6, 40, generator=gen).cuda()
    res = torch.randn(1, 40, generator=gen).cuda().requires_grad_()
    w = torch.randn(40, generator=gen).cuda()
    gy = torch.randn(6, 40, generator=gen).cuda()
    y, _ = norm.rms_norm(x, w, EPS, residual=res.expand(6, 40))
    (got,) = torch.autograd.grad((y,), (res,), (gy,))
    full = res.detach().expand(6, 40).contiguous().requires_grad_()
    y, _ = norm.rms_norm(x, w, EPS, residual=full)
    (rows,) = torch.autograd.grad((y,), (full,), (gy,))
    assert torch.equal(got, rows.sum(0, keepdim=True))


def test_extreme_rows():
    """Zero rows give zeros; rows near the ends of fp32's range are normalised like others (the squares are 64 bits); an
    infinity or NaN spoils its own row alone, with NaN codes and a finite scale beside it."""
    width = 260
    gen = torch.Generator().manual_seed(6)
    base = torch.randn(8, width, generator=gen)
    x = base.clone()
    x[1] = 0.0
    x[2] *= 1e30
    x[3] *= 1e-30
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    w = torch.rand(width, generator=gen) + 0.5
    xg = x.cuda().requires_grad_()
    y, _ = norm.rms_norm(xg, w.cuda(), 0.0 + 1e-70)
    fine = [0, 2, 3, 6, 7]
    y64, z, r = o.rms_norm(x.double(), w.double(), 1e-70, False)
    o.assert_within(y[fine], y64[fine], 4 * o.HALF32 * y64[fine].abs(), "y")
    assert bool((y[1] == 0).all())
    assert bool(y[4].isnan().any()) and bool(y[5].isnan().all())
    gy = torch.randn(8, width, generator=gen)
    (gx,) = torch.autograd.grad((y,), (xg,), (gy.cuda(),))
    gw = gy.double() * w.double()
    c = (gw * z).mean(-1, keepdim=True)
    dx = (gw - z * c) * r
    terms = (gw.abs() + z.abs() * c.abs()) * r
    bound = 8 * o.HALF32 * terms + 2 * o.HALF32 * z.abs() * r * (gw * z).abs().mean(-1, keepdim=True)
    o.assert_within(gx[[0, 2, 6, 7]], dx[[0, 2, 6, 7]], bound[[0, 2, 6, 7]], "grad x")
    assert bool(gx[5].isnan().all()) and not bool(gx[6].isnan().any())
    q, _ = norm.rms_norm_fp8(x.cuda(), w.cuda(), 1e-6)
    codes = q.codes.float().cpu()
    assert bool(codes[5, :width].isnan().all()) and not bool(codes[[0, 1, 2, 3, 6, 7]].isnan().any())
    assert bool(torch.isfinite(q.scales.float()).all())


def test_empty_and_unused_outputs():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y, h = norm.rms_norm(x, w, EPS)
    assert y.shape == (0, 16)
    gx, gw = torch.autograd.grad((y,), (x, w), (torch.empty_like(y),))
    assert gx.shape == (0, 16) and bool((gw == 0).all())
    q, _ = norm.rms_norm_fp8(x.detach(), w.detach(), EPS)
    assert q.codes.shape == (0, 128)
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    r = torch.randn(4, 16, device="cuda", requires_grad=True)
    y, h = norm.rms_norm(x, w, EPS, residual=r)
    gx, gr = torch.autograd.grad((h.sum(),), (x, r), retain_graph=True)  # only the stream is used
    assert bool((gx == 1).all()) and bool((gr == 1).all())
    gx, = torch.autograd.grad((y.sum(),), (x,))                        # only y is used
    assert bool(torch.isfinite(gx).all())


def test_weight_in_fp32_with_bf16_rows_and_equal_calls():
    x, res, _, gy, gh = data(300, 172, torch.bfloat16, True, seed=11)
    w = 1 + 0.3 * torch.randn(172, generator=torch.Generator().manual_seed(1))
    runs = []
    for _ in range(2):
        xg, wg, rg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), res.cuda().requires_grad_()
        y, h = norm.rms_norm(xg, wg, EPS, residual=rg)
        runs.append((y, h) + torch.autograd.grad((y, h), (xg, wg, rg), (gy.cuda(), gh.cuda())))
    assert all(torch.equal(a, b) for a, b in zip(*runs)) and runs[0][3].dtype == torch.float32
    y64, _, _ = o.rms_norm(stream_of(x, res).double(), w.double(), EPS, False)
    o.assert_within(runs[0][0], y64, (4 * o.HALF32 + o.HALF16 * 1.01) * y64.abs(), "y")


def test_another_stream():
    x = torch.randn(5000, 256, device="cuda")
    w = torch.rand(256, device="cuda")
    want, _ = norm.rms_norm(x, w, EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = norm.rms_norm(x, w, EPS)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
