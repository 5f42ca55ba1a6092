"""Products in 8-bit floating point: the format bit for bit, products exactly on whole numbers and within their roundings
on random ones, gradients against the formula and against differences.

Tolerances: a product of K terms accumulated in fp32 is off by at most 2 (K + 8) half steps of the sum of its terms'
magnitudes (2: the matrix unit may cut where it adds), plus the store's half step; operands on whole numbers below 2^24
leave no rounding at all.  Products stored as bf16 run on the matrix unit's 8-bit instruction.  Among the products of eight
neighbouring codes it cuts each to a multiple of 2^-13 of the largest one's power of two (65536 + 7 gives 65536 there and
65536 + 8 gives 65544): less than 7 * 2^-13 of the largest product for the eight, so of the sum of magnitudes for all."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import fp8, norm

pytestmark = pytest.mark.gpu


def check_rows(q, x):
    codes, e, _ = o.quantize_rows(x.double())
    assert q.cols == x.size(1) and o.same(q.codes, codes) and o.same(q.scales, torch.exp2(e))


ROWS = [(1, 1), (3, 1), (1, 128), (5, 127), (7, 129), (64, 100), (33, 300), (2, 4097), (1000, 47), (257, 512)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_into_the_format(dtype):
    for rows, width in ROWS:
        print(f"quantize_rows {rows} x {width} {dtype}", flush=True)
        gen = torch.Generator().manual_seed(rows * 7919 + width)
        spread = torch.exp(3 * torch.randn(rows, width, generator=gen))
        x = (torch.randn(rows, width, generator=gen) * spread).to(dtype)
        check_rows(fp8.quantize_rows(x.cuda()), x)
        values = o.quantize_rows(x.double())[2]
        assert o.same(fp8.quantize_rows(x.cuda()).dequantize(), values)
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(30, 333, generator=gen).to(dtype)
    for cut in (wide[:, 1:130], wide[:, 4:260], wide[::2, :47], wide.t()):
        check_rows(fp8.quantize_rows(wide.cuda()[:, 1:130]), wide[:, 1:130])
        g = cut.cuda() if cut.is_contiguous() else torch.empty_strided(cut.shape, cut.stride(), dtype=dtype, device="cuda").copy_(cut)
        check_rows(fp8.quantize_rows(g), cut)
    assert fp8.quantize_rows(torch.empty(0, 5, dtype=dtype, device="cuda")).codes.shape == (0, 128)


def test_borders_of_the_format():
    """Ties, subnormal codes, zero blocks, tops at a power's border, the ends of fp32's range, infinities and NaN."""
    ticks = torch.arange(0, 128, dtype=torch.float32)
    rows = [ticks / 16 * 2.0 ** -6,                            # halves of subnormal codes among normal ones
            torch.cat([torch.tensor([448.0]), 16 + ticks[:127] / 2]),   # ties between codes of step 2
            torch.zeros(128), torch.full((128,), 448.0), torch.full((128,), 448.00003),
            torch.cat([torch.tensor([3.4e38, -3.4e38]), ticks[:126] * 1e36]),
            torch.cat([torch.tensor([1e-38, 1e-45]), ticks[:126] * 1e-40]),
            torch.cat([torch.tensor([float("inf"), float("nan"), -float("inf")]), ticks[:125]]),
            torch.full((128,), float("nan")), -ticks]
    x = torch.stack(rows)
    check_rows(fp8.quantize_rows(x.cuda()), x)
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 128)
    check_rows(fp8.quantize_rows(every.cuda()), every)         # every bf16 value there is
    check_rows(fp8.quantize_rows(every.float().cuda()), every)


WEIGHTS = [(1, 1), (1, 200), (200, 1), (128, 128), (127, 129), (129, 127), (300, 172), (512, 256), (47, 260)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_into_the_format(dtype):
    for k, n in WEIGHTS:
        print(f"quantize_weight {k} x {n} {dtype}", flush=True)
        gen = torch.Generator().manual_seed(k * 7919 + n)
        w = (torch.randn(k, n, generator=gen) * torch.exp(2 * torch.randn(k, 1, generator=gen))).to(dtype)
        codes, e, _ = o.quantize_weight(w.double())
        for g in (w.cuda(), w.t().contiguous().cuda().t()):    # stored by input, stored by output
            q = fp8.quantize_weight(g, for_gradient=True)
            assert (q.k, q.n) == (k, n) and o.same(q.scales, torch.exp2(e))
            full = torch.zeros(n, o.padded(k), dtype=torch.float64)
            full[:, :k] = codes.t()
            assert o.same(q.codes, full)
            full = torch.zeros(k, o.padded(n), dtype=torch.float64)
            full[:, :n] = codes
            assert o.same(q.codes_by_input, full)
    w = torch.randn(40, 77).to(dtype)
    w[3, 5], w[20, 70] = float("inf"), float("nan")
    codes, e, _ = o.quantize_weight(w.double())
    q = fp8.quantize_weight(w.cuda())
    assert o.same(q.codes[:, :40], codes.t()) and o.same(q.scales, torch.exp2(e)) and q.codes_by_input is None


def whole_rows(rows, width, gen, scale_from=-3):
    """Codes that are whole numbers up to 8 with scales of a few powers of two, and the values they stand for."""
    codes = torch.zeros(rows, o.padded(width), dtype=torch.float64)
    codes[:, :width] = torch.randint(-8, 9, (rows, width), generator=gen).double()
    e = torch.randint(scale_from, scale_from + 4, (rows, o.padded(width) // 128), generator=gen)
    values = (codes.view(rows, -1, 128) * torch.exp2(e.double()).unsqueeze(2)).view(rows, -1)[:, :width]
    return codes, e, values


def as_quantized_rows(codes, e, width):
    return fp8.QuantizedRows(codes.float().to(torch.float8_e4m3fn).cuda(),
                             (e + 127).to(torch.uint8).cuda().view(torch.float8_e8m0fnu), width)


def whole_weight(k, n, gen):
    kb, nb = o.padded(k) // 128, o.padded(n) // 128
    codes = torch.randint(-8, 9, (k, n), generator=gen).double()
    e = torch.randint(-2, 2, (kb, nb), generator=gen)
    values = codes * torch.exp2(e.double()).repeat_interleave(128, 0).repeat_interleave(128, 1)[:k, :n]
    by_output, by_input = torch.zeros(n, kb * 128), torch.zeros(k, nb * 128)
    by_output[:, :k], by_input[:, :n] = codes.t(), codes
    q = fp8.QuantizedWeight(k, n, by_output.to(torch.float8_e4m3fn).cuda(),
                            (e + 127).to(torch.uint8).cuda().view(torch.float8_e8m0fnu),
                            by_input.to(torch.float8_e4m3fn).cuda())
    return q, values


PRODUCTS = [(1, 1, 1), (1, 128, 16), (2, 300, 17), (15, 127, 3), (16, 129, 100), (17, 512, 172), (31, 16, 128),
            (33, 1024, 129), (63, 300, 256), (64, 128, 128), (65, 256, 130), (127, 47, 47), (128, 512, 256),
            (129, 1300, 260), (200, 640, 511), (1000, 172, 300), (3000, 128, 16), (40, 5000, 33), (300, 2048, 1)]


def test_products_of_whole_numbers_are_exact():
    for m, k, n in PRODUCTS:
        print(f"product {m} x {k} x {n}", flush=True)
        gen = torch.Generator().manual_seed(m * 31 + k * 17 + n)
        codes, e, x = whole_rows(m, k, gen)
        q = as_quantized_rows(codes, e, k)
        w, values = whole_weight(k, n, gen)
        bias = torch.randint(-8, 9, (n,), generator=gen).float()
        want = x @ values
        assert o.same(fp8.product(q, w), want)
        assert o.same(fp8.product(q, w, bias.cuda()), want + bias.double())
        assert o.same(fp8.product(q, w, bias.cuda(), out_dtype=torch.bfloat16), (want + bias.double()).float().bfloat16())
        codes, e, g = whole_rows(m, n, gen)
        assert o.same(fp8.product(as_quantized_rows(codes, e, n), w, input_gradient=True), g @ values.t())
        wide = torch.full((m, n + 9), 7.0, device="cuda")       # a column block of a wider array, off its alignment
        fp8.product(q, w, out=wide[:, 5:5 + n])
        assert o.same(wide[:, 5:5 + n], want) and bool((wide[:, :5] == 7).all()) and bool((wide[:, 5 + n:] == 7).all())
        g = torch.randint(-8, 9, (m, n), generator=gen).float()
        for dtype in (torch.float32, torch.bfloat16):
            dw, db = fp8.weight_gradient(q, g.to(dtype).cuda(), with_bias=True)
            assert o.same(dw, x.t() @ g.double()) and o.same(db, g.double().sum(0))


@pytest.mark.parametrize("m,k,n", [(20000, 256, 172), (70001, 130, 47), (5000, 1000, 1100), (30000, 16, 8)])
def test_many_rows_of_whole_numbers(m, k, n):
    """Enough rows for several tiles a compute unit and several slices of the weight gradient."""
    gen = torch.Generator().manual_seed(m)
    codes, e, x = whole_rows(m, k, gen, scale_from=0)
    w, values = whole_weight(k, n, gen)
    q = as_quantized_rows(codes, e, k)
    assert o.same(fp8.product(q, w), (x.float() @ values.float()))     # (below 2^24 eighths: fp32 is exact too)
    g = torch.randint(-1, 2, (m, n), generator=gen).float()
    dw, db = fp8.weight_gradient(q, g.cuda(), with_bias=True)
    assert o.same(dw, x.t() @ g.double()) and o.same(db, g.double().sum(0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_and_its_gradients(dtype):
    store = 0.0 if dtype == torch.float32 else o.HALF16 * 1.01
    for m, k, n in [(1, 128, 64), (5, 47, 172), (64, 300, 129), (130, 256, 172), (1000, 128, 256), (77, 1500, 40)]:
        print(f"linear {m} x {k} x {n} {dtype}", flush=True)
        gen = torch.Generator().manual_seed(m + k + n)
        x = torch.randn(m, k, generator=gen).to(dtype)
        w = (torch.randn(k, n, generator=gen) * k ** -0.5).to(dtype)
        b = torch.randn(n, generator=gen).to(dtype)
        g = torch.randn(m, n, generator=gen).to(dtype)
        xg, wg, bg = (t.cuda().requires_grad_() for t in (x, w, b))
        out = fp8.linear(xg, wg, bg)
        got = torch.autograd.grad((out,), (xg, wg, bg), (g.cuda(),))
        xq, wq, gq = o.quantize_rows(x.double())[2], o.quantize_weight(w.double())[2], o.quantize_rows(g.double())[2]
        gh = g.bfloat16().double()
        acc = lambda terms, a, b: 2 * (terms + 8) * o.HALF32 * (a.abs() @ b.abs())  # noqa: E731
        for name, value, a, c, terms, extra in (("out", out, xq, wq, k, b.double()), ("grad x", got[0], gq, wq.t(), n, 0.0),
                                                ("grad w", got[1], xq.t(), gh, m, 0.0)):
            want = a @ c + extra
            slack = acc(terms, a, c) + (o.HALF32 * 4 * want.abs() if name == "out" else 0.0)
            if dtype == torch.bfloat16 and name != "grad w":
                slack = slack + 7 * 2.0 ** -13 * (a.abs() @ c.abs())
            o.assert_within(value, want, slack * 1.01 + store * want.abs() + 1e-30, name)
        want = g.double().sum(0)
        o.assert_within(got[2], want, (m + 8) * o.HALF32 * g.double().abs().sum(0) + store * want.abs(), "grad b")
        # a Linear's weight, stored by output, and leading dimensions: the same bits
        lin = w.t().contiguous().cuda()
        assert torch.equal(fp8.linear(x.cuda(), lin.t(), b.cuda()), out.detach())
        assert torch.equal(fp8.linear(x.cuda().view(1, m, 1, k), w.cuda(), b.cuda()).view(m, n), out.detach())


def test_gradient_against_differences_on_the_grid():
    """Operands on the format's grid that stay on it when moved by one (a top of 448 in every block keeps the scale at 1):
    the product is bilinear there, so the difference quotient is the derivative, and whole numbers make both exact."""
    gen = torch.Generator().manual_seed(2)
    m, k, n = 40, 256, 130
    x = torch.randint(-7, 8, (m, k), generator=gen).float()
    x[:, ::128] = 448.0
    w = torch.randint(-7, 8, (k, n), generator=gen).float()
    w[::128, ::128] = 448.0
    g = torch.randint(-7, 8, (m, n), generator=gen).float()
    g[:, ::128] = 448.0
    dx, dw = torch.randint(-1, 2, (m, k), generator=gen).float(), torch.randint(-1, 2, (k, n), generator=gen).float()
    dx[:, ::128], dw[::128, ::128] = 0.0, 0.0
    f = lambda x, w: (fp8.linear(x.cuda(), w.cuda()).double() * g.cuda().double()).sum().item()  # noqa: E731
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    gx, gw = torch.autograd.grad((fp8.linear(xg, wg),), (xg, wg), (g.cuda(),))
    assert (f(x + dx, w) - f(x - dx, w)) / 2 == (gx.double() * dx.cuda().double()).sum().item()
    assert (f(x, w + dw) - f(x, w - dw)) / 2 == (gw.double() * dw.cuda().double()).sum().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_linear_is_the_norm_then_the_layer(dtype, residual):
    """The pair's bits are those of its parts; its gradient is theirs, where the parts hand the rows' gradient on in the
    same type."""
    for m, k, n in [(1, 4096, 300), (50, 129, 172), (700, 256, 130)]:
        gen = torch.Generator().manual_seed(m + k)
        x = torch.randn(m, k, generator=gen).to(dtype).cuda().requires_grad_()
        r = torch.randn(m, k, generator=gen).to(dtype).cuda().requires_grad_() if residual else None
        nw = (1 + 0.2 * torch.randn(k, generator=gen)).to(dtype).cuda().requires_grad_()
        w = (torch.randn(k, n, generator=gen) * k ** -0.5).to(dtype).cuda().requires_grad_()
        b = torch.randn(n, generator=gen).to(dtype).cuda().requires_grad_()
        g, gh = torch.randn(m, n, generator=gen).to(dtype).cuda(), torch.randn(m, k, generator=gen).to(dtype).cuda()
        out, h = fp8.norm_linear(x, nw, 1e-6, w, b, residual=r, relu=True)
        with torch.no_grad():
            rows, h2 = norm.rms_norm_fp8(x, nw, 1e-6, residual=r, relu=True)
            assert torch.equal(out, fp8.product(rows, fp8.quantize_weight(w), b, out_dtype=dtype)) and torch.equal(h, h2)
            rows_grad = fp8.product(fp8.quantize_rows(g), fp8.quantize_weight(w, True), out_dtype=dtype, input_gradient=True)
        leaves = [t for t in (x, r, nw, w, b) if t is not None]
        outs, grads = ((out, h), (g, gh)) if residual else ((out,), (g,))
        got = torch.autograd.grad(outs, leaves, grads)
        y, h3 = norm.rms_norm(x, nw, 1e-6, residual=r, relu=True)
        want = torch.autograd.grad((y, h3) if residual else (y,), leaves[:-2],
                                   (rows_grad, gh) if residual else (rows_grad,))
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        dw, db = fp8.weight_gradient(rows, g, True)
        assert torch.equal(got[-2], dw.to(dtype)) and torch.equal(got[-1], db.to(dtype))


def test_a_spoiled_row_spoils_no_other():
    x = torch.randn(200, 256, device="cuda")
    w = torch.randn(256, 130, device="cuda")
    spoiled = x.clone()
    spoiled[17, 3], spoiled[120, 200] = float("inf"), float("nan")
    for rows in (slice(None), slice(100, 130)):                # the tiled and the few-row kernel, each beside itself
        want, out = fp8.linear(x[rows], w), fp8.linear(spoiled[rows], w)
        bad = spoiled[rows].isfinite().all(1).logical_not()
        assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], want[~bad])


def test_refusals():
    x = torch.randn(8, 256, device="cuda")
    w = torch.randn(256, 64, device="cuda")
    q, qw = fp8.quantize_rows(x), fp8.quantize_weight(w)
    bad = [lambda: fp8.quantize_rows(x.half()), lambda: fp8.quantize_rows(x[0]), lambda: fp8.quantize_weight(w[0]),
           lambda: fp8.product(q, fp8.quantize_weight(w[:128])), lambda: fp8.product(q, qw, torch.ones(63, device="cuda")),
           lambda: fp8.product(q, qw, out=torch.empty(8, 63, device="cuda")),
           lambda: fp8.product(q, qw, out=torch.empty(64, 8, device="cuda").t()),
           lambda: fp8.product(q, qw, out_dtype=torch.float16), lambda: fp8.product(q, qw, input_gradient=True),
           lambda: fp8.product(fp8.QuantizedRows(q.codes[:, 16:], q.scales, 240), qw),
           lambda: fp8.product(fp8.QuantizedRows(q.codes, q.scales[:, :1], 256), qw),
           lambda: fp8.product(fp8.QuantizedRows(q.codes.view(torch.uint8), q.scales, 256), qw),
           lambda: fp8.product(q, fp8.QuantizedWeight(256, 64, qw.codes, qw.scales.view(torch.uint8))),
           lambda: fp8.weight_gradient(q, x[:4]), lambda: fp8.linear(x, w.t()), lambda: fp8.linear(x, w, torch.ones(5, device="cuda")),
           lambda: fp8.linear(x, w.cpu()), lambda: fp8.linear(x.double(), w.double()),
           lambda: fp8.quantize_rows(x.requires_grad_()), lambda: norm.rms_norm_fp8(x.requires_grad_(), torch.ones(256, device="cuda")),
           lambda: norm.rms_norm(x, torch.ones(255, device="cuda")), lambda: norm.rms_norm(x, torch.ones(256, device="cuda").bfloat16()),
           lambda: norm.rms_norm(x, torch.ones(256, device="cuda"), residual=x[:4])]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            print("refusal", i, flush=True)
            call()
    with pytest.raises(RuntimeError, match="16384"):
        norm.rms_norm(torch.ones(1, 16385, device="cuda"), torch.ones(16385, device="cuda"))
