"""The training operators in the ways a program calls them: many rows and large tiles of the products in every form, on
another stream, and a whole step captured into a HIP graph and replayed between eager work."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import fp8, norm, optim
from test_gpu_fp8 import as_quantized_rows, whole_rows, whole_weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", [(40003, 300, 131), (60000, 512, 172), (45001, 1, 1), (8200, 4100, 4099)])
def test_every_form_of_the_large_products(m, k, n):
    """Whole numbers, so every form is exact: fp32 and bf16 results, with a bias, into a column block off its alignment,
    the input gradient; a spoiled row spoils no other."""
    gen = torch.Generator().manual_seed(m)
    codes, e, x = whole_rows(m, k, gen, scale_from=0)
    w, values = whole_weight(k, n, gen)
    q, x, values = as_quantized_rows(codes, e, k), x.cuda(), values.cuda()
    bias = torch.randint(-8, 9, (n,), generator=gen).float().cuda()
    want = x @ values
    assert torch.equal(fp8.product(q, w).double(), want)
    want += bias.double()
    for dtype in (torch.float32, torch.bfloat16):
        rounded = want.float().to(dtype)
        assert torch.equal(fp8.product(q, w, bias, out_dtype=dtype), rounded)
        wide = torch.full((m, n + 9), 7.0, device="cuda", dtype=dtype)
        fp8.product(q, w, bias, out=wide[:, 5:5 + n])
        assert torch.equal(wide[:, 5:5 + n], rounded) and bool((wide[:, :5] == 7).all()) and bool((wide[:, 5 + n:] == 7).all())
        q.codes.view(torch.uint8)[m // 2, 0] = 0x7f  # NaN
        spoiled = fp8.product(q, w, bias, out_dtype=dtype)
        assert bool(spoiled[m // 2].isnan().all())
        spoiled[m // 2] = rounded[m // 2]
        assert torch.equal(spoiled, rounded)
        q.codes[m // 2] = codes[m // 2].float().cuda().to(torch.float8_e4m3fn)
    codes, e, g = whole_rows(m, n, gen, scale_from=0)
    grad = fp8.product(as_quantized_rows(codes, e, n), w, input_gradient=True)
    assert torch.equal(grad.double(), g.cuda() @ values.t())


def training_step(dtype, rows=700, width=300, hidden=260):
    """The operators of a training step on tensors of its own: what it computes, every time from the same values."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    x, r = normal(rows, width).to(dtype), normal(rows, width).to(dtype)
    nw, w, b = (1 + 0.1 * normal(width)), normal(width, hidden) / 16, normal(hidden)
    w2 = normal(hidden, 50) / 16
    g, gh = normal(rows, 50).to(dtype), normal(rows, width).to(dtype)
    moments = torch.rand(4, width * hidden, device="cuda", generator=gen) * 1e-3

    def work():
        leaves = [t.clone().requires_grad_() for t in (x, r, nw, w, b, w2)]
        hid, h = fp8.norm_linear(leaves[0], leaves[2], 1e-6, leaves[3], leaves[4], residual=leaves[1], relu=True)
        y, _ = norm.rms_norm(hid, torch.ones_like(b), 1e-6, relu=True)
        out = fp8.linear(y, leaves[5])
        grads = torch.autograd.grad((out, h), leaves, (g, gh))
        params = [leaves[i].detach().clone() for i in (3, 4)]
        step = [grads[3].contiguous(), grads[4].contiguous()]
        m = [moments[0].clone(), moments[1, :hidden].clone()]
        v = [moments[2].clone(), moments[3, :hidden].clone()]
        steps = torch.full((2,), 3, dtype=torch.int32, device="cuda")
        optim.adamw_step(params, step, m, v, steps, lr=0.01)
        big = leaves[3].detach().clone()
        eight = [fp8.quantize_rows(torch.nn.functional.pad(t, (0, -t.numel() % 128)).view(-1, 128))
                 for t in (moments[0], moments[2])]
        codes = [q.codes.view(-1)[:width * hidden] for q in eight]
        optim.adamw_step([big], [grads[3].contiguous()], codes[:1], codes[1:], steps[:1], lr=0.01, seed=9,
                         exp_avg_scales=[eight[0].scales], exp_avg_sq_scales=[eight[1].scales])
        rows8, _ = norm.rms_norm_fp8(x, nw)
        return [out.detach(), h.detach(), *grads, *params, *m, *v, steps, big, eight[0].codes.view(torch.uint8),
                eight[1].codes.view(torch.uint8), eight[1].scales.view(torch.uint8), rows8.codes.view(torch.uint8)]

    return work


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 700, 41000])
def test_a_step_replays_from_a_hip_graph(dtype, rows):
    work = training_step(dtype, rows)
    eager = [t.clone() for t in work()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for got, want in zip(work(), eager):                # another stream, the same bits
            assert torch.equal(got, want)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    with torch.cuda.graph(second):                          # a second graph beside it: workspaces are each one's own
        held2 = work()
    for replay in range(3):
        noise = torch.randn(512, 512, device="cuda")
        float((noise * noise).max())
        for t in held + held2:
            t.zero_()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for i, (got, got2, want) in enumerate(zip(held, held2, eager)):
            assert torch.equal(got, want), (replay, i)
            assert torch.equal(got2, want), (replay, i)


def test_two_streams_at_once():
    """The same calls side by side on two streams, each with its own results."""
    work = training_step(torch.float32, 5000)
    eager = [t.clone() for t in work()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(work())
    torch.cuda.synchronize()
    for got in results:
        for i, (a, b) in enumerate(zip(got, eager)):
            assert torch.equal(a, b), i


def test_the_same_memory_twice_is_refused():
    p, q, g = (torch.ones(300, device="cuda") for _ in range(3))
    states = [torch.zeros(300, device="cuda") for _ in range(4)]
    steps = torch.zeros(2, dtype=torch.int32, device="cuda")
    empty = torch.zeros(0, device="cuda")
    for ps, ms, vs in (([p, p], states[:2], states[2:]), ([p, q], states[:1] * 2, states[2:]),
                       ([p, q], states[:2], [states[2], states[0]])):
        with pytest.raises(RuntimeError, match="same memory"):
            optim.adamw_step(ps, [g, g], ms, vs, steps, lr=0.1)
    assert bool((p == 1).all()) and bool((q == 1).all()) and int(steps.sum()) == 0
    optim.adamw_step([p, q], [g, g], states[:2], states[2:], steps, lr=0.1)    # one gradient for two is fine
    assert torch.equal(p, q) and bool((p < 1).all())
    optim.adamw_step([empty, empty], [empty, empty], [empty, empty], [empty, empty], steps, lr=0.1)


def test_a_gradients_gradient_is_refused():
    x = torch.randn(40, 96, device="cuda", requires_grad=True)
    w = torch.randn(96, 33, device="cuda", requires_grad=True)
    nw = torch.ones(96, device="cuda", requires_grad=True)
    for out in (fp8.linear(x, w), norm.rms_norm(x, nw)[0], fp8.norm_linear(x, nw, 1e-6, w, residual=x)[0]):
        (once,) = torch.autograd.grad((out.sum(),), (x,), create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            (once.sum() + x.sum()).backward()


def test_only_what_is_wanted_gets_a_gradient():
    """Every choice of leaves that want a gradient gives the gradients that all of them together give."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    values = [normal(50, 200), normal(50, 200), 1 + 0.1 * normal(200), normal(200, 70) / 14, normal(70)]
    g, gh = normal(50, 70), normal(50, 200)

    def grads(which):
        leaves = [v.clone().requires_grad_(i in which) for i, v in enumerate(values)]
        out, h = fp8.norm_linear(leaves[0], leaves[2], 1e-6, leaves[3], leaves[4], residual=leaves[1])
        used = [leaves[i] for i in which]
        return torch.autograd.grad((out, h) if {0, 1} & set(which) else (out,), used, (g, gh) if {0, 1} & set(which) else (g,))

    every = grads([0, 1, 2, 3, 4])
    for which in ([0], [1], [3], [4], [0, 3], [1, 4], [3, 4]):
        for i, got in zip(which, grads(which)):
            assert torch.equal(got, every[i]), (which, i)
    only_norm = grads([2])[0]                               # (h needs no gradient there, so none comes back through it)
    x = (values[0] + values[1]).requires_grad_()
    nw = values[2].clone().requires_grad_()
    out, _ = fp8.norm_linear(x, nw, 1e-6, values[3], values[4])
    assert torch.equal(only_norm, torch.autograd.grad((out,), (nw,), (g,))[0])


def test_arrays_beyond_2_to_31_elements():
    """The last rows of arrays of more than 2^31 elements get what they get by themselves (rows do not depend on others; the
    last 50 000 go through the same kernels as all)."""
    rows, width, tail = (1 << 23) + 70_001, 256, 50_000
    assert rows * width > 1 << 31
    x = torch.empty(rows, width, device="cuda").normal_()
    nw = torch.rand(width, device="cuda") + 0.5
    w = fp8.quantize_weight(torch.randn(width, 256, device="cuda") / 16, True)
    q, part = fp8.quantize_rows(x), fp8.quantize_rows(x[-tail:])
    same = lambda a, b: torch.equal(a[-tail:].view(torch.uint8), b.view(torch.uint8))  # noqa: E731
    assert same(q.codes, part.codes) and same(q.scales, part.scales)
    assert torch.equal(fp8.product(q, w)[-tail:], fp8.product(part, w))
    assert torch.equal(fp8.product(q, w, out_dtype=torch.bfloat16)[-tail:], fp8.product(part, w, out_dtype=torch.bfloat16))
    got, h = norm.rms_norm_fp8(x, nw, residual=x, relu=True)
    want, h_tail = norm.rms_norm_fp8(x[-tail:], nw, residual=x[-tail:], relu=True)
    assert same(got.codes, want.codes) and same(got.scales, want.scales) and torch.equal(h[-tail:], h_tail)
    del got, h
    leaf = x.requires_grad_()
    y, _ = norm.rms_norm(leaf, nw)
    (dx,) = torch.autograd.grad((y,), (leaf,), (x.detach(),))
    small = x.detach()[-tail:].clone().requires_grad_()
    y_tail, _ = norm.rms_norm(small, nw)
    (dx_tail,) = torch.autograd.grad((y_tail,), (small,), (small.detach(),))
    assert torch.equal(y[-tail:], y_tail) and torch.equal(dx[-tail:], dx_tail)
    del y, dx
    # columns of g that are one in the last row alone and zero elsewhere: the weight gradient is that row of x
    g = torch.zeros(rows, width, device="cuda")
    g[-1] = 1.0
    dw, db = fp8.weight_gradient(q, g, True)
    assert torch.equal(dw, part.dequantize()[-1].unsqueeze(1).expand(width, width)) and bool((db == 1).all())
    del q
    # the optimizer, in 32 and in 8 bits (whose second state alone depends on the element's number)
    x = x.detach().view(-1)
    at = x.numel() - 5000 // 128 * 128 - x.numel() % 128
    for bits in (32, 8):
        def states(n):
            if bits == 32:
                return [torch.zeros(n, device="cuda") for _ in "mv"], {}
            codes = [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "mv"]
            scales = [torch.ones(-(-n // 128), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in "mv"]
            return codes, dict(exp_avg_scales=scales[:1], exp_avg_sq_scales=scales[1:])

        p, p_tail = x.clone(), x[at:].clone()
        g = g.view(-1).normal_()
        for param, grad in ((p, g), (p_tail, g[at:])):
            (m, v), more = states(param.numel())
            optim.adamw_step([param], [grad], [m], [v], torch.zeros(1, dtype=torch.int32, device="cuda"), lr=0.1, **more)
        assert torch.equal(p[at:], p_tail)
