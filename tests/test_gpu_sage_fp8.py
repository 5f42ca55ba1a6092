"""The SAGE layer and model with 8-bit products, the residual stream's RMS norm and AdamW, as a training step runs them.

* A layer's output and gradients against the formula in 64 bits: quantised operands (the oracle's format), the aggregation
  and its transpose on the CPU.  The layer's left operand is taken as the aggregation wrote it, so that a value beside a
  border of the format is quantised from the same bits on both sides; its own rounding is checked apart.  Tolerances: those
  of test_gpu_fp8.py for the products, and for a gradient through the aggregation of a row's d terms 2 (d + 2) half steps
  of the sum of their magnitudes, on top of the product's error carried along.
* The model with RMS norms and products of fp32 accuracy against autograd on the CPU, at the 1e-4 relative that
  test_gpu_sage.py derives for the same products behind LayerNorm.
* The whole step in 8 bits against the same step composed by hand from the public entry points: bit for bit.
"""
import copy

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import fp8_oracle as o
from gnn_benchmark_amd import aggregator, fp8, gcn, norm, optim, sage, synthetic
from test_gpu_sage import CpuAggregate, CpuSageLayer, ReplayExchange, _cpu_mats

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def partition(n, width, is_pre_delay, seed=11):
    part = synthetic.partition_edges(n, 4, 2, 6, 1.8, 800, 1500, 9000, seed=seed, device=DEV)
    exchange = ReplayExchange(5)
    return synthetic.build_partition_graph(part, width, is_pre_delay, exchange=exchange, device=DEV), exchange


def dense64(m):
    return m.to_dense().double()


def product_slack(terms, a, b):
    return 2 * (terms + 8) * o.HALF32 * (a.abs() @ b.abs())


@pytest.mark.parametrize("is_pre_delay", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("fi,fo", [(32, 47), (172, 64)])
def test_layer_against_the_formula(is_pre_delay, bias, fi, fo):
    n = 2000
    graph, exchange = partition(n, max(fi, 2 * fo), is_pre_delay)
    a_local, a_in, a_out_t = (dense64(m) for m in _cpu_mats(graph, is_pre_delay))
    deg = graph.in_degrees.double().cpu()
    gen = torch.Generator(device=DEV).manual_seed(fi)
    x = torch.randn(n, fi, device=DEV, generator=gen)
    g = torch.randn(n, fo, device=DEV, generator=gen)
    torch.manual_seed(1)
    conv = sage.DistSAGEConvGrad(fi, fo, 32, is_pre_delay, bias=bias, gemm="fp8").to(DEV).train()
    if bias:
        with torch.no_grad():
            conv.bias.uniform_(-1, 1)
    w, b = conv.weight.detach().double().cpu(), conv.bias.detach().double().cpu() if bias else 0.0
    g64, x64 = g.double().cpu(), x.double().cpu()

    def carried_back(grad_agg, slack):
        """A^T of the gradient that reaches the aggregated rows, its error bound, the rows received on the way back
        apart."""
        terms = 2 * (a_local != 0).sum(0).unsqueeze(1) + 2 * (a_out_t != 0).sum(1).unsqueeze(1) + 8
        incoming = a_out_t @ exchange.rows["backward0"].double()
        want = a_local.t() @ grad_agg + incoming
        size = a_local.abs().t() @ grad_agg.abs() + a_out_t.abs() @ exchange.rows["backward0"].double().abs()
        return want, a_local.abs().t() @ slack + terms * o.HALF32 * size

    # ---- aggregate, then multiply
    staged = sage.stage_input(x).requires_grad_()
    out = conv(graph, staged, 0)
    got = torch.autograd.grad((out,), [staged, *conv.parameters()], (g,))
    rows = staged.detach().double().cpu()
    agg = (a_local @ x64 + a_in @ exchange.rows["forward0"].double()) / deg
    size = (a_local.abs() @ x64.abs() + a_in.abs() @ exchange.rows["forward0"].double().abs()) / deg
    terms = 2 * ((a_local != 0).sum(1) + (a_in != 0).sum(1)).unsqueeze(1) + 8
    o.assert_within(rows[:, :fi].float(), agg, terms * o.HALF32 * size, "aggregated rows")
    rq, wq, gq = o.quantize_rows(rows)[2], o.quantize_weight(w)[2], o.quantize_rows(g64)[2]
    o.assert_within(out, rq @ wq + b, product_slack(2 * fi, rq, wq) + 4 * o.HALF32 * (rq @ wq + b).abs() + 1e-30, "out")
    gh = g.bfloat16().double().cpu()
    o.assert_within(got[1], rq.t() @ gh, product_slack(n, rq.t(), gh), "grad w")
    if bias:
        o.assert_within(got[2], g64.sum(0), (n + 8) * o.HALF32 * g64.abs().sum(0), "grad b")
    both, slack = gq @ wq.t(), product_slack(fo, gq, wq.t())
    want, off = carried_back(both[:, :fi] / deg, slack[:, :fi] / deg * 1.01 + 2 * o.HALF32 * both[:, :fi].abs() / deg)
    want = want + both[:, fi:]
    o.assert_within(got[0][:, fi:], want, off + slack[:, fi:] + 4 * o.HALF32 * (want.abs() + both[:, fi:].abs()), "grad x")

    # ---- the same for some of the nodes: their rows' bits are the full layer's where the product's kernel is the same
    some = torch.randperm(n, device=DEV, generator=gen)[:333]
    again = sage.stage_input(x).requires_grad_()
    part = conv(graph, again, 0, some)
    o.assert_within(part, (rq @ wq + b)[some.cpu()], (product_slack(2 * fi, rq, wq)
                    + 4 * o.HALF32 * (rq @ wq + b).abs() + 1e-30)[some.cpu()], "restricted out")
    grad_part, grad_w = torch.autograd.grad((part,), [again, conv.weight], (g[some],))
    cut = some.cpu()
    o.assert_within(grad_w, rq[cut].t() @ gh[cut], product_slack(len(cut), rq[cut].t(), gh[cut]), "restricted grad w")
    only = torch.zeros(n, 2 * fi, dtype=torch.float64)
    only[cut] = both[cut]
    loose = torch.zeros_like(only)
    loose[cut] = slack[cut]
    want, off = carried_back(only[:, :fi] / deg, loose[:, :fi] / deg * 1.01 + 2 * o.HALF32 * only[:, :fi].abs() / deg)
    want = want + only[:, fi:]
    o.assert_within(grad_part[:, fi:], want, off + loose[:, fi:] + 4 * o.HALF32 * (want.abs() + only[:, fi:].abs()),
                    "restricted grad x")
    assert bool((grad_part[:, :fi] == 0).all())

    # ---- multiply, then aggregate
    conv.linear_first = True
    staged = sage.stage_input(x).requires_grad_()
    out = conv(graph, staged, 0)
    assert torch.equal(conv(graph, x, 0), out)
    got = torch.autograd.grad((out,), [staged, *conv.parameters()], (g,))
    stacked = torch.cat([w[:fi], w[fi:]], 1)
    xq, sq = o.quantize_rows(x64)[2], o.quantize_weight(stacked)[2]
    first, slack = xq @ sq, product_slack(fi, xq, sq)
    received = exchange.rows["forward0"].double()
    out_want = (a_local @ first[:, :fo] + a_in @ received) / deg + first[:, fo:] + b
    size = (a_local.abs() @ first[:, :fo].abs() + a_in.abs() @ received.abs()) / deg + first[:, fo:].abs() + abs(b)
    o.assert_within(out, out_want, a_local.abs() @ slack[:, :fo] / deg * 1.01 + slack[:, fo:] * 1.01
                    + (terms + 4) * o.HALF32 * size, "out, product first")
    grad_left, off = carried_back(g64 / deg, 2 * o.HALF32 * g64.abs() / deg)
    # its codes come from the run's own rows; here both sides of the check share them through a half step of the format
    grad_both = torch.cat([grad_left, g64], 1)
    gq = o.quantize_rows(grad_both)
    step = 2 * o.STEP8 * grad_both.abs() + torch.exp2(gq[1]).repeat_interleave(128, 1)[:, :2 * fo] * 2.0 ** -8
    off = torch.cat([off, torch.zeros_like(off)], 1) + step
    o.assert_within(got[0][:, fi:], gq[2] @ sq.t(), off @ sq.abs().t() + product_slack(2 * fo, gq[2], sq.t()) * 1.2,
                    "grad x, product first")
    gh, loose = grad_both, torch.cat([carried_back(g64 / deg, 2 * o.HALF32 * g64.abs() / deg)[1], 0 * g64], 1)
    grad_w = xq.t() @ gh
    off = xq.abs().t() @ (loose + o.HALF16 * gh.abs()) * 1.01 + product_slack(n, xq.t(), gh) * 1.01
    for half, cols in ((slice(0, fi), slice(0, fo)), (slice(fi, None), slice(fo, None))):
        o.assert_within(got[1][half], grad_w[:, cols], off[:, cols], "grad w, product first")
    if bias:
        o.assert_within(got[2], g64.sum(0), (n + 8) * o.HALF32 * g64.abs().sum(0), "grad b, product first")


@pytest.mark.parametrize("linear_first", [False, True])
def test_residual_model_matches_cpu_autograd(linear_first):
    """``norm="rms"`` with products of fp32 accuracy: loss, gradients and AdamW's update."""
    n, f_in, hidden, classes, layers = 5000, 32, 64, 12, 4
    graph, exchange = partition(n, hidden, True)
    torch.manual_seed(0)
    model = sage.DistSAGE(f_in, hidden, classes, num_layers=layers, dropout=0.5, is_pre_delay=True,
                          linear_first_when_narrowing=linear_first, norm="rms").to(DEV)
    with torch.no_grad():
        for layer_norm in model.norms:
            layer_norm.weight.uniform_(0.5, 1.5)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(n, f_in, device=DEV, generator=gen)
    labels = torch.randint(0, classes, (n,), device=DEV, generator=gen)
    train_idx = torch.randperm(n, device=DEV, generator=gen)[: n // 10]
    masks = sage.make_dropout_masks(n, hidden, layers, 0.5, 7, DEV)
    model.train()
    loss = F.nll_loss(model(graph, sage.stage_input(x), masks)[train_idx], labels[train_idx])
    loss.backward()

    a_local, a_in, a_out_t = _cpu_mats(graph, True)
    deg = graph.in_degrees.cpu()
    cpu_layers = [CpuSageLayer(conv) for conv in model.convs]
    weights = [m.weight.detach().cpu().clone().requires_grad_() for m in model.norms]
    y, h = x.cpu(), None
    for i, layer in enumerate(cpu_layers):
        def aggregate(t, i=i):
            incoming = exchange.rows.get(f"backward{i}", torch.zeros(a_out_t.shape[1], t.size(1)))
            return CpuAggregate.apply(t, a_local, a_in, a_out_t, exchange.rows[f"forward{i}"], incoming)

        z = layer(aggregate, y, deg, model.convs[i].linear_first)
        if i == layers - 1:
            break
        d = z * masks[i].cpu() * 2.0
        h = d if h is None else h + d
        y = torch.relu(h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * weights[i])
    cpu_loss = F.nll_loss(F.log_softmax(z, dim=1)[train_idx.cpu()], labels.cpu()[train_idx.cpu()])
    cpu_loss.backward()

    tol = 1e-4
    assert abs(float(loss.detach()) - float(cpu_loss.detach())) <= tol * max(1.0, abs(float(cpu_loss.detach())))
    pairs = [(f"gamma{i}", m.weight.grad, w.grad) for i, (m, w) in enumerate(zip(model.norms, weights))]
    for i, (conv, ref) in enumerate(zip(model.convs, cpu_layers)):
        pairs += [(f"weight{i}", conv.weight.grad, ref.stacked_grad()), (f"bias{i}", conv.bias.grad, ref.bias.grad)]
    for name, got, want in pairs:
        assert float((got.cpu() - want).abs().max()) <= 10 * tol * (float(want.abs().max()) + 1e-12), name

    # the update of those gradients, next to torch's on the CPU (test_gpu_adamw.py holds the step to its roundings)
    ours, theirs = list(model.parameters()), [p.detach().cpu().clone().requires_grad_() for p in model.parameters()]
    for p, q in zip(ours, theirs):
        q.grad = p.grad.cpu()
    optim.AdamW(ours, lr=0.01).step()
    torch.optim.AdamW(theirs, lr=0.01, eps=1e-8, weight_decay=1e-2).step()
    for p, q in zip(ours, theirs):
        assert float((p.detach().cpu() - q.detach()).abs().max()) <= 1e-6


def by_hand(model, state, graph, x, labels, train_idx, masks, step):
    """A training step from the operators one by one: gradients by autograd.grad, the update by adamw_step."""
    last = len(model.convs) - 1
    leaves = [p.detach().clone().requires_grad_() for p in model.parameters()]
    names = [name for name, _ in model.named_parameters()]
    value = dict(zip(names, leaves))
    y, h, both = sage.stage_input(x), None, None
    for i, conv in enumerate(model.convs):
        w, b = value[f"convs.{i}.weight"], value[f"convs.{i}.bias"]
        fo = conv.out_channels
        if both is not None:
            agg = aggregator.Aggregator.apply(graph, both[:, :fo], i, 32, True, True)
            z = both[:, fo:] + agg / graph.in_degrees
            both = None
        else:
            staged = y if i == 0 else torch.cat([torch.zeros_like(y), y], 1)
            z = fp8.linear(sage._StagedRows.apply(graph, staged, i, 32, True, True, True), w, b)
        if i == last:
            break
        z = z * masks[i] * 2.0
        weight = value[f"norms.{i}.weight"]
        after = model.convs[i + 1]
        if after.linear_first:
            w, b = value[f"convs.{i + 1}.weight"], value[f"convs.{i + 1}.bias"]
            both, h = fp8.norm_linear(z, weight, 1e-6, torch.cat([w[:after.in_channels], w[after.in_channels:]], 1),
                                      F.pad(b, (after.out_channels, 0)), residual=h, relu=True)
        else:
            y, h = norm.rms_norm(z, weight, 1e-6, residual=h, relu=True)
    loss = gcn._mean_nll(F.log_softmax(z[train_idx], dim=1), labels[train_idx])
    grads = torch.autograd.grad((loss,), leaves)
    with torch.no_grad():
        values = [p.detach() for p in leaves]
        big = [i for i, p in enumerate(values) if p.numel() >= 4096]
        small = [i for i, p in enumerate(values) if p.numel() < 4096]
        for group in (big, small):  # the optimizer's order: the first parameter is a big one
            number, bits8 = 0 if group is big else len(big), group is big
            if step == 0:
                for i in group:
                    size = values[i].numel()
                    if bits8:
                        state[i] = [torch.zeros(size, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in "mv"]
                        state[i] += [torch.ones(-(-size // 128), dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
                                     for _ in "mv"]
                    else:
                        state[i] = [torch.zeros(size, device=DEV) for _ in "mv"]
            steps = torch.full((len(group),), step, dtype=torch.int32, device=DEV)
            scales = dict(exp_avg_scales=[state[i][2] for i in group],
                          exp_avg_sq_scales=[state[i][3] for i in group]) if bits8 else {}
            optim.adamw_step([values[i] for i in group], [grads[i].contiguous() for i in group],
                             [state[i][0] for i in group], [state[i][1] for i in group], steps, lr=0.01, seed=3,
                             first=number, **scales)
    return loss.detach(), values


@pytest.mark.parametrize("linear_first", [False, True])
def test_a_training_step_in_8_bits_is_its_parts(linear_first, monkeypatch):
    """8-bit products, RMS norms with the residual stream and AdamW with 8-bit states in ``sage.train_step``, with every
    library product taken away: three steps, loss and parameters bit for bit those of the operators called by hand."""
    n, dims = 6000, [128, 256, 256, 172]
    graph, _ = partition(n, 2 * 256, True)
    torch.manual_seed(0)
    model = sage.DistSAGE(dims[0], dims[1], dims[-1], num_layers=3, dropout=0.5, is_pre_delay=True, gemm="fp8",
                          norm="rms", linear_first_when_narrowing=linear_first).to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(n, dims[0], device=DEV, generator=gen)
    labels = torch.randint(0, dims[-1], (n,), device=DEV, generator=gen)
    train_idx = torch.randperm(n, device=DEV, generator=gen)[: n // 10]
    masks = sage.make_dropout_masks(n, dims[1], 3, 0.5, 7, DEV)
    other = copy.deepcopy(model)
    opt = optim.AdamW(model.parameters(), lr=0.01, state_bits=8, seed=3)
    staged, state = sage.stage_input(x), {}

    def taken_away(*a, **k):
        raise AssertionError("a BLAS-library product inside the train step")

    for name in ("mm", "addmm", "matmul", "bmm", "baddbmm", "einsum"):
        monkeypatch.setattr(torch, name, taken_away)
    monkeypatch.setattr(torch.nn.functional, "linear", taken_away)
    with gcn.forbid_library_products():
        for step in range(3):
            got = sage.train_step(model, opt, graph, staged, labels, train_idx, masks, restrict_last_layer=False)
            want, values = by_hand(other, state, graph, x, labels, train_idx, masks, step)
            assert np.isfinite(float(got)) and torch.equal(got, want), step
            with torch.no_grad():
                for p, q, v in zip(model.parameters(), other.parameters(), values):
                    assert torch.equal(p.detach(), v), step
                    q.copy_(v)
        # only the scored nodes through the last layer: the same loss, its rows through another product kernel
        ref = float(sage.train_step(copy.deepcopy(model), optim.AdamW([torch.zeros(1, device=DEV)]), graph, staged, labels,
                                    train_idx, masks, restrict_last_layer=False))
        got = float(sage.train_step(model, opt, graph, staged, labels, train_idx, masks))
        assert abs(got - ref) <= 1e-4 * max(1.0, abs(ref))


def test_a_partition_without_nodes_and_refusals():
    with pytest.raises(ValueError, match="gemm"):
        sage.DistSAGEConvGrad(8, 8, 32, True, gemm="fp4")
    with pytest.raises(ValueError, match="norm"):
        sage.DistSAGE(8, 8, 8, norm="batch")
    w = torch.randn(96, 40, device=DEV, requires_grad=True)
    b = torch.randn(40, device=DEV, requires_grad=True)
    x = torch.randn(0, 96, device=DEV, requires_grad=True)
    out = fp8.linear(x, w, b)
    assert out.shape == (0, 40)
    gx, gw, gb = torch.autograd.grad((out,), (x, w, b), (torch.empty(0, 40, device=DEV),))
    assert gx.shape == (0, 96) and bool((gw == 0).all()) and bool((gb == 0).all())
    nw = torch.ones(96, device=DEV, requires_grad=True)
    out, h = fp8.norm_linear(x, nw, 1e-6, w, b, residual=x)
    got = torch.autograd.grad((out, h), (x, nw, w, b), (torch.empty(0, 40, device=DEV), torch.empty(0, 96, device=DEV)))
    assert got[0].shape == (0, 96) and all(bool((t == 0).all()) for t in got[1:])
    # a frozen weight beside a trained bias
    x = torch.randn(300, 96, device=DEV)
    g = torch.randint(-4, 5, (300, 40), device=DEV).float()
    (gb,) = torch.autograd.grad((fp8.linear(x, w.detach(), b),), (b,), (g,))
    assert torch.equal(gb.double(), g.double().sum(0))


@pytest.mark.parametrize("linear_first", [False, True])
@pytest.mark.parametrize("num_bits", [32, 16, 2])
def test_model_in_evaluation_and_with_narrow_exchanges(linear_first, num_bits):
    """Without dropout, evaluation gives the training pass's bits where rows travel as they are; with rows of 16 or
    2 bits a step runs to finite gradients.  Features that are staged or not give the same."""
    n = 3000
    part = synthetic.partition_edges(n, 4, 2, 6, 1.8, 800, 1500, 9000, seed=11, device=DEV)
    graph = synthetic.build_partition_graph(part, 128, True, exchange=synthetic.SeededHaloExchange(4), bits=num_bits,
                                            device=DEV, exchange_quantized=synthetic.SeededQuantizedHaloExchange(4),
                                            exchange_bf16=synthetic.SeededBf16HaloExchange(4))
    torch.manual_seed(0)
    model = sage.DistSAGE(100, 128, 47, num_layers=3, dropout=0.0, num_bits=num_bits, is_pre_delay=True, gemm="fp8",
                          norm="rms", linear_first_when_narrowing=linear_first).to(DEV)
    x = torch.randn(n, 100, device=DEV)
    out = model.train()(graph, sage.stage_input(x))
    assert torch.equal(model(graph, x).detach(), out.detach()) and bool(out.isfinite().all())
    if num_bits == 32:
        with torch.no_grad():
            assert torch.equal(model.eval()(graph, x), out.detach())
    out.square().mean().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()) and bool((p.grad != 0).any()), name


def test_degrees_folded_into_the_matrices():
    """The layer over a graph whose matrices hold the division: the same to rounding, which moves a value to the next code of
    its block now and then where rows are aggregated before they are quantised (a code's step is 2^-3 of the value at
    most; a value within 1e-6 of a border between codes is one in 10^5)."""
    n, fi, fo = 2000, 64, 47
    graph, _ = partition(n, 2 * fi, True)
    folded = sage.fold_in_degrees(graph)
    x = torch.randn(n, fi, device=DEV)
    g = torch.randn(n, fo, device=DEV)
    for linear_first in (False, True):
        torch.manual_seed(1)
        conv = sage.DistSAGEConvGrad(fi, fo, 32, True, gemm="fp8", linear_first=linear_first).to(DEV)
        results = []
        for over in (graph, folded):
            staged = sage.stage_input(x).requires_grad_()
            out = conv(over, staged, 0)
            results.append([out.detach(), *torch.autograd.grad((out,), [staged, *conv.parameters()], (g,))])
            results[-1][1] = results[-1][1][:, fi:]
        for a, b in zip(*results):
            assert float((a - b).norm()) <= 2e-3 * float(a.norm())
        if linear_first:
            assert float((results[0][0] - results[1][0]).abs().max()) <= 1e-5 * float(results[0][0].abs().max())
