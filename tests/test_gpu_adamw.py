"""AdamW over many tensors: one step against the formula in 64 bits, the 8-bit states against their definition, the
optimizer class against torch's, checkpoints, and captured steps.

Tolerances, in half steps of fp32 (2^-24): m and v are two products and a sum: 4 of their terms' magnitudes.  The update
u = lr / c1 * m / (sqrt(v / c2) + eps): m and v 4 each (v halved by the root), the two corrections 4 each (their logarithm,
product and expm1), five more operations: 24 of |u|, taken twice for m's terms cancelling: 24 |u'| with u' from the terms'
magnitudes; p itself 3 of |p|."""
import copy

import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import optim

pytestmark = pytest.mark.gpu
H = o.HALF32
SIZES = [1, 3, 127, 128, 129, 1000, 4095, 4096, 4097, 8192, 20001]
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.999), 1e-8, 0.02


def case(sizes, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    t = {"p": [torch.randn(n, generator=gen) for n in sizes]}
    t["g"] = [(torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen))).to(dtype) for n in sizes]
    t["m"] = [0.3 * torch.randn(n, generator=gen) for n in sizes]
    t["v"] = [torch.rand(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen)) for n in sizes]
    return t


def formula(p, g, m, v, t, lr=LR, betas=BETAS, eps=EPS, wd=WD):
    """(p, m, v) after step t in 64 bits, and what each may be off by in fp32."""
    b1, b2 = betas
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v2 / (1 - b2 ** t)).sqrt() + eps
    rate = lr / (1 - b1 ** t)
    mt = b1 * m.abs() + (1 - b1) * g.abs()
    p2 = p * (1 - lr * wd) - rate * m2 / denom
    return p2, m2, v2, 3 * H * p.abs() + 24 * H * rate * mt / denom, 4 * H * mt, 4 * H * v2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_step_with_states_in_32_bits(dtype, grad_dtype, shift):
    """Every size; ``shift`` 1: tensors that start 4 (2) bytes off a wide load's alignment, in one allocation whose other
    values stay as they are; a step count of its own for each tensor."""
    t = case(SIZES, 1, grad_dtype)
    place = lambda x: torch.cat([torch.full((shift,), 9.0).to(x.dtype), x, torch.full((5,), 9.0).to(x.dtype)]).cuda()  # noqa: E731
    whole = {k: [place(x) for x in xs] for k, xs in t.items()}
    cut = {k: [w[shift:shift + n] for w, n in zip(ws, SIZES)] for k, ws in whole.items()}
    masters = cut["p"] if dtype == torch.bfloat16 else None
    params = [torch.zeros(n, dtype=dtype, device="cuda") for n in SIZES] if masters else cut["p"]
    taken = [7 * i for i in range(len(SIZES))]
    steps = torch.tensor(taken, dtype=torch.int32, device="cuda")
    optim.adamw_step(params, cut["g"], cut["m"], cut["v"], steps, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD,
                     masters=masters)
    assert steps.tolist() == [s + 1 for s in taken]
    for i, n in enumerate(SIZES):
        args = [t[k][i].double() for k in ("p", "g", "m", "v")]
        p, m, v, ep, em, ev = formula(*args, taken[i] + 1)
        o.assert_within(cut["p"][i], p, ep, f"p {n}")
        o.assert_within(cut["m"][i], m, em, f"m {n}")
        o.assert_within(cut["v"][i], v, ev, f"v {n}")
        if masters:
            assert torch.equal(params[i], cut["p"][i].bfloat16())
        for k in ("p", "g", "m", "v"):
            assert bool((whole[k][i][:shift] == 9).all()) and bool((whole[k][i][shift + n:] == 9).all())


def states8(t):
    """The 8-bit form of a case's states by the oracle's quantiser, and the values they stand for."""
    out = {"m": [], "u": [], "m_scales": [], "u_scales": [], "m64": [], "u64": []}
    for m, v in zip(t["m"], t["v"]):
        for key, x in (("m", m.double()), ("u", v.double().sqrt())):
            full = torch.zeros(o.padded(x.numel()), dtype=torch.float64)
            full[:x.numel()] = x
            codes, e = o.quantize_blocks(full.view(-1, 128))
            out[key].append(codes.view(-1)[:x.numel()].float().to(torch.float8_e4m3fn).cuda())
            out[key + "_scales"].append((e.view(-1) + 127).to(torch.uint8).cuda().view(torch.float8_e8m0fnu))
            out[key + "64"].append((codes * torch.exp2(e)).view(-1)[:x.numel()])
    return out


def blocks(x):
    full = torch.zeros(o.padded(x.numel()), dtype=torch.float64)
    full[:x.numel()] = x
    return full.view(-1, 128)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_with_states_in_8_bits(dtype):
    """m's code is the nearest to an m that is 4 half steps off; sqrt(v)'s is one of the two neighbours (a whole step away
    at most); the scales are the smallest that hold the block; zero stays zero and nothing above zero becomes zero."""
    t = case(SIZES, 2, dtype)
    t["g"][5][:300] = 0.0
    t["m"][5][:300] = 0.0
    t["v"][5][:300] = 0.0
    s = states8(t)
    masters = [p.cuda() for p in t["p"]]
    params = masters if dtype == torch.float32 else [p.bfloat16() for p in masters]
    steps = torch.full((len(SIZES),), 41, dtype=torch.int32, device="cuda")
    again = copy.deepcopy((params, s, steps, masters))
    for params_, s_, steps_, masters_ in ((params, s, steps, masters), again):
        optim.adamw_step(params_, [g.cuda() for g in t["g"]], s_["m"], s_["u"], steps_, lr=LR, betas=BETAS, eps=EPS,
                         weight_decay=WD, masters=masters_ if dtype == torch.bfloat16 else None,
                         exp_avg_scales=s_["m_scales"], exp_avg_sq_scales=s_["u_scales"], seed=77)
    for key in ("m", "u", "m_scales", "u_scales"):              # the same call gives the same bits
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(s[key], again[1][key]))
    for i, n in enumerate(SIZES):
        args = [t["p"][i].double(), t["g"][i].double(), s["m64"][i], s["u64"][i] ** 2]
        p, m, v, ep, em, ev = formula(*args, 42)
        o.assert_within(masters[i], p, ep, f"p {n}")
        if dtype == torch.bfloat16:
            assert torch.equal(params[i], masters[i].bfloat16())
        u, eu = v.sqrt(), 4 * H * v.sqrt()
        for key, want, slack in (("m", m, em), ("u", u, eu)):
            scale = s[key + "_scales"][i].double().cpu()
            top = blocks(want).abs().amax(1)
            assert bool((top <= 448 * scale * (1 + 16 * H)).all())
            assert bool(((top * (1 + 16 * H) > 224 * scale) | (scale == 2.0 ** -126)).all())
            got = s[key][i].double().cpu() * scale.repeat_interleave(128)[:n]
            step = torch.maximum(2 * o.STEP8 * want.abs(), scale.repeat_interleave(128)[:n] * 2.0 ** -9)
            if key == "m":  # its terms may cancel: its own error beside the half step
                o.assert_within(got, want, step / 2 * (1 + 2 ** -10) + em, "m code")
            else:
                # (a value that carries into the next power of two is a step of that power away)
                o.assert_within(got, want, step * (1 + 2 ** -10) + eu, "sqrt(v) code")
                assert bool(((got > 0) == (want > 0)).all())
    assert bool((s["m"][5][:256].float() == 0).all()) and bool((s["u"][5][:256].float() == 0).all())


def test_second_moment_is_rounded_without_bias():
    """One million values between two codes: the mean of the rounded ones is the value, to 5 standard deviations of a mean
    of a million two-valued variables (at most half a step each: 5 * 0.5 / 1000 of a step)."""
    n = 1 << 20
    for fraction in (0.03, 0.25, 0.5, 0.8):
        want = (8 + fraction) / 8                               # codes 1 and 1.125 around it, the block's top fixed at 448
        u = torch.full((n,), want, dtype=torch.float64)
        u[::128] = 448.0
        zero = torch.zeros(n, device="cuda")
        # v with beta2 = 0: v = g^2, so sqrt(v) is |g|
        p, steps = torch.zeros(n, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        m8, u8 = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        ms, us = (torch.ones(n // 128, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
        seen = []
        for seed in (1, 2):
            optim.adamw_step([p], [u.float().cuda()], [m8], [u8], steps, lr=0.0, betas=(0.0, 0.0), eps=1.0,
                             weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[us], seed=seed)
            got = (u8.double() * us.double().repeat_interleave(128)).view(-1, 128)[:, 1:]
            assert set(got.unique().tolist()) == {1.0, 1.125}
            assert abs(((got - want) / 0.125).mean().item()) <= 2.5e-3, (fraction, seed)
            seen.append(got)
        assert torch.equal(p, zero) and not torch.equal(seen[0], seen[1])


def test_more_tensors_than_one_launch_takes_and_empty_ones():
    sizes = [0, 5, 4096, 0] * 30 + [0]                          # 121 tensors, three launches
    t = case(sizes, 3, torch.float32)
    dev_ = {k: [x.cuda() for x in xs] for k, xs in t.items()}
    steps = torch.zeros(len(sizes), dtype=torch.int32, device="cuda")
    optim.adamw_step(dev_["p"], dev_["g"], dev_["m"], dev_["v"], steps, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    assert steps.tolist() == [1] * len(sizes)
    for i in range(len(sizes)):
        p, m, v, ep, em, ev = formula(*[t[k][i].double() for k in ("p", "g", "m", "v")], 1)
        o.assert_within(dev_["p"][i], p, ep, f"p {i}")
        o.assert_within(dev_["v"][i], v, ev, f"v {i}")


def test_spoiled_gradients_stay_where_they_are():
    """An infinity or NaN reaches its own element (32 bits); in 8 bits its code becomes NaN and its block keeps a finite
    scale and the other elements' codes."""
    n = 256
    g = torch.randn(n)
    g[3], g[200] = float("nan"), float("inf")
    clean = torch.where(g.isfinite(), g, 0.0)
    ps = []
    for grad in (g, clean):
        p, m8, u8 = torch.ones(n, device="cuda"), *(torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        ms, us = (torch.ones(2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
        optim.adamw_step([p], [grad.cuda()], [m8], [u8], torch.zeros(1, dtype=torch.int32, device="cuda"), lr=LR,
                         exp_avg_scales=[ms], exp_avg_sq_scales=[us])
        ps.append((p.cpu(), m8.float().cpu(), u8.float().cpu(), ms.float().cpu(), us.float().cpu()))
    fine = g.isfinite()
    for a, b in zip(ps[0][:3], ps[1][:3]):
        assert torch.equal(a[fine], b[fine]) and not bool(a[~fine].isfinite().all())
    for a, b in zip(ps[0][3:], ps[1][3:]):
        assert torch.equal(a, b)


def models(dtype, seed=0):
    torch.manual_seed(seed)
    make = lambda: torch.nn.Sequential(torch.nn.Linear(70, 130), torch.nn.LayerNorm(130), torch.nn.Linear(130, 9)).to(dtype).cuda()  # noqa: E731
    a = make()
    b = copy.deepcopy(a)
    return a, b


def test_class_follows_torchs():
    """Eight steps beside torch.optim.AdamW in 64 bits with the same gradients, in two groups, one parameter without a
    gradient in some steps: each step adds its own error, 24 half steps of a rate's size (|u| <= 10 lr here)."""
    a, b = models(torch.float32)
    b = b.double()
    groups = lambda m: [dict(params=list(m[0].parameters()) + list(m[1].parameters())),  # noqa: E731
                        dict(params=list(m[2].parameters()), lr=2e-2, weight_decay=0.0)]
    ours, theirs = optim.AdamW(groups(a), lr=1e-2), torch.optim.AdamW(groups(b), lr=1e-2)
    gen = torch.Generator().manual_seed(5)
    for step in range(8):
        for i, (p, q) in enumerate(zip(a.parameters(), b.parameters())):
            g = torch.randn(p.shape, generator=gen)
            skip = i == 3 and step in (0, 4)
            p.grad, q.grad = (None, None) if skip else (g.cuda(), g.double().cuda())
        ours.step()
        theirs.step()
    for p, q in zip(a.parameters(), b.parameters()):
        o.assert_within(p, q.detach().cpu(), 8 * (3 * H * (q.abs().cpu() + 0.2) + 24 * H * 10 * 2e-2), "parameter")
    assert [int(ours.state[p]["step"]) for p in a.parameters()] == [8, 8, 8, 6, 8, 8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_continue_bit_for_bit(dtype, bits):
    a, b = models(dtype)
    ours = optim.AdamW(a.parameters(), lr=1e-2, state_bits=bits, min_8bit_size=1000, seed=3)
    gen = torch.Generator().manual_seed(6)

    def step(model, opt, gs):
        for p, g in zip(model.parameters(), gs):
            p.grad = g.to(dtype).cuda()
        opt.step()

    grads = [[torch.randn(p.shape, generator=gen) for p in a.parameters()] for _ in range(6)]
    for gs in grads[:3]:
        step(a, ours, gs)
    kinds = {ours.state[p]["exp_avg"].dtype for p in a.parameters()}
    assert kinds == ({torch.float32} if bits == 32 else {torch.float32, torch.float8_e4m3fn})
    saved = copy.deepcopy(ours.state_dict())
    b.load_state_dict(a.state_dict())
    other = optim.AdamW(b.parameters(), lr=5.0, state_bits=bits, min_8bit_size=1000, seed=3)
    other.load_state_dict(saved)
    assert other.param_groups[0]["lr"] == 1e-2
    third = copy.deepcopy(other.state_dict())                   # saved again before any step
    assert set(third["state"][0]) == set(saved["state"][0])
    for gs in grads[3:]:
        step(a, ours, gs)
        step(b, other, gs)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
        for key, t in ours.state[p].items():
            u = other.state[q][key]
            assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, u.view(torch.uint8) if u.element_size() == 1 else u), key
    wrong = optim.AdamW(b.parameters(), state_bits=40 - bits, min_8bit_size=1000)
    bad = copy.deepcopy(saved)
    for g in bad["param_groups"]:
        g["state_bits"] = 40 - bits
    with pytest.raises(RuntimeError, match="does not fit"):
        wrong.load_state_dict(bad)


def test_takes_over_torchs_states():
    a, b = models(torch.float32)
    theirs = torch.optim.AdamW(a.parameters(), lr=1e-2)
    for p in a.parameters():
        p.grad = torch.ones_like(p)
    theirs.step()
    b.load_state_dict(a.state_dict())
    ours = optim.AdamW(b.parameters())
    ours.load_state_dict(theirs.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(theirs.state[p]["exp_avg"], ours.state[q]["exp_avg"]) and int(ours.state[q]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_their_replays(bits):
    """A captured step, replayed with the program's own work in between and the learning rate changed on the device, does
    what eager steps do, bit for bit."""
    a, b = models(torch.float32)
    lr = [torch.tensor(1e-2, device="cuda") for _ in range(2)]
    opts = [optim.AdamW(m.parameters(), lr=r, state_bits=bits, min_8bit_size=1000) for m, r in zip((a, b), lr)]
    gen = torch.Generator().manual_seed(8)
    grads = [[torch.randn(p.shape, generator=gen).cuda() for p in a.parameters()] for _ in range(6)]
    for m in (a, b):
        for p in m.parameters():
            p.grad = torch.zeros_like(p)

    def give(m, gs):
        for p, g in zip(m.parameters(), gs):
            p.grad.copy_(g)

    fresh = optim.AdamW(a.parameters())
    graph = torch.cuda.CUDAGraph()
    for opt, m in zip(opts, (a, b)):
        give(m, grads[0])
        opt.step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opts[1].step()
        with pytest.raises(RuntimeError, match="before capturing"):
            fresh.step()
    for i, gs in enumerate(grads[1:]):
        noise = torch.randn(256, 256, device="cuda")
        float((noise @ noise).sum())
        for m, opt, r in zip((a, b), opts, lr):
            r.fill_(1e-2 / (i + 1))
            give(m, gs)
        opts[0].step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.equal(p, q), i
            for key, t in opts[0].state[p].items():
                u = opts[1].state[q][key]
                assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, u.view(torch.uint8) if u.element_size() == 1 else u)


def test_refusals():
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    m, v = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    s = torch.zeros(1, dtype=torch.int32, device="cuda")
    eight = torch.zeros(300, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.ones(3, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    bad = [([p], [g[:299]], [m], [v], s, {}), ([p], [g, g], [m], [v], s, {}), ([p], [g.half()], [m], [v], s, {}),
           ([p], [g.cpu()], [m], [v], s, {}), ([p], [g], [m], [v], s.long(), {}), ([p], [g], [m], [v], s.cpu(), {}),
           ([p[::2]], [g[:150]], [m[:150]], [v[:150]], s, {}), ([p], [g], [eight], [eight], s, {}),
           ([p], [g], [eight], [v], s, {}), ([p], [g], [m], [v], s, dict(exp_avg_scales=[scales])),
           ([p], [g], [eight], [eight], s, dict(exp_avg_scales=[scales[:2]], exp_avg_sq_scales=[scales])),
           ([p.bfloat16()], [g], [m], [v], s, {}), ([p], [g], [m], [v], s, dict(masters=[p])),
           ([p], [g], [m], [v], s, dict(lr=torch.ones(2, device="cuda")))]
    for i, (ps, gs, ms, vs, steps, more) in enumerate(bad):
        print("refusal", i, flush=True)
        with pytest.raises(RuntimeError, match="Input mismatch"):
            optim.adamw_step(ps, gs, ms, vs, steps, **{"lr": 0.1, **more})
    assert bool((p == 1).all()) and int(s) == 0
    q = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
    q.grad = torch.ones(4, 4, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        optim.AdamW([q]).step()
