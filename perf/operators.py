"""The 8-bit training operators -- RMS norm with the residual's addition, products in 8-bit floating point with one scale
per block of 128, AdamW over many tensors -- as cases to be measured, with a plain form of each.

``run(state)`` is one pass through an operator.  With ``own`` false it is written in elementary torch operations, with
``own`` true it makes the calls a user of gnn_benchmark_amd makes.

One 8-bit format throughout: e4m3 codes, blocks of 128 values, a scale per block that is a power of two in one byte
(e8m0), the smallest for which the block's largest finite magnitude stays at or below 448.  Rows are stored padded with
zeros to a whole number of blocks.
"""
import math

import torch

own = False
BLOCK = 128
EPS = 1e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a serving loop: residual added, normalised, handed on in 8 bits; latency is all there is
        {"name": "norm_fp8_token", "kind": "norm_fp8", "rows": 1, "width": 4096, "dtype": "bf16", "residual": True,
         "relu": False},
        # the pass between two residual SAGE layers of hidden width 256, its output kept in 8 bits for the next product
        {"name": "norm_fp8_hidden", "kind": "norm_fp8", "rows": 500009, "width": 256, "dtype": "fp32", "residual": True,
         "relu": True},
        # a narrow layer of an odd width (47 classes), training, no residual
        {"name": "norm_train_odd", "kind": "norm_train", "rows": 1000003, "width": 47, "dtype": "fp32",
         "residual": False, "relu": True},
        # wide rows in 16 bits with a residual stream, training
        {"name": "norm_train_wide", "kind": "norm_train", "rows": 8192, "width": 5120, "dtype": "bf16",
         "residual": True, "relu": False},
        # one token against a square weight: bound by the weight's bytes
        {"name": "product_token", "kind": "product", "rows": 1, "inner": 4096, "outer": 4096, "dtype": "bf16",
         "bias": False},
        # the stacked product of a SAGE layer, [A x | x] of 2 * 256 features to 256, a million nodes
        {"name": "product_hidden", "kind": "product", "rows": 1000003, "inner": 512, "outer": 256, "dtype": "fp32",
         "bias": True},
        # a large square product: bound by the matrix units
        {"name": "product_square", "kind": "product", "rows": 8192, "inner": 8192, "outer": 8192, "dtype": "bf16",
         "bias": False},
        # the last hidden layer to 172 outputs, forward and backward, an odd number of nodes
        {"name": "linear_hidden", "kind": "linear", "rows": 300007, "inner": 256, "outer": 172, "dtype": "fp32",
         "bias": True},
        # a wide layer in 16 bits, forward and backward
        {"name": "linear_wide", "kind": "linear", "rows": 8192, "inner": 4096, "outer": 4096, "dtype": "bf16",
         "bias": False},
        # the optimizer step of a three-layer SAGE model (128 -> 256 -> 256 -> 172): a few small tensors, launch-bound
        {"name": "adamw_model", "kind": "adamw", "count": 10, "total": 287916, "dtype": "fp32", "bits": 32, "taken": 9},
        # a learned table of node embeddings with its states in 8 bits
        {"name": "adamw_table_8bit", "kind": "adamw", "count": 2, "total": 128000384, "dtype": "fp32", "bits": 8,
         "taken": 200},
        # many 16-bit tensors with 32-bit masters and states
        {"name": "adamw_many", "kind": "adamw", "count": 200, "total": 60000007, "dtype": "bf16", "bits": 32,
         "taken": 1000},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm_fp8", "norm_train", "product", "linear", "adamw"])
    dtype = rng.choice(["fp32", "bf16"])
    if kind in ("norm_fp8", "norm_train"):
        width = _spread(rng, 1, 8192)
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(1000000, 40000000 // width))), "width": width,
                "dtype": dtype, "residual": rng.random() < 0.7, "relu": rng.random() < 0.3}
    if kind in ("product", "linear"):
        inner, outer = _spread(rng, 16, 8192 if kind == "product" else 4096), _spread(rng, 8, 4096)
        most = min(1000000, int((4e11 if kind == "product" else 1e11) / (inner * outer)), 400000000 // (inner + outer))
        return {"kind": kind, "rows": _spread(rng, 1, max(1, most if kind == "product" else most // 3)),
                "inner": inner, "outer": outer, "dtype": dtype, "bias": rng.random() < 0.5}
    count = _spread(rng, 1, 200)
    return {"kind": kind, "count": count, "total": max(count, _spread(rng, 100, 60000000)), "dtype": dtype,
            "bits": rng.choice([8, 32]), "taken": rng.randrange(0, 3000)}


# --------------------------------------------------------------------------------------------- inputs
def _features(gen, rows, width, dtype):
    """Activations: every feature has a spread of its own, as hidden units have."""
    spread = torch.exp(0.5 * torch.randn(width, generator=gen, device="cuda"))
    return (torch.randn(rows, width, generator=gen, device="cuda") * spread).to(DTYPES[dtype])


def _sizes(case):
    """``count`` tensor sizes that sum to ``total``: pairs of a matrix and its much shorter vector."""
    weights = [(1.0 + (i * 7) % 5) * (1.0 if i % 2 == 0 else 0.002) for i in range(case["count"])]
    sizes = [max(1, int(case["total"] * w / sum(weights))) for w in weights]
    sizes[0] = max(1, sizes[0] + case["total"] - sum(sizes))
    return sizes


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    if kind in ("norm_fp8", "norm_train"):
        rows, width = case["rows"], case["width"]
        state = {"case": case, "x": _features(gen, rows, width, case["dtype"]),
                 "weight": (1.0 + 0.1 * torch.randn(width, generator=gen, device="cuda")).to(DTYPES[case["dtype"]]),
                 "residual": _features(gen, rows, width, case["dtype"]) if case["residual"] else None}
        if kind == "norm_train":
            state["dy"] = (1e-3 * torch.randn(rows, width, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
            if case["residual"]:
                state["dh"] = (1e-3 * torch.randn(rows, width, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
            for k in ("x", "weight", "residual"):
                if state[k] is not None:
                    state[k].requires_grad_()
        return state
    if kind in ("product", "linear"):
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        w = torch.randn(inner, outer, generator=gen, device="cuda") * inner ** -0.5
        bias = 0.1 * torch.randn(outer, generator=gen, device="cuda") if case["bias"] else None
        x = _features(gen, rows, inner, case["dtype"])
        if kind == "linear":
            state = {"case": case, "x": x.requires_grad_(), "w": w.to(DTYPES[case["dtype"]]).requires_grad_(),
                     "bias": None if bias is None else bias.to(DTYPES[case["dtype"]]).requires_grad_()}
            state["g"] = (1e-3 * torch.randn(rows, outer, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
            return state
        # what a serving program keeps: the weight in 8 bits, stored by output; and the rows its norm has left in 8 bits
        codes, scales = _quantize_rows(x.float())
        w_codes, w_scales = _quantize_weight(w)
        return {"case": case, "codes": codes, "scales": scales, "w_codes": w_codes, "w_scales": w_scales, "bias": bias}
    # one allocation for each kind of value, the tensors at multiples of 128 in it, as a program with flat buffers has
    # them; what lies between the tensors has to stay as it is
    sizes = _sizes(case)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += _padded(n)

    def flat(spread):
        return torch.randn(at, generator=gen, device="cuda") * spread

    p = flat(0.05)
    scale = torch.exp(1.5 * torch.randn(at, generator=gen, device="cuda"))  # gradients differ in size by parameter
    g = flat(1e-3) * scale
    m = flat(3e-4) * scale
    v = (1e-6 * scale * scale) * (0.5 + torch.rand(at, generator=gen, device="cuda"))
    if case["taken"] == 0:
        m.zero_()
        v.zero_()
    state = {"case": case, "sizes": sizes, "starts": starts, "flat": {"p": p.to(DTYPES[case["dtype"]]),
                                                                     "g": g.to(DTYPES[case["dtype"]])},
             "lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "seed": 12345 + int(seed) % 1000,
             "steps": torch.full((len(sizes),), case["taken"], dtype=torch.int32, device="cuda")}
    if case["dtype"] == "bf16":
        state["flat"]["master"] = p
    if case["bits"] == 32:
        state["flat"] |= {"m": m, "v": v}
    else:
        for k, t in (("m", m), ("u", v.sqrt())):
            codes, e = _encode(t.view(-1, BLOCK))
            state["flat"] |= {k: codes.view(-1), k + "_scales": _scale_bytes(e)}
    for k, t in state["flat"].items():
        per = BLOCK if k.endswith("_scales") else 1
        state[k] = [t[a // per:a // per + -(-n // per)] for a, n in zip(starts, sizes)]
    return state


# ------------------------------------------------------------------------------------- the 8-bit format, plainly
def _exponents(x, dims):
    """Block exponents: the smallest e with max|x| * 2^-e <= 448 = 0.875 * 2^9 over the finite values."""
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dims, keepdim=True)
    mantissa, exponent = torch.frexp(top)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    return torch.where(top > 0, e, -126).clamp(-126, 120)


def _scale_bytes(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).reshape(-1)


def _power(e):
    """2^e in fp32 from its bits, -126 <= e <= 127: pow() is a rounding away from it for some e."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x):
    """Codes and exponents of fp32 [..., 128] blocks."""
    e = _exponents(x, -1)
    return (x * _power(-e)).to(torch.float8_e4m3fn), e


def _quantize_rows(x):
    """fp32 [M, K] -> codes e4m3 [M, padded K], scales e8m0 [M, padded K / 128]."""
    rows, width = x.shape
    blocks = torch.nn.functional.pad(x, (0, _padded(width) - width)).view(rows, -1, BLOCK)
    codes, e = _encode(blocks)
    return codes.view(rows, -1), _scale_bytes(e).view(rows, -1)


def _dequantize_rows(codes, scales, width):
    rows = codes.size(0)
    x = codes.float().view(rows, -1, BLOCK) * scales.float().unsqueeze(-1)
    return x.view(rows, -1)[:, :width]


def _quantize_weight(w):
    """fp32 [K, N] -> codes stored by output, e4m3 [N, padded K], scales e8m0 [K blocks, N blocks]."""
    inner, outer = w.shape
    kb, nb = _padded(inner) // BLOCK, _padded(outer) // BLOCK
    grid = torch.nn.functional.pad(w, (0, nb * BLOCK - outer, 0, kb * BLOCK - inner)).view(kb, BLOCK, nb, BLOCK)
    e = _exponents(grid, (1, 3))
    codes = (grid * _power(-e)).to(torch.float8_e4m3fn).view(kb * BLOCK, nb * BLOCK)
    return codes.t()[:outer].contiguous(), _scale_bytes(e).view(kb, nb)


def _dequantize_weight(codes, scales, inner):
    """fp32 [K, N] of codes stored by output."""
    grid = scales.float().repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    return codes.float().t()[:inner] * grid[:inner, :codes.size(0)]


def _hash(seed, tensor, taken, n):
    """20 random bits for each of n elements: what the stochastic rounding of the second moment adds."""
    key = (seed + tensor * 0x9E3779B9 + taken * 0x85EBCA6B) & 0xFFFFFFFF
    x = (torch.arange(n, device="cuda") & 0xFFFFFFFF) ^ key
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE3D) & 0xFFFFFFFF
    return x >> 12


def _encode_up_or_down(u, bits):
    """Codes and exponents of non-negative fp32 [..., 128] blocks, rounded to one of the two neighbouring codes with the
    odds of the distance; a value above zero never becomes zero."""
    e = _exponents(u, -1)
    y = u * _power(-e)
    _, exponent = torch.frexp(y)
    step = _power(torch.where(y >= 2.0 ** -6, exponent - 4, -9))
    t = torch.floor(y / step + bits.view(y.shape).float() * 2.0 ** -20) * step
    t = torch.where(y > 0, t.clamp(2.0 ** -9, 448.0), 0.0)
    return t.to(torch.float8_e4m3fn), e


# --------------------------------------------------------------------------------------------- the plain forms
def _plain_norm(x, weight, residual, relu):
    """y, h in fp32 and the row's 1 / rms: the mean square in 64 bits, because a code may hang on its last place."""
    h = x.float() if residual is None else x.float() + residual.float()
    h = h.to(x.dtype).float()                     # the stream is kept in the input's type, and its norm taken of that
    r = (h.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    y = h * r * weight.float()
    return (y.clamp_min(0.0) if relu else y), h, r


def _plain_norm_backward(h, r, weight, relu, dy, dh):
    w, gy = weight.float(), dy.float()
    if relu:
        gy = torch.where(h * r * w > 0, gy, 0.0)
    gw = gy * w
    s = (gw.double() * h.double()).mean(-1, keepdim=True).float()
    dx = r * gw - h * (r * r * r * s)
    dx = dx if dh is None else dx + dh.float()
    return dx, (gy * (h * r)).double().sum(0)


def _plain_adamw(s):
    case, b1, b2 = s["case"], s["betas"][0], s["betas"][1]
    for i, n in enumerate(s["sizes"]):
        t = case_step(s, i)
        g = s["g"][i].float()
        p = s["master"][i] if "master" in s else s["p"][i]
        if case["bits"] == 32:
            m, v = s["m"][i], s["v"][i]
        else:
            m = _decode_state(s["m"][i], s["m_scales"][i])
            v = _decode_state(s["u"][i], s["u_scales"][i]).square()
        m.mul_(b1).add_((1 - b1) * g)
        v.mul_(b2).add_((1 - b2) * (g * g))
        p.mul_(1 - s["lr"] * s["weight_decay"])
        p.sub_((s["lr"] / (1 - b1 ** t)) * m / ((v * (1 / (1 - b2 ** t))).sqrt() + s["eps"]))
        if "master" in s:
            s["p"][i].copy_(p)
        if case["bits"] == 8:
            codes, e = _encode(_blocks(m))
            s["m"][i].copy_(codes.view(-1)[:n])
            s["m_scales"][i].copy_(_scale_bytes(e))
            bits = _blocks(_hash(s["seed"], i, t, n))
            codes, e = _encode_up_or_down(_blocks(v.sqrt()), bits)
            s["u"][i].copy_(codes.view(-1)[:n])
            s["u_scales"][i].copy_(_scale_bytes(e))
    s["steps"].add_(1)


def case_step(s, i):
    """The number of the step that is being taken, counted by the program beside the tensor that the kernels read."""
    if i == 0:
        s["calls"] = s.get("calls", 0) + 1
    return s["case"]["taken"] + s["calls"]


def _blocks(x):
    return torch.nn.functional.pad(x, (0, _padded(x.numel()) - x.numel())).view(-1, BLOCK)


def _decode_state(codes, scales):
    return (_blocks(codes.float()) * scales.float().unsqueeze(-1)).view(-1)[:codes.numel()]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind in ("norm_fp8", "norm_train"):
        with torch.no_grad():
            x, w, relu = state["x"], state["weight"], state["case"]["relu"]
            y, h, r = _plain_norm(x, w, state["residual"], relu)
            if kind == "norm_fp8":
                codes, scales = _quantize_rows(y)
                return {"codes": codes, "scales": scales, "h": h.to(x.dtype)}
            dx, dw = _plain_norm_backward(h, r, w, relu, state["dy"], state.get("dh"))
            return {"y": y.to(x.dtype), "h": h.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(x.dtype)}
    if kind == "product":
        case = state["case"]
        x = _dequantize_rows(state["codes"], state["scales"], case["inner"])
        out = x @ _dequantize_weight(state["w_codes"], state["w_scales"], case["inner"])
        return (out if state["bias"] is None else out + state["bias"]).to(DTYPES[case["dtype"]])
    if kind == "linear":
        with torch.no_grad():
            x, w, g, bias = state["x"], state["w"], state["g"], state["bias"]
            xq = _dequantize_rows(*_quantize_rows(x.float()), x.size(1))
            wq = _dequantize_weight(*_quantize_weight(w.float()), x.size(1))
            out = xq @ wq
            out = out if bias is None else out + bias.float()
            gq = _dequantize_rows(*_quantize_rows(g.float()), g.size(1))
            grads = [(gq @ wq.t()).to(x.dtype), (xq.t() @ g.bfloat16().float()).to(w.dtype)]
            if bias is not None:
                grads.append(g.double().sum(0).to(bias.dtype))
            return {"out": out.to(x.dtype), "grads": grads}
    _plain_adamw(state)
    return {**state["flat"], "steps": state["steps"]}


def _run_own(state, kind):
    from gnn_benchmark_amd import fp8, norm, optim

    if kind == "norm_fp8":
        rows, h = norm.rms_norm_fp8(state["x"], state["weight"], EPS, residual=state["residual"],
                                    relu=state["case"]["relu"])
        return {"codes": rows.codes, "scales": rows.scales, "h": h}
    if kind == "norm_train":
        x, w, residual = state["x"], state["weight"], state["residual"]
        y, h = norm.rms_norm(x, w, EPS, residual=residual, relu=state["case"]["relu"])
        if residual is None:
            dx, dw = torch.autograd.grad((y,), (x, w), (state["dy"],))
        else:
            dx, dw, _ = torch.autograd.grad((y, h), (x, w, residual), (state["dy"], state["dh"]))
        return {"y": y, "h": h, "dx": dx, "dw": dw}
    if kind == "product":
        case = state["case"]
        rows = fp8.QuantizedRows(state["codes"], state["scales"], case["inner"])
        weight = fp8.QuantizedWeight(case["inner"], case["outer"], state["w_codes"], state["w_scales"])
        return fp8.product(rows, weight, state["bias"], out_dtype=DTYPES[case["dtype"]])
    if kind == "linear":
        x, w, bias = state["x"], state["w"], state["bias"]
        out = fp8.linear(x, w, bias)
        wanted = (x, w) if bias is None else (x, w, bias)
        return {"out": out, "grads": list(torch.autograd.grad((out,), wanted, (state["g"],)))}
    eight = state["case"]["bits"] == 8
    optim.adamw_step(state["p"], state["g"], state["m"], state["u"] if eight else state["v"], state["steps"],
                     lr=state["lr"], betas=state["betas"], eps=state["eps"], weight_decay=state["weight_decay"],
                     masters=state.get("master"), exp_avg_scales=state["m_scales"] if eight else None,
                     exp_avg_sq_scales=state["u_scales"] if eight else None, seed=state["seed"])
    return {**state["flat"], "steps": state["steps"]}


# --------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind in ("norm_fp8", "norm_train"):
        n, streams = case["rows"] * case["width"], 2 if case["residual"] else 1
        if kind == "norm_fp8":
            return {"bytes": n * size * (streams + 1) + case["rows"] * _padded(case["width"]) * (1 + 1 / BLOCK)
                    + case["width"] * size, "flops": 8 * n}
        # forward: x (+ residual) read, y written, h written where it is not x itself; backward: dy, h (+ dh) read, dx written
        return {"bytes": n * size * (streams + 1 + (streams - 1) + 3 + (streams - 1)) + 3 * case["width"] * size,
                "flops": 16 * n}
    if kind in ("product", "linear"):
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        if kind == "product":
            return {"bytes": rows * _padded(inner) + outer * _padded(inner) + rows * outer * size,
                    "flops": 2 * rows * inner * outer}
        return {"bytes": size * (2 * rows * inner + 2 * rows * outer + 2 * inner * outer),
                "flops": 6 * rows * inner * outer}
    states = 16 if case["bits"] == 32 else 4 * (1 + 1 / BLOCK)
    params = 8 if case["dtype"] == "fp32" else 10  # 16 bits: the master read and written, the parameter written
    return {"bytes": case["total"] * (params + size + states), "flops": 14 * case["total"]}


# ------------------------------------------------------------------------- the definitions in 64 bits, written apart
def _exact_e4m3(y):
    """The e4m3 value nearest to y (ties to the even code), |y| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_block_scale(top):
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
    e = torch.where(top * torch.exp2(-e) > 448.0, e + 1, e)
    e = torch.where(top * torch.exp2(1 - e) <= 448.0, e - 1, e)
    return torch.exp2(e.clamp(-126, 120))


def _exact_rows(x):
    """(code values [M, padded K], scales [M, blocks]) of fp64 rows."""
    rows, width = x.shape
    full = torch.zeros(rows, _padded(width), dtype=torch.float64, device=x.device)
    full[:, :width] = x
    full = full.view(rows, -1, BLOCK)
    scale = _exact_block_scale(full.abs().amax(2))
    return _exact_e4m3(full / scale.unsqueeze(2)).view(rows, -1), scale


def _exact_weight(w):
    """fp64 values that the 8-bit form of w [K, N] stands for."""
    out = torch.empty_like(w)
    for k in range(0, w.size(0), BLOCK):
        rows = w[k:k + BLOCK]
        pad = torch.nn.functional.pad(rows, (0, _padded(w.size(1)) - w.size(1))).view(rows.size(0), -1, BLOCK)
        scale = _exact_block_scale(pad.abs().amax((0, 2))).view(1, -1, 1)
        out[k:k + BLOCK] = (_exact_e4m3(pad / scale) * scale).view(rows.size(0), -1)[:, :w.size(1)]
    return out


def _exact_values(codes, scales, width):
    return (codes.view(codes.size(0), -1, BLOCK) * scales.unsqueeze(2)).reshape(codes.size(0), -1)[:, :width]


def _exact_random(seed, tensor, step, n):
    """The 20 bits of each element, in Python's whole numbers' arithmetic modulo 2^32 kept in two halves."""
    def times(x, c):
        low, high = x & 0xFFFF, x >> 16
        return (low * c + ((high * c & 0xFFFF) << 16)) & 0xFFFFFFFF

    x = torch.arange(n, device="cuda") % 2 ** 32 ^ ((seed + 0x9E3779B9 * tensor + 0x85EBCA6B * step) % 2 ** 32)
    x = times(x, 0x7FEB352D)
    x = times(x ^ x >> 15, 0x846CA68B)
    x = times(x ^ x >> 13, 0xC2B2AE3D)
    return (x >> 12).double() / 2 ** 20


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind in ("norm_fp8", "norm_train"):
            # the residual stream is a value of the input's type: its rounding belongs to the definition
            h = s["x"].double()
            if s["residual"] is not None:
                h = (h + s["residual"].double()).to(s["x"].dtype).double()
            w, n = s["weight"].double(), case["width"]
            rms = torch.sqrt((h * h).sum(1, keepdim=True) / n + EPS)
            z = h / rms
            y = z * w
            on = (y > 0) if case["relu"] else torch.ones_like(y, dtype=torch.bool)
            y = torch.where(on, y, torch.zeros_like(y))
            if kind == "norm_fp8":
                codes, scales = _exact_rows(y)
                return {"codes": codes, "scales": scales, "h": h}
            g = torch.where(on, s["dy"].double(), torch.zeros_like(y))
            gz = g * w
            dx = (gz - z * (gz * z).sum(1, keepdim=True) / n) / rms
            if s.get("dh") is not None:
                dx += s["dh"].double()
            return {"y": y, "h": h, "dx": dx, "dw": (g * z).sum(0)}
        if kind == "product":
            x = _exact_values(s["codes"].double(), s["scales"].double(), case["inner"])
            w = s["w_codes"].double()[:, :case["inner"]].t().contiguous()
            for i in range(s["w_scales"].size(0)):
                for j in range(s["w_scales"].size(1)):
                    w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= s["w_scales"][i, j].double()
            out = torch.mm(x, w)
            return out if s["bias"] is None else out + s["bias"].double()
        if kind == "linear":
            x = _exact_values(*_exact_rows(s["x"].double()), case["inner"])
            w = _exact_weight(s["w"].double())
            g = s["g"].double()
            out = torch.mm(x, w)
            grads = [torch.mm(_exact_values(*_exact_rows(g), case["outer"]), w.t().contiguous()),
                     torch.mm(x.t().contiguous(), s["g"].bfloat16().double())]
            if s["bias"] is not None:
                out += s["bias"].double()
                grads.append(g.sum(0))
            return {"out": out, "grads": grads}
        return _exact_adamw(case, s)


def _exact_adamw(case, s):
    step, (b1, b2) = case["taken"] + 1, s["betas"]
    out = {k: t.double() for k, t in s["flat"].items()}
    for i, (n, a) in enumerate(zip(s["sizes"], s["starts"])):
        at = slice(a, a + n)
        blocks = slice(a // BLOCK, a // BLOCK + _padded(n) // BLOCK)
        g = out["g"][at]
        p = out["master" if "master" in out else "p"][at]
        if case["bits"] == 32:
            m, v = out["m"][at], out["v"][at]
        else:
            m, u = (out[k][at] * out[k + "_scales"][blocks].repeat_interleave(BLOCK)[:n] for k in ("m", "u"))
            v = u ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        p = p - s["lr"] * (s["weight_decay"] * p + m / (1 - b1 ** step) / ((v / (1 - b2 ** step)) ** 0.5 + s["eps"]))
        out["p"][at] = p
        if "master" in out:
            out["master"][at] = p
        if case["bits"] == 32:
            out["m"][at], out["v"][at] = m, v
            continue
        codes, scales = _exact_rows(torch.nn.functional.pad(m, (0, _padded(n) - n)).view(-1, BLOCK))
        out["m"][at], out["m_scales"][blocks] = codes.view(-1)[:n], scales.view(-1)
        u = torch.nn.functional.pad(v.sqrt(), (0, _padded(n) - n)).view(-1, BLOCK)
        scale = _exact_block_scale(u.amax(1, keepdim=True))
        y = (u / scale).view(-1)[:n]
        gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
        y = torch.where(y > 0, (torch.floor(y / gap + _exact_random(s["seed"], i, step, n)) * gap).clamp(2.0 ** -9, 448), 0)
        out["u"][at], out["u_scales"][blocks] = y, scale.view(-1)
    return {**out, "steps": None}
