"""CPU-only: the training operators' header and binding agree, what they refuse is refused before any GPU work, and the
64-bit formulas that their GPU tests compare with have the gradients that differences give."""
import ctypes
import os
import re

import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import _lib, fp8, norm, optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _text():
    with open(os.path.join(ROOT, "include", "gnn_train.h")) as f:
        return re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)


def test_header_and_binding_agree():
    declared = sorted(set(re.findall(r"\b(gnnagg_[a-z0-9_]+)\s*\(", _text())))
    assert declared == sorted(_lib.TRAIN_EXPORTS)
    assert not set(declared) & set(_lib.EXPORTS)
    if os.path.exists(_lib.LIB_PATH):
        cdll = ctypes.CDLL(_lib.LIB_PATH)
        for name in declared:
            assert hasattr(cdll, name), name
        assert _lib.lib().gnnagg_train_abi_version() == _lib.TRAIN_ABI_VERSION


# GNNAGG_TRAIN_ABI_VERSION -> digest of the prototypes and the record it stands for
TRAIN_ABI_DIGESTS = {1: "5fc735e6e35e1dd2"}


def test_a_changed_prototype_needs_a_new_version():
    import hashlib

    text = _text()
    version = int(re.search(r"#define GNNAGG_TRAIN_ABI_VERSION (\d+)", text).group(1))
    assert version == _lib.TRAIN_ABI_VERSION
    body = re.sub(r"\s+", " ", text[text.index("int gnnagg_train_abi_version"):])
    assert hashlib.sha256(body.encode()).hexdigest()[:16] == TRAIN_ABI_DIGESTS[version], (
        "a prototype changed: raise GNNAGG_TRAIN_ABI_VERSION / _lib.TRAIN_ABI_VERSION and record the digest "
        + hashlib.sha256(body.encode()).hexdigest()[:16])


def _library():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libgnnagg.so not built yet")
    return _lib.lib()


def test_entry_points_refuse_bad_arguments_before_any_launch():
    L = _library()
    p = 4096  # a stand-in for a device address: nothing below gets as far as using it
    bad, no = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
    norm_args = lambda **k: [k.get("x", p), k.get("xs", 64), k.get("res"), 64, p, k.get("wd", 0), 1e-6, 0, k.get("h"), 64,  # noqa: E731
                             k.get("y", p), k.get("ys", 64), k.get("rows", 4), k.get("width", 64), k.get("dtype", 0), None]
    assert L.gnnagg_rms_norm(*norm_args(rows=0)) == _lib.OK
    assert L.gnnagg_rms_norm(*norm_args(rows=-1)) == bad
    assert L.gnnagg_rms_norm(*norm_args(width=0)) == no
    assert L.gnnagg_rms_norm(*norm_args(width=16385, xs=16385, ys=16385)) == no
    assert b"16384" in L.gnnagg_last_error()
    assert L.gnnagg_rms_norm(*norm_args(x=None)) == bad
    assert L.gnnagg_rms_norm(*norm_args(y=None)) == bad
    assert L.gnnagg_rms_norm(*norm_args(res=p)) == bad         # a residual without a place for h
    assert L.gnnagg_rms_norm(*norm_args(h=p)) == bad
    assert L.gnnagg_rms_norm(*norm_args(xs=63)) == bad
    assert L.gnnagg_rms_norm(*norm_args(ys=63)) == bad
    assert L.gnnagg_rms_norm(*norm_args(dtype=2)) == bad
    assert L.gnnagg_rms_norm(*norm_args(wd=1)) == bad          # bf16 weight with fp32 rows
    assert L.gnnagg_rms_norm_fp8(p, 64, None, 0, p, 0, 1e-6, 0, None, 0, p + 1, p, 4, 64, 0, None) == bad
    need = L.gnnagg_rms_norm_backward_workspace_bytes(4, 64)
    assert need > 0 and L.gnnagg_rms_norm_backward_workspace_bytes(0, 64) == 0
    assert L.gnnagg_rms_norm_backward(p, 64, None, 0, p, 64, p, 0, 1e-6, 0, p, 64, p, p, need - 1, 4, 64, 0, None) == bad
    assert b"workspace" in L.gnnagg_last_error()
    assert L.gnnagg_rms_norm_backward(p, 64, None, 0, p, 64, p, 0, 1e-6, 0, p, 64, None, p, need, 4, 64, 0, None) == bad
    assert L.gnnagg_fp8_quantize_rows(p, 64, p, p, 0, 64, 0, None) == _lib.OK
    assert L.gnnagg_fp8_quantize_rows(None, 64, p, p, 4, 64, 0, None) == bad
    assert L.gnnagg_fp8_quantize_rows(p, 63, p, p, 4, 64, 0, None) == bad
    assert L.gnnagg_fp8_quantize_rows(p, 64, p + 2, p, 4, 64, 0, None) == bad
    assert L.gnnagg_fp8_quantize_weight(p, 8, None, None, p, 8, 8, 0, None) == bad
    assert L.gnnagg_fp8_quantize_weight(p, 7, p, None, p, 8, 8, 0, None) == bad
    assert L.gnnagg_fp8_product(p, p, p, p, 1, 1, None, p, 8, 0, 0, 16, 8, None) == _lib.OK
    assert L.gnnagg_fp8_product(p, p, p, p, 1, 1, None, p, 8, 0, 4, 0, 8, None) == bad
    assert L.gnnagg_fp8_product(p + 8, p, p, p, 1, 1, None, p, 8, 0, 4, 16, 8, None) == bad
    assert b"16-byte" in L.gnnagg_last_error()
    assert L.gnnagg_fp8_product(p, p, p, p, 1, 1, None, p, 7, 0, 4, 16, 8, None) == bad
    assert L.gnnagg_fp8_product(p, p, p, p, 1, 1, None, p, 8, 5, 4, 16, 8, None) == bad
    need = L.gnnagg_fp8_weight_gradient_workspace_bytes(100000, 64, 64)
    assert need > 0
    assert L.gnnagg_fp8_weight_gradient(p, p, p, 64, 0, p, None, p, need - 1, 100000, 64, 64, None) == bad
    assert L.gnnagg_fp8_weight_gradient(p, p, p, 64, 0, p, None, None, need, 100000, 64, 64, None) == bad
    assert L.gnnagg_fp8_weight_gradient(p, p, p, 63, 0, p, None, p, need, 100000, 64, 64, None) == bad
    t = (_lib.AdamwTensor * 1)()
    step = lambda **k: L.gnnagg_adamw_step(t, k.get("count", 1), k.get("steps", p), k.get("dtype", 0), 0, k.get("bits", 32),  # noqa: E731
                                           1e-3, None, k.get("b1", 0.9), 0.999, 1e-8, 0.0, 0, 0, None)
    assert step(count=0) == _lib.OK
    assert step(count=-1) == bad
    assert step(steps=None) == bad
    t[0].n = -1
    assert step() == bad
    t[0].n = 4
    assert step() == bad                                       # null pointers
    t[0].param = t[0].grad = t[0].exp_avg = t[0].exp_avg_sq = p
    assert step(bits=16) == bad
    assert step(bits=8) == bad                                 # no scales
    assert step(dtype=1) == bad                                # no master
    assert b"master" in L.gnnagg_last_error()
    assert step(b1=1.0) == bad


def test_python_entry_points_refuse_cpu_tensors_and_other_types():
    x, w = torch.ones(3, 8), torch.ones(8)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.rms_norm_fp8(x, w), lambda: fp8.quantize_rows(x),
                 lambda: fp8.quantize_weight(torch.ones(8, 8)), lambda: fp8.linear(x, torch.ones(8, 8)),
                 lambda: fp8.norm_linear(x, w, 1e-6, torch.ones(8, 8)),
                 lambda: fp8.weight_gradient(fp8.QuantizedRows.empty(3, 8, "cpu"), x),
                 lambda: fp8.product(fp8.QuantizedRows.empty(3, 8, "cpu"), fp8.QuantizedWeight(8, 8, None, x)),
                 lambda: optim.adamw_step([x], [x], [x], [x], torch.zeros(1, dtype=torch.int32), lr=0.1)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    optim.adamw_step([], [], [], [], torch.zeros(0, dtype=torch.int32), lr=0.1)  # nothing to do


def test_optimizer_refuses_bad_settings():
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    opt = optim.AdamW([p])
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        opt.step()


def test_the_oracles_format():
    """Every e4m3 value is its own nearest; scales are the smallest that hold the block; values at the borders."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    fine = codes[codes.isfinite()]
    assert o.same(o.e4m3_nearest(fine), fine)
    y = torch.linspace(-448, 448, 20001, dtype=torch.float64)
    assert o.same(o.e4m3_nearest(y.float().double()), y.float().to(torch.float8_e4m3fn))
    near = o.e4m3_nearest(y)
    assert bool(((near - y).abs() <= torch.maximum(o.STEP8 * y.abs(), torch.tensor(2.0 ** -10))).all())
    tops = torch.tensor([0.0, 448.0, 448.0000001, 1.75, 1.7500001, 3.4e38, 1e-38, 1e-45], dtype=torch.float64)
    assert o.block_exponent(tops).tolist() == [-126.0, 0.0, 1.0, -8.0, -7.0, 120.0, -126.0, -126.0]


def test_norm_gradient_formula_against_differences():
    gen = torch.Generator().manual_seed(0)
    h = torch.randn(4, 9, generator=gen, dtype=torch.float64)
    w = torch.randn(9, generator=gen, dtype=torch.float64)
    g = torch.randn(4, 9, generator=gen, dtype=torch.float64)
    for relu in (False, True):
        f = lambda h, w: (o.rms_norm(h, w, 1e-6, relu)[0] * g).sum()  # noqa: E731
        y, z, r = o.rms_norm(h, w, 1e-6, relu)
        gn = torch.where(y > 0, g, 0.0) if relu else g
        gw = gn * w
        dx, dw = (gw - z * (gw * z).mean(-1, keepdim=True)) * r, (gn * z).sum(0)
        step = 1e-5
        for i in range(4):
            for j in range(9):
                e = torch.zeros_like(h)
                e[i, j] = step
                # truncation: step^2 times a third derivative of order r^3 |g w|; cancellation: 1e-16 / step
                assert abs((f(h + e, w) - f(h - e, w)) / (2 * step) - dx[i, j]) < 1e-7
        for j in range(9):
            e = torch.zeros_like(w)
            e[j] = step
            assert abs((f(h, w + e) - f(h, w - e)) / (2 * step) - dw[j]) < 1e-7
