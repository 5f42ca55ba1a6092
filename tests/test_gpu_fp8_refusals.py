"""Calls without a gradient refuse what wants one."""
import pytest
import torch

from gnn_benchmark_amd import fp8

pytestmark = pytest.mark.gpu


def test_weight_gradient_refuses_what_wants_a_gradient():
    x = fp8.quantize_rows(torch.randn(300, 130, device="cuda"))
    g = torch.randn(300, 40, device="cuda")
    want = fp8.weight_gradient(x, g)
    leaf = g.clone().requires_grad_()
    for call in (lambda: fp8.weight_gradient(x, leaf), lambda: fp8.weight_gradient(x, leaf * 1.0, True)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        assert torch.equal(fp8.weight_gradient(x, leaf), want)
    assert torch.equal(fp8.weight_gradient(x, leaf.detach()), want)
