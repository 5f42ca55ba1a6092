"""Keep masks of the model with RMS norms: what the LayerNorm model takes and refuses, this one does too."""
import pytest
import torch

from gnn_benchmark_amd import sage
from test_gpu_sage_fp8 import partition

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("gemm", ["fp32", "fp8"])
def test_masks_of_bytes_and_refusals(gemm):
    """Any byte but zero keeps; a mask of another shape or type is refused, not broadcast or read as something else."""
    n, hidden = 1000, 64
    graph, _ = partition(n, 2 * hidden, True)
    torch.manual_seed(0)
    model = sage.DistSAGE(32, hidden, 16, num_layers=2, dropout=0.5, is_pre_delay=True, gemm=gemm, norm="rms").to(DEV).train()
    x = torch.randn(n, 32, device=DEV)
    keep = torch.rand(n, hidden, device=DEV) < 0.5

    def run(mask):
        model.zero_grad()
        out = model(graph, x, [mask])
        out.square().mean().backward()
        return [out.detach()] + [p.grad.clone() for p in model.parameters()]

    want = run(keep)
    for value in (1, 2, 255):
        got = run(keep.to(torch.uint8) * value)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), value
    spread = torch.where(keep, torch.randint(1, 256, keep.shape, device=DEV), 0).to(torch.uint8)
    assert all(torch.equal(a, b) for a, b in zip(run(spread), want))
    for bad in (keep.float(), keep.to(torch.int32), keep[:1], keep[:, :1], keep[:-1], keep.half()):
        with pytest.raises(RuntimeError, match="keep must be"):
            run(bad)
