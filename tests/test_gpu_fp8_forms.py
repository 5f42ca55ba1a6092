"""Products on both sides of the borders between the product's kernels: whole numbers, so that every kernel is exact."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import fp8
from test_gpu_fp8 import as_quantized_rows, whole_rows, whole_weight

pytestmark = pytest.mark.gpu

SHAPES = [(64, 4096, 4100), (65, 4096, 4096), (128, 4096, 4096), (129, 4096, 4096), (2048, 512, 256), (2049, 512, 256),
          (4160, 300, 128), (4160, 300, 129), (4097, 512, 100), (19999, 256, 172), (20000, 256, 172), (20001, 130, 260),
          (4096, 4096, 4096), (3900, 4000, 4000), (3900, 3968, 4000), (5000, 4097, 1030), (59001, 4096, 200), (66000, 100, 1)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_beside_the_borders(m, k, n):
    gen = torch.Generator().manual_seed(m + k + n)
    codes, e, x = whole_rows(m, k, gen, scale_from=0)
    w, values = whole_weight(k, n, gen)
    q, want = as_quantized_rows(codes, e, k), x.cuda() @ values.cuda()
    bias = torch.randint(-8, 9, (n,), generator=gen).float().cuda()
    assert torch.equal(fp8.product(q, w).double(), want)
    want = (want + bias.double()).float()
    assert torch.equal(fp8.product(q, w, bias), want)
    assert torch.equal(fp8.product(q, w, bias, out_dtype=torch.bfloat16), want.bfloat16())
    assert o.same(fp8.product(q, w, bias)[-1:], want[-1:])
