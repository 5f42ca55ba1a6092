"""Column sums of many rows (the bias's gradient): how much the rounding of long fp32 chains may cost.

Equal values are the worst case: the roundings of neighbouring additions go the same way.  A thread adds its rows eight at a
time, a stage of 32 rows in each of `stages` additions: the i-th rounds a sum of i eights by half a step at most, all together
(stages + 1) / 2 half steps of the whole; the eights themselves 3, the block's eight parts 4, the store 1; the slices' results
are added in 64 bits."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [7, 8, 12])
@pytest.mark.parametrize("rows", [600_001, 2_400_000])
def test_long_columns_of_equal_values(rows, n, dtype):
    q = fp8.quantize_rows(torch.zeros(rows, 8, device="cuda"))
    values = torch.tensor([4 / 3, 5 / 3, 1.1, 1.9, 1.7, 1.3, 7 / 3, -4 / 3, -1.9, 1.57, 1.01, 1.99])[:n].to(dtype)
    g = values.cuda().expand(rows, n).contiguous()
    dw, db = fp8.weight_gradient(q, g, True)
    assert bool((dw == 0).all())
    want = rows * values.double()
    stages = -(-(-(-rows // 256)) // 32) + 1                # 256 slices: one tile of the result, as many as there are compute units
    o.assert_within(db, want, ((stages + 1) / 2 + 8) * o.HALF32 * want.abs(), "column sums")
