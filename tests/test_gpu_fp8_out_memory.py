"""The array that a product writes into may lie beside its operands, between their columns too, but not over them."""
import pytest
import torch

from gnn_benchmark_amd import fp8

pytestmark = pytest.mark.gpu


def test_out_over_an_operand_is_refused():
    m, k, n = 40, 128, 32
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    x, w = torch.randn(m, k, device="cuda"), torch.randn(k, n, device="cuda")
    q, qw = fp8.quantize_rows(x), fp8.quantize_weight(w)
    bias = torch.randn(n, device="cuda")
    want = fp8.product(q, qw, bias)

    def at(offset, t):                                       # t's bytes at a place of `raw`
        place = raw[offset:offset + t.numel() * t.element_size()]
        place.copy_(t.contiguous().view(torch.uint8).view(-1))
        return place.view(t.dtype).view(t.shape)

    operands = {"codes": q.codes, "scales": q.scales, "weight": qw.codes, "weight's scales": qw.scales, "bias": bias}
    size = 4 * m * n
    for name, t in operands.items():
        nbytes = t.numel() * t.element_size()
        moved = at(16384, t)
        x8 = fp8.QuantizedRows(moved if name == "codes" else q.codes, moved if name == "scales" else q.scales, k)
        w8 = fp8.QuantizedWeight(k, n, moved if name == "weight" else qw.codes, moved if name == "weight's scales" else qw.scales)
        b = moved if name == "bias" else bias
        before = raw.clone()
        last = 16384 + (nbytes - 1) // 4 * 4                 # the word with the operand's last byte
        for start in (16384, last, 16384 - size + 4):
            with pytest.raises(RuntimeError, match="shares memory"):
                print("refusal", name, start, flush=True)
                fp8.product(x8, w8, b, out=raw[start:start + size].view(torch.float32).view(m, n))
        wide = raw[16384 - 256:16384 - 256 + 4 * m * (n + 40)].view(torch.float32).view(m, n + 40)
        with pytest.raises(RuntimeError, match="shares memory"):
            fp8.product(x8, w8, b, out=wide[:, 40:])         # (its first rows begin in front of the operand)
        assert torch.equal(raw, before)
        for start in (16384 - size, 16384 + (nbytes + 3) // 4 * 4):   # right in front, right behind
            out = raw[start:start + size].view(torch.float32).view(m, n)
            assert torch.equal(fp8.product(x8, w8, b, out=out), want), (name, start)
    wide = torch.zeros(m, n + 40, device="cuda")             # the bias between the columns of a wider array
    wide[3, n + 2:n + 2 + n] = bias
    assert torch.equal(fp8.product(q, qw, wide[3, n + 2:n + 2 + n], out=wide[:, :n]), want)
    with pytest.raises(RuntimeError, match="shares memory"):
        fp8.product(q, qw, wide.view(-1)[3 * (n + 40) + n + 28:][:n], out=wide[:, :n])    # (reaches into the next row)
