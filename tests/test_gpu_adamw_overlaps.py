"""What an AdamW step reads may not lie where it writes: a gradient, or a learning rate on the device, that shares bytes with
a parameter, state, master, scale or step count is refused, before anything is launched.  Neighbours are not."""
import pytest
import torch

from gnn_benchmark_amd import optim

pytestmark = pytest.mark.gpu


def test_gradients_and_rates_in_written_memory_are_refused():
    n = 300
    flat = torch.ones(8 * n, device="cuda")
    p, m, v, g = (flat[i * n:(i + 1) * n] for i in range(4))
    m.zero_()
    v.zero_()
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = flat.clone()
    bad = [flat[1:n + 1], p, flat[n - 1:2 * n - 1], m, v, flat[2 * n + 7:3 * n + 7]]
    for i, grad in enumerate(bad):
        print("refusal", i, flush=True)
        with pytest.raises(RuntimeError, match="same memory"):
            optim.adamw_step([p], [grad], [m], [v], steps, lr=0.1)
    for i, rate in enumerate((p[5], m[0], v[n - 1:], steps.view(torch.float32))):
        print("rate", i, flush=True)
        with pytest.raises(RuntimeError, match="same memory"):
            optim.adamw_step([p], [g], [m], [v], steps, lr=rate)
    master = torch.ones(n, device="cuda")
    with pytest.raises(RuntimeError, match="same memory"):
        optim.adamw_step([p.bfloat16()], [master], [m], [v], steps, lr=0.1, masters=[master])
    codes = [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    raw = torch.ones(n * 2, dtype=torch.uint8, device="cuda")
    scales = [raw[i:i + 3].view(torch.float8_e8m0fnu) for i in (0, 64)]
    with pytest.raises(RuntimeError, match="same memory"):
        optim.adamw_step([p], [raw.view(torch.bfloat16)], *[[c] for c in codes], steps, lr=0.1,
                         exp_avg_scales=scales[:1], exp_avg_sq_scales=scales[1:])
    assert torch.equal(flat, before) and int(steps) == 0


def test_neighbours_are_not():
    """Gradients right in front of, between and right behind what is written, one of them for two parameters; an empty one
    inside; the learning rate in between."""
    n = 128
    flat = torch.ones(10 * n, device="cuda")
    part = [flat[i * n:(i + 1) * n] for i in range(10)]
    for i in (2, 4, 6, 8):
        part[i].zero_()
    flat[9 * n] = 0.5
    rate, empty = flat[9 * n], flat[1 * n + 5:1 * n + 5]
    steps = torch.zeros(3, dtype=torch.int32, device="cuda")
    states = [part[2], part[4], torch.zeros(0, device="cuda")], [part[6], part[8], torch.zeros(0, device="cuda")]
    optim.adamw_step([part[1], part[7], empty[:0]], [part[0], part[0], empty], *states, steps, lr=rate, weight_decay=0.0)
    assert steps.tolist() == [1, 1, 1] and torch.equal(part[1], part[7])
    # first step of a gradient of ones: the update is lr / (1 + eps), to 24 half steps of it
    assert float((part[1] - 0.5).abs().max()) <= 24 * 2.0 ** -24 + 1e-8
    for i in (0, 3, 5):
        assert bool((part[i] == 1).all())
    optim.adamw_step([part[1]], [part[3]], [part[2]], [part[6]], steps[:1], lr=0.1)
    assert bool((part[3] == 1).all())
