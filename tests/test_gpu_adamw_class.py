"""The optimizer class when a program changes what the optimizer holds in public: its states, its parameter lists, its
groups, its step counts.  Beside torch.optim.AdamW in 64 bits with the same gradients and the same changes.

Tolerance: each step adds its own error, 24 half steps of fp32 of a rate's size (the update stays below 10 lr here) and 3 of
the parameter, as derived for a single step in test_gpu_adamw.py."""
import pytest
import torch

import fp8_oracle as o
from gnn_benchmark_amd import optim

pytestmark = pytest.mark.gpu
H = o.HALF32
LR = 1e-2


class Pair:
    """An optimizer of this package and torch's, over equal parameters in two groups."""

    def __init__(self, seed, shapes=((40, 30), (30,), (300,), (7, 5)), bits=32):
        self.gen = torch.Generator().manual_seed(seed)
        start = [torch.randn(s, generator=self.gen) for s in shapes]
        self.ours = [torch.nn.Parameter(t.cuda()) for t in start]
        self.theirs = [torch.nn.Parameter(t.double().cuda()) for t in start]
        groups = lambda ps: [dict(params=ps[:2]), dict(params=ps[2:], lr=2 * LR, weight_decay=0.1)]  # noqa: E731
        self.a = optim.AdamW(groups(self.ours), lr=LR, state_bits=bits)
        self.b = torch.optim.AdamW(groups(self.theirs), lr=LR)
        self.taken = 0

    def step(self, count=1, opts=None):
        for _ in range(count):
            for p, q in zip(self.ours, self.theirs):
                g = torch.randn(p.shape, generator=self.gen)
                p.grad, q.grad = g.cuda(), g.double().cuda()
            self.a.step()
            self.b.step()
            self.taken += 1

    def check(self, what):
        for i, (p, q) in enumerate(zip(self.ours, self.theirs)):
            q = q.detach().cpu()
            bound = self.taken * (3 * H * (q.abs() + 10 * self.taken * 2 * LR) + 24 * H * 10 * 2 * LR)
            o.assert_within(p, q, bound, f"{what}, parameter {i}")


@pytest.mark.parametrize("how", ["clear", "another dict", "one entry"])
def test_a_state_that_was_taken_away_starts_again(how):
    pair = Pair(1)
    pair.step(50)
    if how == "clear":
        for opt in (pair.a, pair.b):
            opt.state.clear()
    elif how == "another dict":
        for opt in (pair.a, pair.b):
            opt.state = type(opt.state)(dict)
    else:
        del pair.a.state[pair.ours[2]]
        del pair.b.state[pair.theirs[2]]
    pair.step(3)
    pair.check(how)
    steps = [int(pair.a.state[p]["step"]) for p in pair.ours]
    assert steps == [int(pair.b.state[q]["step"]) for q in pair.theirs]


def test_a_replaced_parameter_is_the_one_that_moves():
    pair = Pair(2)
    pair.step(5)
    old = pair.ours[1]
    before = old.detach().clone()
    start = torch.randn(30, generator=pair.gen)
    pair.ours[1], pair.theirs[1] = torch.nn.Parameter(start.cuda()), torch.nn.Parameter(start.double().cuda())
    pair.a.param_groups[0]["params"][1] = pair.ours[1]
    pair.b.param_groups[0]["params"][1] = pair.theirs[1]
    pair.step(4)
    pair.check("replaced")
    assert torch.equal(old, before)
    assert int(pair.a.state[pair.ours[1]]["step"]) == 4 and int(pair.a.state[pair.ours[0]]["step"]) == 9


def test_parameters_in_another_order_and_a_group_taken_out():
    pair = Pair(3)
    pair.step(5)
    for opt in (pair.a, pair.b):
        opt.param_groups[0]["params"].reverse()
    pair.step(2)
    pair.check("reversed")
    for opt in (pair.a, pair.b):
        del opt.param_groups[0]
    pair.step(3)
    pair.check("a group less")
    assert int(pair.a.state[pair.ours[2]]["step"]) == 10 and int(pair.a.state[pair.ours[0]]["step"]) == 7


@pytest.mark.parametrize("form", ["tensor", "number", "in place"])
def test_a_step_count_that_was_set_is_read(form):
    pair = Pair(4)
    pair.step(5)
    for i in (0, 2):
        pair.b.state[pair.theirs[i]]["step"] = torch.tensor(100.0)
        state = pair.a.state[pair.ours[i]]
        if form == "in place":
            state["step"].fill_(100)
        else:
            state["step"] = torch.tensor(100.0) if form == "tensor" else 100
    pair.step(3)
    pair.check(form)
    assert [int(pair.a.state[p]["step"]) for p in pair.ours] == [103, 8, 103, 8]


def test_a_parameter_and_a_group_added_between_steps():
    pair = Pair(5)
    pair.step(4)
    more = torch.randn(11, 13, generator=pair.gen)
    pair.ours.append(torch.nn.Parameter(more.cuda()))
    pair.theirs.append(torch.nn.Parameter(more.double().cuda()))
    pair.a.add_param_group(dict(params=[pair.ours[-1]]))
    pair.b.add_param_group(dict(params=[pair.theirs[-1]]))
    pair.step(4)
    more = torch.randn(70, generator=pair.gen)
    pair.ours.append(torch.nn.Parameter(more.cuda()))
    pair.theirs.append(torch.nn.Parameter(more.double().cuda()))
    pair.a.param_groups[0]["params"].append(pair.ours[-1])
    pair.b.param_groups[0]["params"].append(pair.theirs[-1])
    pair.step(4)
    pair.check("added")
    assert [int(pair.a.state[p]["step"]) for p in pair.ours] == [12, 12, 12, 12, 8, 4]


def test_what_changed_cannot_be_captured_before_a_step():
    """A capture needs the step counts' array: a change behind it is refused there, and a step mends it."""
    pair = Pair(6)
    pair.step(2)
    pair.a.state.clear()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda").add_(1)
        with pytest.raises(RuntimeError, match="before capturing"):
            pair.a.step()
    pair.b.state.clear()
    pair.step(2)
    pair.check("after the refusal")


def test_a_captured_step_goes_on_behind_a_count_that_was_set():
    """The counts' array stays in its place, so a graph captured before raises the count that was set."""
    pair = Pair(7)
    for p in pair.ours:
        p.grad = torch.zeros_like(p)
    pair.step(2)
    grads = [torch.randn(p.shape, generator=pair.gen) for p in pair.ours]
    for p, q, g in zip(pair.ours, pair.theirs, grads):
        p.grad, q.grad = g.cuda(), g.double().cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pair.a.step()
    for i in range(len(pair.ours)):
        pair.a.state[pair.ours[i]]["step"] = 40
        pair.b.state[pair.theirs[i]]["step"] = torch.tensor(40.0)
    pair.a.step()                                           # finds the counts
    pair.b.step()
    for _ in range(2):
        graph.replay()
        float(torch.randn(64, device="cuda").sum())
        pair.b.step()
    pair.taken += 3
    pair.check("replayed")
    assert [int(pair.a.state[p]["step"]) for p in pair.ours] == [43] * 4


def test_counts_that_a_graph_raises_outlive_a_change():
    """A parameter that joins makes new arrays of step counts; a graph captured before goes on raising the old one, whose
    memory belongs to nobody else."""
    pair = Pair(8)
    pair.step(2)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pair.a.step()
    counts = [int(pair.a.state[p]["step"]) for p in pair.ours]
    more = torch.nn.Parameter(torch.zeros(50, device="cuda"))
    pair.a.param_groups[0]["params"].append(more)
    more.grad = torch.ones_like(more)
    pair.a.step()
    assert [int(pair.a.state[p]["step"]) for p in pair.ours] == [c + 1 for c in counts]
    torch.cuda.synchronize()
    small = [torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2000)]     # takes what is free of that size
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert int(torch.stack(small).abs().sum()) == 0
    assert [int(pair.a.state[p]["step"]) for p in pair.ours[:2]] == [c + 1 for c in counts[:2]]
