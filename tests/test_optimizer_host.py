"""CPU-only: optimizer states that another rule wrote are refused, and a refusal leaves the optimizer as it was."""
import copy

import pytest
import torch

from gnn_benchmark_amd import optim


def saved(cls, steps=0, **settings):
    p = torch.nn.Parameter(torch.ones(6))
    opt = cls([p], lr=0.25, **settings)
    for _ in range(steps):
        p.grad = torch.ones(6)
        opt.step()
    return opt.state_dict()


OTHER_RULES = [(torch.optim.AdamW, dict(maximize=True)), (torch.optim.Adam, dict(maximize=True)),
               (torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.Adam, dict(amsgrad=True)),
               (torch.optim.Adam, dict(weight_decay=0.1)), (torch.optim.NAdam, {}), (torch.optim.RAdam, {}),
               (torch.optim.SGD, {})]


@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("cls,settings", OTHER_RULES)
def test_states_of_another_rule_are_refused(cls, settings, steps):
    opt = optim.AdamW([torch.nn.Parameter(torch.ones(6))], lr=0.5)
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(RuntimeError, match="another rule"):
        opt.load_state_dict(saved(cls, steps, **settings))
    assert opt.state_dict() == before


def test_states_of_the_same_rule_are_taken_without_torchs_switches():
    for cls, settings in ((torch.optim.AdamW, {}), (torch.optim.Adam, {}), (torch.optim.AdamW, dict(foreach=True))):
        opt = optim.AdamW([torch.nn.Parameter(torch.ones(6))], lr=0.5, state_bits=8, seed=4)
        opt.load_state_dict(saved(cls, **settings))
        group = opt.param_groups[0]
        assert group["lr"] == 0.25 and group["state_bits"] == 8 and group["seed"] == 4
        assert not {"maximize", "amsgrad", "decoupled_weight_decay"} & set(group)
    scheduled = optim.AdamW([torch.nn.Parameter(torch.ones(6))], lr=0.5)
    torch.optim.lr_scheduler.StepLR(scheduled, 1)
    opt = optim.AdamW([torch.nn.Parameter(torch.ones(6))])
    opt.load_state_dict(scheduled.state_dict())
    assert opt.param_groups[0]["initial_lr"] == 0.5


def test_a_state_that_does_not_fit_changes_nothing():
    a, b = (torch.nn.Parameter(torch.ones(6)) for _ in range(2))
    opt = optim.AdamW([a, b], lr=0.5)
    opt.state[a] = {"exp_avg": torch.ones(6), "exp_avg_sq": torch.ones(6), "step": torch.tensor(3)}
    state = opt.state[a]
    with pytest.raises(RuntimeError):                      # (two parameters on the CPU, whose states it does not make)
        two = [torch.nn.Parameter(torch.ones(6)) for _ in range(2)]
        theirs = torch.optim.AdamW(two, lr=0.25)
        for p in two:
            p.grad = torch.ones(6)
        theirs.step()
        opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and opt.state[a] is state and opt.param_groups[0]["params"][0] is a
    with pytest.raises(ValueError):
        opt.load_state_dict(saved(torch.optim.AdamW))
    assert opt.param_groups[0]["lr"] == 0.5 and opt.state[a] is state
