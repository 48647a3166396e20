"""OptimizerPair where PyTorch expects an optimiser: schedulers, closures, hooks,
copies; Muon's groups (CPU)."""

import copy
import pickle

import pytest
import torch

import llattn_b200
from llattn_b200.optim import OptimizerPair


def pair():
    a, b, c = (torch.nn.Parameter(torch.full(s, float(i + 1))) for i, s in enumerate(((3,), (2, 2), (4,))))
    return OptimizerPair(torch.optim.SGD([{"params": [a], "lr": 0.5}, {"params": [b]}], lr=0.1, momentum=0.9),
                         torch.optim.AdamW([c], lr=0.2)), (a, b, c)


def fill(ps, v=1.0):
    for p in ps:
        p.grad = torch.full_like(p, v)


def test_learning_rate_schedulers_take_it():
    opt, ps = pair()
    assert isinstance(opt, torch.optim.Optimizer)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 1 / (1 + step))
    for step in range(3):
        assert [g["lr"] for g in opt.param_groups] == pytest.approx([0.5 / (1 + step), 0.1 / (1 + step), 0.2 / (1 + step)])
        before = ps[0].detach().clone()
        fill(ps, 1.0 if step == 0 else 0.0)
        opt.step()
        if step == 0:
            assert torch.equal(before - ps[0].detach(), torch.full((3,), 0.5))
        sched.step()
    assert [g["lr"] for o in opt.optimizers for g in o.param_groups] == [g["lr"] for g in opt.param_groups]
    # loaded, the groups are the optimisers' own still
    opt.load_state_dict(opt.state_dict())
    opt.param_groups[2]["lr"] = 7.0
    assert opt.optimizers[1].param_groups[0]["lr"] == 7.0
    assert torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1.0, total_steps=4, cycle_momentum=False).get_last_lr()


def test_closure_hooks_and_state():
    opt, ps = pair()
    calls = []
    opt.register_step_pre_hook(lambda o, args, kw: calls.append("pre"))
    opt.register_step_post_hook(lambda o, args, kw: calls.append("post"))

    def closure():
        assert torch.is_grad_enabled()
        calls.append("closure")
        opt.zero_grad()
        loss = sum(p.square().sum() for p in ps)
        loss.backward()
        return loss

    with torch.no_grad():
        loss = opt.step(closure)
    assert loss.item() == 3 * 1 + 4 * 4 + 4 * 9 and calls == ["pre", "closure", "post"]
    assert all(p in opt.state and opt.state[p] for p in ps)
    assert opt.step() is None


def test_copies_and_pickles():
    opt, ps = pair()
    fill(ps)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert len(other.optimizers) == 2 and len(other.param_groups) == 3
        mine = [p for g in other.param_groups for p in g["params"]]
        fill(mine)
        other.step()
        fill(ps)
        snap, state = [p.detach().clone() for p in ps], copy.deepcopy(opt.state_dict())
        opt.step()
        for a, b in zip(ps, mine):
            assert torch.equal(a, b)
        with torch.no_grad():
            for p, s in zip(ps, snap):
                p.copy_(s)
        opt.load_state_dict(state)


def test_groups_are_added_to_one_of_the_two():
    opt, _ = pair()
    p = torch.nn.Parameter(torch.zeros(2))
    with pytest.raises(RuntimeError, match="one of its optimizers"):
        opt.add_param_group({"params": [p]})
    opt.optimizers[0].add_param_group({"params": [p], "lr": 3.0})
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.1, 3.0, 0.2]


def test_muon_takes_matrices_only_whenever_they_come():
    m = llattn_b200.Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError, match="matrices"):
        m.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(m.param_groups) == 1
