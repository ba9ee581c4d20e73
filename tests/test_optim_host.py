"""The AdamW optimiser's own work on the CPU, with core.adamw replaced by a record of its calls: the seeds of the calls' rounding,
parameter groups that are refused, states that are loaded."""
import copy
import pickle

import numpy as np
import pytest
import torch

from sdmchat_amd import AdamW, core

A = 2654435761   # what the library multiplies a step's number by before it is hashed


def mix(x):
    x = ((x ^ (x >> 16)) * A) & 0xffffffff
    x = ((x ^ (x >> 15)) * 3144134277) & 0xffffffff
    return x ^ (x >> 16)


@pytest.fixture
def calls(monkeypatch):
    """core.adamw's calls: (params, step, seed, lr)."""
    out = []

    def adamw(params, grads, *moments, step, seed, lr, **rest):
        if torch.is_tensor(step):
            step += 1
        out.append((params, int(step), seed & 0xffffffff, lr))
    monkeypatch.setattr(core, "adamw", adamw)
    return out


def params(*sizes):
    return [torch.nn.Parameter(torch.full((n,), float(i))) for i, n in enumerate(sizes)]


def step(opt, grads):
    for g in opt.param_groups:
        for p in g["params"]:
            p.grad = torch.ones_like(p) if any(p is q for q in grads) else None
    opt.step()


@pytest.mark.parametrize("capturable", [False, True])
def test_no_two_calls_round_alike(calls, capturable):
    """Every call's key, the hash of seed and step that its values' random bits come from, is one of its own: with two groups, a
    group without gradients for some steps, and parameters whose step counts differ."""
    ps = params(300, 200, 100, 50, 20)
    opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:4]), dict(params=ps[4:])], lr=1e-3, state_bits=8, seed=7, capturable=capturable)
    live = [ps, ps, ps[2:], ps, ps[:3], ps[:1] + ps[3:], ps[4:], ps, ps[1:], ps, ps[1:4], ps, ps]
    for grads in live:
        step(opt, grads)
    assert len(calls) > 3 * len(live) - 5 and any(c[0][0] is ps[1] for c in calls)
    keys = [mix((seed + t * A) & 0xffffffff) for _, t, seed, _ in calls]
    assert len(set(keys)) == len(keys)


def test_keys_of_far_steps_and_many_groups(calls):
    """Groups of one parameter each, over as many steps as a training run has."""
    ps = params(*[1] * 40)
    opt = AdamW([dict(params=[p]) for p in ps], lr=1e-3, state_bits=8)
    step(opt, ps)
    seeds = np.array([seed for _, _, seed, _ in calls], np.uint64)
    assert len(seeds) == len(ps)
    t = np.arange(1, 100001, dtype=np.uint64)
    keys = (seeds[:, None] + t * np.uint64(A)) & np.uint64(0xffffffff)   # the hash maps different numbers to different ones
    assert len(np.unique(keys)) == keys.size


def test_seeds_do_not_hang_on_what_else_steps(calls):
    """A group's rounding is the same whether the groups before it have gradients or not, and the first call's is the seed's."""
    ps = params(300, 200)
    opt = AdamW([dict(params=ps[:1]), dict(params=ps[1:])], lr=1e-3, state_bits=8, seed=11)
    step(opt, ps)
    step(opt, ps[1:])
    first, second, alone = calls
    assert first[2] == 11 and second[0][0] is alone[0][0] is ps[1] and second[2] == alone[2] != 11


@pytest.mark.parametrize("over", [dict(betas=(0.9, 1.5)), dict(betas=0.9), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1),
                                  dict(state_bits=4), dict(max_norm=2.0), dict(lr=torch.ones(())), dict(capturable=True)])
def test_a_refused_group_is_not_kept(calls, over):
    a, b = params(3, 4)
    opt = AdamW([a], lr=1e-3)
    with pytest.raises((ValueError, TypeError)):
        opt.add_param_group(dict(dict(params=[b]), **over))
    with pytest.raises(ValueError, match="float64"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))]))
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[a]))   # torch's own refusal
    assert [g["params"] for g in opt.param_groups] == [[a]]
    step(opt, [a, b])
    assert [c[0] for c in calls] == [[a]]
    opt.add_param_group(dict(params=[b], lr=1e-2))   # a refusal does not spoil the parameter
    step(opt, [a, b])
    assert [c[0] for c in calls] == [[a], [a], [b]]


@pytest.mark.parametrize("capturable", [False, True])
def test_states_are_loaded_again(calls, capturable):
    """A second state after a first, and one into a copy of the optimiser: torch adds options of its own to those that a loaded or
    copied optimiser has, which no state of this one holds."""
    ps = params(300, 200)
    opt = AdamW(ps, lr=1e-3, state_bits=8, capturable=capturable)
    step(opt, ps)
    first = opt.state_dict()
    for other in (opt, copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        for _ in range(2):
            other.load_state_dict(first)
        assert [int(st["step"]) for st in other.state.values()] == [1, 1]
