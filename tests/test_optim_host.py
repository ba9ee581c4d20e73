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


def trained(bits, capturable, lr):
    ps = params(300, 200)
    opt = AdamW([dict(params=ps[:1]), dict(params=ps[1:])], lr=lr, state_bits=bits, capturable=capturable)
    step(opt, ps)
    step(opt, ps[:1])
    for st in opt.state.values():
        for k, v in st.items():
            if k != "step":
                v.fill_(3)
    return ps, opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("mine", ["number", "tensor", "row"])
@pytest.mark.parametrize("loaded", ["number", "tensor", "row"])
def test_a_rate_that_is_a_tensor_is_loaded_into(calls, bits, mine, loaded):
    """The tensor that a schedule writes and a graph holds stays the group's and takes the loaded value; a number becomes a copy
    of a loaded tensor."""
    def rate(kind, value):
        return value if kind == "number" else torch.full(() if kind == "tensor" else (1,), value)
    _, old = trained(bits, True, rate(loaded, 0.25))
    lr = rate(mine, 0.5)
    ps, new = trained(bits, True, lr)
    sd = old.state_dict()
    new.load_state_dict(sd)
    for g, s in zip(new.param_groups, sd["param_groups"]):
        assert float(g["lr"]) == 0.25 and torch.is_tensor(g["lr"]) == (mine != "number" or loaded != "number")
        if mine != "number":
            assert g["lr"] is lr
            lr.fill_(0.125)
            assert float(s["lr"]) == 0.25   # the checkpoint's is another
            lr.fill_(0.25)
        elif loaded != "number":
            assert g["lr"] is not s["lr"] and g["lr"].device == g["params"][0].device
    step(new, ps)
    assert float(calls[-1][3]) == 0.25
    if mine != "number":   # its own state again
        new.load_state_dict(new.state_dict())
        assert all(g["lr"] is lr for g in new.param_groups) and float(lr) == 0.25


def test_a_rate_of_several_values_is_refused(calls):
    _, opt = trained(32, True, torch.full((), 0.5))
    sd = opt.state_dict()
    sd["param_groups"][1]["lr"] = torch.ones(2)
    with pytest.raises(ValueError, match="lr"):
        opt.load_state_dict(sd)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("what", ["no step", "step of another kind", "negative step", "no moments", "another size", "a number", "groups"])
def test_a_refused_state_changes_nothing(calls, bits, capturable, what):
    ps, opt = trained(bits, capturable, 0.5)
    keep = {p: {k: v.clone() if torch.is_tensor(v) else v for k, v in st.items()} for p, st in opt.state.items()}
    held = {p: dict(st) for p, st in opt.state.items()}
    sd = trained(bits, capturable, 0.25)[1].state_dict()
    sd["state"] = {k: dict(st) for k, st in sd["state"].items()}
    key = "moments" if bits == 8 else "exp_avg"
    if what == "no step":
        del sd["state"][1]["step"]
    elif what == "step of another kind":
        sd["state"][1]["step"] = torch.ones(2) if capturable else "many"
    elif what == "negative step":
        sd["state"][1]["step"] = -1
    elif what == "no moments":
        del sd["state"][1][key]
    elif what == "another size":
        sd["state"][1][key] = sd["state"][1][key][:1]
    elif what == "a number":
        sd["state"][1][key] = 3.0
    else:
        sd["param_groups"] = sd["param_groups"][:1]
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.5] and list(opt.state) == list(keep)
    for p, st in opt.state.items():
        assert all(held[p][k] is v for k, v in st.items())
        assert all(torch.equal(v, keep[p][k]) if torch.is_tensor(v) else v == keep[p][k] for k, v in st.items())


@pytest.mark.parametrize("capturable", [False, True])
def test_hooks_of_a_loaded_state(calls, capturable):
    """A hook before sees, and may replace, the whole state; one after finds the new state in place."""
    _, old = trained(8, capturable, 0.25)
    ps, new = trained(8, capturable, 0.5)
    seen = []

    def before(opt, sd):
        seen.append(sorted(sd["state"]))
        return dict(sd, state={k: dict(st, step=st["step"] + 5) for k, st in sd["state"].items()})
    new.register_load_state_dict_pre_hook(before)
    new.register_load_state_dict_post_hook(lambda opt: seen.append([int(opt.state[p]["step"]) for p in ps]))
    new.load_state_dict(old.state_dict())
    assert seen == [[0, 1], [7, 6]]
    assert [int(new.state[p]["step"]) for p in ps] == [7, 6]
    new.load_state_dict(old.state_dict())   # the optimiser's own hooks were for one call
    assert seen[2:] == [[0, 1], [7, 6]] and len(seen) == 4
