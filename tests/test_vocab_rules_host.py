"""TokenRules in a model and in a captured decode loop, what needs no GPU."""
import contextlib
import gc
import types
import weakref

import pytest
import torch

from sdmchat_amd import DecodeGraph, OneSdmLM, TokenRules

B, V = 3, 40


class _Model:
    """What DecodeGraph asks of a model, on the CPU."""
    emb = types.SimpleNamespace(weight=torch.zeros(V, 4))

    def decode_state(self, batch, device=None):
        return types.SimpleNamespace(layers=[types.SimpleNamespace(mem=torch.zeros(batch, 1))], pos=0)

    def step(self, idx_t, state, rules=None):
        state.pos += 1
        return torch.zeros(idx_t.shape[0], V)


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", lambda g: contextlib.nullcontext())


NAMES = ("tokens", "lengths", "prompt", "repetition", "frequency", "presence", "bias", "mask")


def _rules():
    return TokenRules(B, 5, "cpu", repetition=torch.ones(B), frequency=torch.zeros(B), presence=torch.zeros(B), bias=torch.zeros(V),
                      mask=torch.zeros(B, 2, dtype=torch.int32))


@pytest.mark.parametrize("replaced", [False, True])
def test_a_decode_graph_keeps_the_rules_and_the_tensors_it_captured(no_gpu, replaced):
    """The captured steps read and write the rules' tensors of the capture: they live as long as the graph, whether the
    caller drops the rules or puts other tensors into them."""
    m, rules = _Model(), _rules()
    graph = DecodeGraph(m, m.decode_state(B), rules=rules)
    refs = [weakref.ref(getattr(rules, n)) for n in NAMES]
    whole = weakref.ref(rules)
    if replaced:
        for n in NAMES:
            setattr(rules, n, getattr(rules, n).clone())
    del rules
    gc.collect()
    assert whole() is not None and all(r() is not None for r in refs)
    del graph
    gc.collect()
    assert whole() is None and all(r() is None for r in refs)


def test_a_decode_graph_without_rules(no_gpu):
    m = _Model()
    assert DecodeGraph(m, m.decode_state(B)).rules is None


def test_rules_that_cannot_be_applied_are_refused_before_a_step_moves():
    """Rules on the CPU, where the kernels do not run: the state has not taken the token."""
    m = OneSdmLM(V, d=16, layers=1, mlp_f=16, mem=False, ffn="none", heads=4, n_sub=4, d_a=4, k=2)
    state = m.decode_state(B)
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm"):
        m.step(torch.zeros(B, dtype=torch.long), state, TokenRules(B, 4, "cpu"))
    assert state.pos == 0
