"""TokenRules in captured decode loops, on the GPU: what the graph keeps, bit for bit against eager steps."""
import gc

import pytest
import torch

from sdmchat_amd import DecodeGraph, OneSdmLM, TokenRules, core

pytestmark = pytest.mark.gpu
B, V = 4, 211


def _model():
    torch.manual_seed(0)
    return OneSdmLM(V, d=64, layers=2, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4).cuda().eval()


def _rules(window=6):
    g = torch.Generator().manual_seed(4)
    return TokenRules(B, window, "cuda", repetition=1.0 + torch.rand(B, generator=g).cuda(), frequency=torch.rand(B, generator=g).cuda(),
                      presence=0.2, bias=torch.randn(V, generator=g).cuda(),
                      mask=core.pack_mask(torch.rand(B, V, generator=g) < 0.7).cuda())


def _graph(m, state, replaced):
    """A graph whose rules nothing else holds, or whose rules' tensors are no longer the captured ones."""
    rules = _rules()
    graph = DecodeGraph(m, state, rules=rules)
    if replaced:
        rules.mask, rules.bias, rules.repetition = torch.zeros_like(rules.mask), torch.zeros_like(rules.bias), 1.0
        rules.tokens, rules.lengths = torch.zeros_like(rules.tokens), torch.zeros_like(rules.lengths)
    return graph


@pytest.mark.parametrize("replaced", [False, True])
def test_a_graph_outlives_the_callers_rules(replaced):
    m = _model()
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        s1, s2, rules = m.decode_state(B, "cuda"), m.decode_state(B, "cuda"), _rules()
        graph = _graph(m, s1, replaced)
        gc.collect()
        # where dropped tensors would have been: filled, and looked at again at the end
        others = [torch.full((n,), 77, dtype=torch.long, device="cuda") for n in (B, B, B, B * 6, B * 6, V, V, 64, 64) for _ in range(4)]
        for r in range(4):
            toks = torch.randint(0, V, (B,), generator=g).cuda()
            got = graph.run(toks)
            want = m.step(toks, s2, rules)
            torch.cuda.synchronize()
            assert torch.equal(got, want), r
        assert all(bool((t == 77).all()) for t in others)
