"""Token ids outside the table, on the GPU: told by embedding(check=True) and by OneSdmLM, clamped in any case."""
import pytest
import torch

from sdmchat_amd import DecodeGraph, ForwardGraph, OneSdmLM, core

pytestmark = pytest.mark.gpu
V = 97


@pytest.fixture(autouse=True)
def nothing_left_behind():
    core.check_token_ids()
    yield
    core.check_token_ids()


def _model(**kw):
    torch.manual_seed(0)
    return OneSdmLM(V, d=64, layers=1, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4, **kw).cuda()


@pytest.mark.parametrize("bad", [-1, V, 2 ** 40, -2 ** 62])
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("d", [3, 64, 330])
def test_lookup_tells_of_an_id_outside(bad, train, d):
    table = torch.randn(V, d, device="cuda", requires_grad=train)
    ids = torch.arange(V, device="cuda").repeat(30)
    y = core.embedding(ids, table, check=True)
    core.check_token_ids()
    assert torch.equal(y, table[ids])
    ids[-7] = bad
    core.embedding(ids, table)   # not asked for
    core.check_token_ids()
    y = core.embedding(ids, table, check=True)
    assert torch.equal(y, table[ids.clamp(0, V - 1)])
    with pytest.raises(IndexError, match=str(bad)):
        core.check_token_ids("cuda:0")
    core.check_token_ids()   # told once
    core.embedding(ids, table, check=True)
    torch.cuda.synchronize()
    with pytest.raises(IndexError, match="outside"):   # the next call tells as well, before it does anything
        core.embedding(ids[:5], table, check=True)
    core.embedding(ids[:5], table, check=True)


def test_no_tokens():
    core.embedding(torch.zeros(0, dtype=torch.long, device="cuda"), torch.randn(V, 8, device="cuda"), check=True)


@pytest.mark.parametrize("scale", [1.0, 8.0])
def test_model_tells(scale):
    """Training and prefill with a token past the vocabulary, as a tokenizer of another model gives."""
    m = _model(emb_scale=scale)
    idx = torch.randint(0, V, (2, 20), generator=torch.Generator().manual_seed(1)).cuda()
    wrong = idx.clone()
    wrong[1, 3] = V + 4
    m(idx).float().sum().backward()
    core.check_token_ids()
    m(wrong).float().sum().backward()
    torch.cuda.synchronize()
    with pytest.raises(IndexError, match=str(V + 4)):
        m(idx)
    m(idx)
    m.eval()
    with torch.no_grad():
        m.prefill(wrong)
        with pytest.raises(IndexError, match=str(V + 4)):
            core.check_token_ids()
        m.check_ids = False
        m.prefill(wrong)
        core.check_token_ids()


def test_graphs_tell():
    m = _model().eval()
    with torch.no_grad():
        graph, step = ForwardGraph(m, 2, 8), DecodeGraph(m, m.decode_state(3, "cuda"))
        good, wrong = torch.zeros(2, 8, dtype=torch.long, device="cuda"), torch.full((2, 8), V, device="cuda")
        graph.run(good)
        graph.run(wrong)
        torch.cuda.synchronize()
        with pytest.raises(IndexError, match=str(V)):
            graph.run(good)
        graph.run(good)
        step.run(wrong[0, :3])
        torch.cuda.synchronize()
        with pytest.raises(IndexError, match=str(V)):
            step.run(good[0, :3])


def test_a_capture_before_any_call_does_not_allocate(monkeypatch):
    monkeypatch.setattr(core, "_OUTSIDE", {})
    table, ids = torch.randn(V, 8, device="cuda"), torch.tensor([1, V + 9], device="cuda")
    core.embedding(ids, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = core.embedding(ids, table, check=True)
    graph.replay()
    torch.cuda.synchronize()
    assert not core._OUTSIDE and torch.equal(y, table[[1, V - 1]])
