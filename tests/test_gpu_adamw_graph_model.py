"""A model whose optimiser's step is replayed from a graph: a replay counts up no version, and what the layers keep prepared of their
weights has to follow all the same."""
import pytest
import torch

from sdmchat_amd import DecodeGraph, OneSdmLM

pytestmark = pytest.mark.gpu
KW = dict(d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4, sdm_n_sub=8, sdm_heads=2, sdm_d_a=16, sdm_k=8)


def fresh(model, ffn, dtype):
    """The same weights in a model that has prepared none yet."""
    twin = OneSdmLM(211, **KW, ffn=ffn, seed=5).cuda().to(dtype)
    twin.load_state_dict(model.state_dict())
    return twin


@pytest.mark.parametrize("ffn", ["mlp", "sdm"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_replayed_steps_reach_the_next_forward(ffn, dtype, bits):
    torch.manual_seed(3)
    model = OneSdmLM(211, **KW, ffn=ffn, seed=4).cuda().to(dtype)
    opt = model.optimizer(3e-2, state_bits=bits, capturable=True)
    idx = torch.randint(0, 211, (3, 24), device="cuda")
    for p in model.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    with torch.no_grad():
        model(idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    last = None
    for _ in range(4):
        graph.replay()
        with torch.no_grad():
            twin = fresh(model, ffn, dtype)
            now = model(idx)
            assert torch.equal(now, twin(idx))
            assert last is None or not torch.equal(now, last)
            a, b = model.decode_state(3), twin.decode_state(3)
            for t in range(4):
                assert torch.equal(model.step(idx[:, t], a), twin.step(idx[:, t], b))
            with torch.autocast("cuda", dtype=torch.bfloat16):
                assert torch.equal(model(idx), twin(idx))
        last = now
    # a graph of decode steps that is captured now follows the replays after it
    with torch.no_grad():
        decode = DecodeGraph(model, model.decode_state(3))
        for t in range(3):
            graph.replay()
            state = decode.state
            for st, z in zip(state.layers, model.decode_state(3).layers):
                for have, zero in ((st.mem, z.mem), (st.cnt, z.cnt), (st.scale, z.scale), (st.last, z.last)):
                    if have is not None:
                        have.copy_(zero)
            twin = fresh(model, ffn, dtype)
            got = decode.step(idx[:, 0])
            assert torch.equal(got, twin.step(idx[:, 0], twin.decode_state(3)))
