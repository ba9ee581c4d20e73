"""Graphs of a model's decode step and forward after the layers have let go of what the capture used: a larger eager call takes
another workspace, a training step makes the layers prepare their weights anew."""
import pytest
import torch

from sdmchat_amd import DecodeGraph, ForwardGraph, OneSdmLM, core

pytestmark = pytest.mark.gpu
KW = dict(d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4, sdm_n_sub=8, sdm_heads=2, sdm_d_a=16, sdm_k=8)


def tensors_of(held):
    if torch.is_tensor(held):
        yield held
    elif isinstance(held, (tuple, list)):
        for h in held:
            yield from tensors_of(h)


@pytest.mark.parametrize("ffn", ["mlp", "sdm"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_graph_keeps_what_it_captured(ffn, dtype):
    torch.manual_seed(1)
    model = OneSdmLM(211, **KW, ffn=ffn, seed=4).cuda().to(dtype)
    opt = model.optimizer(0.0, weight_decay=0.0)   # steps that leave every weight as it is, but count up its version
    idx = torch.randint(0, 211, (2, 24), device="cuda")
    forward = ForwardGraph(model, 2, 24)
    decode = DecodeGraph(model, model.decode_state(3))
    before = forward.run(idx).clone()
    first = decode.step(idx.view(-1)[:3]).clone()
    held = list(tensors_of(core.prepared(model)))
    sizes = [t.untyped_storage().nbytes() for t in held]
    assert len(held) > 8 and {t.data_ptr() for t in held} <= {t.data_ptr() for g in (forward, decode) for t in tensors_of(g._held)}
    del held
    for p in model.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    with torch.no_grad():
        model(torch.randint(0, 211, (8, 400), device="cuda"))   # larger, on new weights
        model.step(idx.view(-1)[:3], model.decode_state(3))
    now = {t.data_ptr() for t in tensors_of(core.prepared(model))}
    assert sum(t.data_ptr() not in now for t in tensors_of(forward._held)) >= 4   # two layers' weights and workspaces at least
    # what the layers let go of would be these tensors' memory now
    marks = [torch.full((n,), 0x5a, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
    for st, z in zip(decode.state.layers, model.decode_state(3).layers):
        for have, zero in ((st.mem, z.mem), (st.cnt, z.cnt), (st.scale, z.scale), (st.last, z.last)):
            if have is not None:
                have.copy_(zero)
    for _ in range(2):
        assert torch.equal(forward.run(idx), before)
    assert torch.equal(decode.step(idx.view(-1)[:3]), first)
    torch.cuda.synchronize()
    assert all(bool((m == 0x5a).all()) for m in marks)
