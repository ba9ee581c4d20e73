"""Token log probabilities, the gradients' norm and the AdamW step, what needs no GPU: the C ABI's checks of arguments (they run
before anything is launched), the optimiser's own, and that CPU tensors are refused."""
import ctypes
import math

import pytest
import torch

from sdmchat_amd import AdamW, OneSdmLM, _lib, core

P = 0x1000   # a pointer that no check reads


def _fails(rc, code, text):
    lib = _lib.load()
    assert rc == code, (rc, lib.sdm_rt_last_error())
    assert text in lib.sdm_rt_last_error().decode()


def _logprob(**over):
    a = dict(rows=4, vocab=100, top_k=5, temperature=1.0, ignore_index=-100, logits=P, ls=100, dtype=0, targets=P, lp=P, h=P,
             ids=P, tops=P, stats=P, ws=P, nws=1 << 40, dz=P, dzs=100)
    a.update(over)
    dims = _lib.SdmRtLogprob(a["rows"], a["vocab"], a["top_k"], a["temperature"], a["ignore_index"])
    return a, dims, (ctypes.byref(dims), a["logits"], a["ls"], a["dtype"], a["targets"])


BAD = [(dict(dtype=2), -1, "dtype"), (dict(rows=-1), -1, "rows"), (dict(vocab=0), -1, "vocab"), (dict(top_k=-1), -1, "top_k"),
       (dict(top_k=257), -3, "256"), (dict(rows=(1 << 21) + 1), -3, "2^21"),
       (dict(vocab=(1 << 21) + 1, ls=(1 << 21) + 1, dzs=(1 << 21) + 1), -3, "2^21"),
       (dict(temperature=0.0), -1, "temperature"), (dict(temperature=-1.0), -1, "temperature"),
       (dict(temperature=math.nan), -1, "temperature"), (dict(temperature=math.inf), -1, "temperature"),
       (dict(logits=None), -1, "logits"), (dict(ls=99), -1, "stride"), (dict(ls=-100), -1, "stride"),
       (dict(targets=None), -1, "need targets"), (dict(stats=P + 4), -1, "16-byte")]


@pytest.mark.parametrize("over,code,text", BAD + [(dict(ids=None), -1, "top_ids"), (dict(tops=None), -1, "top_ids")])
def test_logprob_checks(over, code, text):
    a, dims, head = _logprob(**over)
    lib = _lib.load()
    _fails(lib.sdm_rt_token_logprobs(*head, a["lp"], a["h"], a["ids"], a["tops"], a["stats"], a["ws"], a["nws"], None), code, text)


@pytest.mark.parametrize("over,code,text", BAD + [(dict(stats=None), -1, "stats"), (dict(dz=None), -1, "d_logits"),
                                                  (dict(dzs=99), -1, "d_logits_row_stride")])
def test_logprob_grad_checks(over, code, text):
    a, dims, head = _logprob(**over)
    lib = _lib.load()
    _fails(lib.sdm_rt_token_logprobs_grad(*head, a["stats"], P, 1, P, 1, a["dz"], a["dzs"], None), code, text)


def test_no_rows_is_nothing_to_do():
    a, dims, head = _logprob(rows=0, logits=None)
    lib = _lib.load()
    assert lib.sdm_rt_token_logprobs(*head, P, P, P, P, P, None, 0, None) == 0
    assert lib.sdm_rt_token_logprobs_grad(*head, P, P, 1, P, 1, P, 100, None) == 0


def test_logprob_workspace():
    lib = _lib.load()
    for dtype in (0, 1):
        a, dims, head = _logprob(rows=3, vocab=1 << 20, top_k=100, dtype=dtype, ls=1 << 20)
        need = lib.sdm_rt_token_logprobs_workspace_bytes(ctypes.byref(dims), dtype)
        if need:
            _fails(lib.sdm_rt_token_logprobs(*head, P, P, P, P, P, P, need - 1, None), -2, "needed")
            _fails(lib.sdm_rt_token_logprobs(*head, P, P, P, P, P, None, need, None), -2, "needed")


def _table(*rows):
    return (ctypes.c_int64 * (6 * len(rows)))(*[x for r in rows for x in r])


def _options(**over):
    a = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, t=1, t_device=None, lr_device=None, norm=None,
             max_norm=1.0, state_bits=32, seed=0)
    a.update(over)
    return _lib.SdmRtAdamwOptions(*a.values())


GOOD = (P, P, P, P, 100, 0)


@pytest.mark.parametrize("over,row,code,text", [
    (dict(t=0), GOOD, -1, "t must"), (dict(beta1=1.0), GOOD, -1, "beta1"), (dict(beta2=-0.1), GOOD, -1, "beta2"),
    (dict(beta1=math.nan), GOOD, -1, "beta1"), (dict(eps=-1.0), GOOD, -1, "eps"), (dict(eps=math.inf), GOOD, -1, "eps"),
    (dict(weight_decay=math.nan), GOOD, -1, "weight_decay"), (dict(lr=math.inf), GOOD, -1, "lr"), (dict(lr=-1.0), GOOD, -1, "lr"),
    (dict(lr_device=P), GOOD, -1, "t_device"), (dict(norm=P, max_norm=0.0), GOOD, -1, "max_norm"),
    (dict(norm=P, max_norm=math.nan), GOOD, -1, "max_norm"), (dict(state_bits=16), GOOD, -1, "state_bits"),
    (dict(), (0, P, P, P, 100, 0), -1, "NULL"), (dict(), (P, 0, P, P, 100, 0), -1, "NULL"), (dict(), (P, P, 0, P, 100, 0), -1, "NULL"),
    (dict(), (P, P, P, 0, 100, 0), -1, "NULL"), (dict(state_bits=8), GOOD, -1, "NULL for 8 bits"),
    (dict(state_bits=8), (P, P, P + 4, 0, 100, 0), -1, "8-byte"), (dict(), (P, P, P, P, -1, 0), -1, "n must"),
    (dict(), (P, P, P, P, 100, 2), -1, "dtype"), (dict(), (P, P, P, P, (1 << 33) + 1, 0), -3, "2^33"), (dict(), (P, P, P, P, 1 << 33, 0), -3, "more than")])
def test_adamw_checks(over, row, code, text):
    lib = _lib.load()
    o = _options(**over)
    _fails(lib.sdm_rt_adamw(ctypes.byref(o), _table(GOOD if not over.get("state_bits", 32) == 8 else (P, P, P, 0, 9, 1), row), 2,
                            None), code, text)


def test_other_checks_of_lists():
    lib = _lib.load()
    _fails(lib.sdm_rt_adamw(None, _table(GOOD), 1, None), -1, "options")
    _fails(lib.sdm_rt_adamw(ctypes.byref(_options()), None, 1, None), -1, "tensors")
    _fails(lib.sdm_rt_adamw(ctypes.byref(_options()), _table(GOOD), -1, None), -1, "count")
    assert lib.sdm_rt_adamw(ctypes.byref(_options()), None, 0, None) == 0
    assert lib.sdm_rt_adamw(ctypes.byref(_options()), _table((0, 0, 0, 0, 0, 0)), 1, None) == 0   # no values
    t = _table((0, P, 0, 0, 100000, 1), (0, P, 0, 0, 3, 0))
    need = lib.sdm_rt_grad_norm_workspace_bytes(t, 2)
    assert need > 0
    _fails(lib.sdm_rt_grad_norm(t, 2, P, P, need - 1, None), -2, "needed")
    _fails(lib.sdm_rt_grad_norm(t, 2, P, P + 4, need, None), -1, "8-byte")
    _fails(lib.sdm_rt_grad_norm(t, 2, None, P, need, None), -1, "norm")
    _fails(lib.sdm_rt_grad_norm(_table((0, 0, 0, 0, 5, 0)), 1, P, P, 1 << 20, None), -1, "grad")
    _fails(lib.sdm_rt_read_moments(_table((P, 0, P, 0, 5, 0)), 1, None), -1, "NULL")
    _fails(lib.sdm_rt_read_moments(_table((P, 0, P + 2, P, 5, 0)), 1, None), -1, "8-byte")
    assert [lib.sdm_rt_moments_bytes(n) for n in (-1, 0, 1, 128, 129)] == [0, 0, 264, 264, 528]


def test_cpu_tensors_are_refused():
    z, y = torch.randn(3, 10), torch.zeros(3, dtype=torch.long)
    for call in (lambda: core.token_logprobs(z, y), lambda: core.grad_norm([z]), lambda: core.adamw([z], [z], [z], [z], step=1),
                 lambda: core.read_moments([z], [z], [z])):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
    p = torch.nn.Parameter(z)
    p.grad = z.clone()
    with pytest.raises(RuntimeError, match="ROCm device"):
        AdamW([p]).step()


def test_new_moments():
    for n in (0, 1, 128, 129):
        m = core.new_moments(torch.zeros(n))
        assert m.dtype == torch.uint8 and m.numel() == _lib.load().sdm_rt_moments_bytes(n) and not m.any()


@pytest.mark.parametrize("over,text", [
    (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(betas=(0.9, 1.0)), "betas"), (dict(betas=(0.9,)), "betas"),
    (dict(eps=-1e-8), "eps"), (dict(weight_decay=-0.1), "weight_decay"), (dict(state_bits=16), "state_bits"),
    (dict(max_norm=0.0), "max_norm"), (dict(lr=torch.ones(())), "capturable")])
def test_optimizer_checks(over, text):
    with pytest.raises(ValueError, match=text):
        AdamW([torch.nn.Parameter(torch.zeros(3))], **over)


def test_optimizer_checks_groups():
    a, b = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ValueError, match="float64"):
        AdamW([a, b])
    with pytest.raises(ValueError, match="same for all"):
        AdamW([dict(params=[a], max_norm=2.0)], max_norm=1.0)
    with pytest.raises(ValueError, match="duplicate|more than one"):
        AdamW([dict(params=[a]), dict(params=[a])])


def test_model_optimizer_groups():
    model = OneSdmLM(100, d=64, layers=1, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4, learn_scale=False)
    opt = model.optimizer(1e-3, 0.3, state_bits=8, max_norm=1.0)
    names = {id(p): n for n, p in model.named_parameters()}
    decayed, rest = ([names[id(p)] for p in g["params"]] for g in opt.param_groups)
    assert [g["weight_decay"] for g in opt.param_groups] == [0.3, 0.0]
    assert "emb.weight" in decayed and "mems.0.wk.weight" in decayed and "mlps.0.down.weight" in decayed
    assert "nf.w" in rest and "mems.0.keys1" in rest and "mems.0.onorm_w" in rest and "mems.0.wg.bias" in rest
    assert sorted(decayed + rest) == sorted(n for n, p in model.named_parameters() if p.requires_grad)


def test_native_lists():
    """What the extension does not pack is left to the caller: CPU tensors, other lengths, no tensors at all."""
    pack = _lib.lists().pack
    a, b = torch.zeros(3), torch.zeros(3)
    assert pack(None, [a], None, None, False, False) is None
    assert pack([a], [a, b], [a], [b], False, False) is None
    assert pack([], [], [], [], False, False) is None
    assert pack(None, None, None, None, False, False) is None
    assert pack([1], [2], [3], [4], False, False) is None
    assert pack((a,), [a], [a], [b], False, False) is None
    with pytest.raises(TypeError):
        pack([a])
    v = a._version
    _lib.lists().written([a], [])
    assert a._version == v + 1 and b._version == 0
    with torch.inference_mode():
        c = torch.zeros(3)
    _lib.lists().written([c])
    rows = _lib.lists().new_rows(torch.zeros(2, dtype=torch.bfloat16), 3, 5, "f-IF")
    assert [None if t is None else (tuple(t.shape), t.dtype) for t in rows] == [
        ((3,), torch.float32), None, ((3, 5), torch.int64), ((3, 5), torch.float32)]
    with pytest.raises(TypeError):
        _lib.lists().new_rows(1, 2, 3, "f")


def test_a_foreign_optimizer_state_is_refused():
    p = torch.nn.Parameter(torch.zeros(3))
    other = torch.optim.AdamW([p])
    with pytest.raises(ValueError, match="not the state"):
        AdamW([p]).load_state_dict(other.state_dict())
    import copy
    opt = copy.deepcopy(AdamW([p], state_bits=8, max_norm=2.0))
    assert opt.norm is None and opt.defaults["max_norm"] == 2.0 and opt.param_groups[0]["state_bits"] == 8
