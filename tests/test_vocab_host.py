"""The operators at the ends of the vocabulary, what needs no GPU: the C ABI's checks of arguments (they run before
anything is launched), the packed grammar mask, the token history's layout, and that CPU tensors are refused."""
import ctypes

import pytest
import torch

from sdmchat_amd import OneSdmLM, TokenRules, _lib, core

P = 0x1000   # a pointer that no check reads


def _fails(rc, code, text):
    lib = _lib.load()
    assert rc == code, (rc, lib.sdm_rt_last_error())
    assert text in lib.sdm_rt_last_error().decode()


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=7), -1, "dtype"), (dict(n=-1), -1, "n must"), (dict(vocab=0), -1, "vocab"), (dict(d=0), -1, "d >= 1"),
    (dict(ids=None), -1, "NULL"), (dict(table=None), -1, "NULL"), (dict(out=None), -1, "NULL"),
    (dict(ts=7), -1, "stride"), (dict(os=7), -1, "stride"), (dict(vocab=(1 << 21) + 1), -3, "2^21"),
    (dict(n=(1 << 27) + 1), -3, "2^27"),
])
def test_embed_checks(over, code, text):
    a = dict(ids=P, n=4, table=P, ts=8, dtype=0, vocab=10, d=8, out=P, os=8)
    a.update(over)
    lib = _lib.load()
    _fails(lib.sdm_rt_embed(a["ids"], a["n"], a["table"], a["ts"], a["dtype"], a["vocab"], a["d"], 1.0, a["out"], a["os"],
                            None), code, text)
    b = dict(a, dy=a["table"], dt=a["out"])
    _fails(lib.sdm_rt_embed_backward(b["ids"], b["n"], b["dy"], b["ts"], b["dtype"], b["vocab"], b["d"], 1.0, -1, b["dt"],
                                     b["os"], P, 1 << 40, None), code, text)


def test_embed_backward_workspace():
    lib = _lib.load()
    need = lib.sdm_rt_embed_backward_workspace_bytes(100, 1000, 64)
    assert need >= 4 * (1000 + 100)
    assert lib.sdm_rt_embed_backward_workspace_bytes(-1, 1000, 64) == 0
    assert lib.sdm_rt_embed_backward_workspace_bytes(100, 0, 64) == 0
    _fails(lib.sdm_rt_embed_backward(P, 100, P, 64, 0, 1000, 64, 1.0, -1, P, 64, P, need - 1, None), -2, "needed")
    _fails(lib.sdm_rt_embed_backward(P, 100, P, 64, 0, 1000, 64, 1.0, -1, P, 64, None, need, None), -1, "workspace")
    wide = 1 << 20
    _fails(lib.sdm_rt_embed_backward(P, 1 << 27, P, wide, 0, 10, wide, 1.0, -1, P, wide, P, 1 << 60, None), -3, "one launch")


def _distill(**over):
    a = dict(rows=4, vocab=100, top_k=8, temperature=2.0, alpha=0.5, ignore_index=-100, reduction=1, logits=P, ls=100, dtype=0,
             ids=P, ids_s=8, top=P, top_s=8, labels=P, loss=P, stats=P, ws=P, nws=1 << 30, go=P, dz=P, dzs=100)
    a.update(over)
    dims = _lib.SdmRtDistill(a["rows"], a["vocab"], a["top_k"], a["temperature"], a["alpha"], a["ignore_index"],
                             a["reduction"])
    head = (ctypes.byref(dims), a["logits"], a["ls"], a["dtype"], a["ids"], a["ids_s"], a["top"], a["top_s"], a["labels"])
    return dims, a, head


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=2), -1, "dtype"), (dict(rows=-1), -1, "rows"), (dict(vocab=0), -1, "vocab"), (dict(top_k=-1), -1, "top_k"),
    (dict(top_k=1025, ids_s=1025, top_s=1025), -3, "1024"), (dict(rows=(1 << 21) + 1), -3, "2^21"),
    (dict(temperature=0.0), -1, "temperature"), (dict(temperature=-1.0), -1, "temperature"),
    (dict(temperature=float("inf")), -1, "temperature"), (dict(temperature=float("nan")), -1, "temperature"),
    (dict(temperature=1e-40), -1, "temperature"), (dict(alpha=1.5), -1, "alpha"), (dict(alpha=float("nan")), -1, "alpha"),
    (dict(reduction=3), -1, "reduction"), (dict(logits=None), -1, "logits"), (dict(ls=99), -1, "logits"),
    (dict(ids=None), -1, "top_ids"), (dict(top=None), -1, "top_logits"), (dict(ids_s=7), -1, "strides"),
    (dict(top_s=7), -1, "strides"), (dict(stats=P + 4), -1, "aligned"),
])
def test_distill_checks(over, code, text):
    lib = _lib.load()
    dims, a, head = _distill(**over)
    _fails(lib.sdm_rt_distill_loss(*head, a["loss"], a["stats"], a["dz"], a["dzs"], a["ws"], a["nws"], None), code, text)
    _fails(lib.sdm_rt_distill_grad(*head, a["stats"], a["go"], 1, a["dz"], a["dzs"], None), code, text)


def test_distill_checks_of_outputs():
    lib = _lib.load()
    dims, a, head = _distill()
    need = lib.sdm_rt_distill_workspace_bytes(ctypes.byref(dims))
    _fails(lib.sdm_rt_distill_loss(*head, None, P, P, 100, P, need, None), -1, "loss")
    _fails(lib.sdm_rt_distill_loss(*head, P, P, P, 99, P, need, None), -1, "d_logits_row_stride")
    _fails(lib.sdm_rt_distill_loss(*head, P, P, P, 100, P, need - 1, None), -2, "needed")
    _fails(lib.sdm_rt_distill_grad(*head, None, P, 0, P, 100, None), -1, "stats")
    _fails(lib.sdm_rt_distill_grad(*head, P, None, 0, P, 100, None), -1, "grad_out")
    _fails(lib.sdm_rt_distill_grad(*head, P, P, 0, P, 99, None), -1, "d_logits_row_stride")
    dims, a, head = _distill(reduction=0)
    _fails(lib.sdm_rt_distill_grad(*head, P, P, 1, P, 100, None), -1, "unless_one")


@pytest.mark.parametrize("over,call,code,text", [
    (dict(tokens=P, width=4, tokens_row_stride=4), {}, -1, "lengths"),
    (dict(tokens=P, width=4, tokens_row_stride=3, lengths=P), {}, -1, "history"),
    (dict(width=-1), {}, -1, "width"), (dict(bias=P, bias_row_stride=99), {}, -1, "bias_row_stride"),
    (dict(mask=P, mask_row_stride=3), {}, -1, "mask_row_stride"), ({}, dict(dtype=9), -1, "dtype"),
    ({}, dict(rows=-1), -1, "rows"), ({}, dict(vocab=0), -1, "vocab"), ({}, dict(rows=65536), -3, "65,535"),
    ({}, dict(logits=None), -1, "NULL"), ({}, dict(out=None), -1, "NULL"), ({}, dict(os=99), -1, "stride"),
    ({}, dict(ls=99), -1, "stride"),
])
def test_process_logits_checks(over, call, code, text):
    r = _lib.SdmRtRules(**over)
    a = dict(logits=P, ls=100, dtype=0, rows=3, vocab=100, out=P, os=100)
    a.update(call)
    lib = _lib.load()
    _fails(lib.sdm_rt_process_logits(ctypes.byref(r), a["logits"], a["ls"], a["dtype"], a["rows"], a["vocab"], a["out"],
                                     a["os"], None), code, text)
    _fails(lib.sdm_rt_process_logits(None, P, 100, 0, 3, 100, P, 100, None), -1, "rules")


def test_append_tokens_checks():
    lib = _lib.load()
    _fails(lib.sdm_rt_append_tokens(P, 4, 0, P, P, 2, None), -1, "width")
    _fails(lib.sdm_rt_append_tokens(P, 3, 4, P, P, 2, None), -1, "stride")
    _fails(lib.sdm_rt_append_tokens(None, 4, 4, P, P, 2, None), -1, "NULL")
    assert lib.sdm_rt_append_tokens(None, 4, 4, None, None, 0, None) == 0


def test_cpu_tensors_are_refused():
    ids = torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="ROCm"):
        core.embedding(ids, torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="ROCm"):
        core.embedding_backward(ids, torch.zeros(3, 8), 4)
    with pytest.raises(RuntimeError, match="ROCm"):
        core.distill_loss(torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match="ROCm"):
        core.process_logits(torch.zeros(3, 8))
    with pytest.raises(RuntimeError, match="ROCm"):
        core.append_tokens(torch.zeros(3, 8, dtype=torch.long), ids, ids)


def test_apart():
    """Which outputs share elements with their input in part."""
    buf = torch.zeros(9, 24)
    for a, b, want in ((buf, buf, True), (buf, torch.zeros(9, 24), True), (buf[:4], buf[4:8], True), (buf[:4], buf[1:5], False),
                       (buf[:, :8], buf[:, 8:16], True), (buf[:, :8], buf[:, 16:], True), (buf[:, :8], buf[:, 7:15], False),
                       (buf[0:1], buf[0:1], True), (buf[0:1, :8], buf[0:1, 4:12], False), (buf[:0], buf[:0], True),
                       # one row repeated: before, at the beginning of, and inside the other
                       (buf[:1].expand(4, 24), buf[1:5], True), (buf[:1].expand(4, 24), buf[:4], False),
                       (buf[2:3].expand(4, 24), buf[:4], False)):
        assert core._apart(a, b) is want and core._apart(b, a) is want


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100, 128])
def test_pack_mask(V):
    allowed = torch.rand(3, V, generator=torch.Generator().manual_seed(V)) < 0.5
    words = core.pack_mask(allowed)
    assert words.dtype == torch.int32 and tuple(words.shape) == (3, (V + 31) // 32)
    v = torch.arange(V)
    assert torch.equal(((words.long()[:, v // 32] >> (v % 32)) & 1).bool(), allowed)
    with pytest.raises(ValueError, match="boolean"):
        core.pack_mask(words)


@pytest.mark.parametrize("window", [1, 3, 8, 20])
def test_token_rules_start_lays_the_prompt_out_as_a_ring(window):
    B, T = 3, 11
    idx = torch.randint(0, 50, (B, T), generator=torch.Generator().manual_seed(window))
    rules = TokenRules(B, window, "cpu")
    for lengths in (None, torch.tensor([0, 4, 11])):
        rules.start(idx, lengths)
        n = [T] * B if lengths is None else lengths.tolist()
        assert rules.lengths.tolist() == n and rules.prompt.tolist() == n
        for b in range(B):
            for p in range(max(0, n[b] - window), n[b]):
                assert rules.tokens[b, p % window] == idx[b, p]
    with pytest.raises(ValueError, match="idx"):
        rules.start(idx[:2])
    with pytest.raises(ValueError, match="lengths"):
        rules.start(idx, torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="window"):
        TokenRules(2, 0, "cpu")


def test_model_embeds_on_the_cpu_as_before():
    """On the CPU the embedding is the module's; emb_scale scales it and leaves the tied head's table alone."""
    idx = torch.tensor([[1, 2, 3]])
    kw = dict(d=16, layers=1, mlp_f=16, mem=False, ffn="none", heads=4, n_sub=4, d_a=4, k=2)
    m = OneSdmLM(20, **kw)
    s = OneSdmLM(20, **kw, emb_scale=4.0)
    s.load_state_dict(m.state_dict(), strict=True)
    assert torch.equal(m.enfold(idx), m.emb(idx)) and torch.equal(s.enfold(idx), m.emb(idx) * 4.0)
