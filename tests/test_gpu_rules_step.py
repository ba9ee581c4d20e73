"""OneSdmLM.step with rules that it has to refuse, on the GPU: nothing has moved, and the right call after it is as if it were
the first."""
import pytest
import torch

from sdmchat_amd import OneSdmLM, TokenRules, core
from tests.test_gpu_rules import check

pytestmark = pytest.mark.gpu
B, V = 3, 211


def _rules(**over):
    g = torch.Generator().manual_seed(4)
    kw = dict(repetition=1.0 + torch.rand(B, generator=g).cuda(), frequency=0.3, presence=0.2, bias=torch.randn(V, generator=g).cuda(),
              mask=core.pack_mask(torch.rand(B, V, generator=g) < 0.7).cuda())
    kw.update(over)
    return TokenRules(B, 6, "cuda", **kw)


def _model(**kw):
    torch.manual_seed(0)
    return OneSdmLM(V, **{**dict(d=64, layers=2, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4), **kw}).cuda().eval()


def _tensors(state, rules):
    out = [rules.tokens, rules.lengths, rules.prompt]
    for st in state.layers:
        out += [t for t in vars(st).values() if torch.is_tensor(t)]
    return out


BAD = {
    "bias of another vocabulary": dict(bias=torch.zeros(V - 1)), "bias of another type": dict(bias=torch.zeros(V).double()),
    "bias of another batch": dict(bias=torch.zeros(B + 1, V)), "mask of another vocabulary": dict(mask=torch.zeros(B, 6, dtype=torch.int32)),
    "mask of another type": dict(mask=torch.zeros(B, 7, dtype=torch.long)), "penalties of another batch": dict(frequency=torch.zeros(B + 1)),
    "penalties of whole numbers": dict(presence=torch.zeros(B, dtype=torch.long)), "no repetition": dict(repetition=0.0),
    "a penalty that is not a number": dict(presence=float("nan")),
}


@pytest.mark.parametrize("bad", list(BAD) + ["bias on the CPU", "history of another type", "tokens of two dimensions"])
def test_a_refused_step_has_moved_nothing(bad):
    m = _model()
    g = torch.Generator().manual_seed(5)
    toks = torch.randint(0, V, (4, B), generator=g).cuda()
    with torch.no_grad():
        state, rules, s2, r2 = m.decode_state(B, "cuda"), _rules(), m.decode_state(B, "cuda"), _rules()
        for t in range(2):
            assert torch.equal(m.step(toks[t], state, rules), m.step(toks[t], s2, r2))
        before = [t.clone() for t in _tensors(state, rules)]
        wrong, idx = _rules(), toks[2]
        if bad in BAD:
            wrong = _rules(**{k: v.cuda() if torch.is_tensor(v) else v for k, v in BAD[bad].items()})
        elif bad == "bias on the CPU":
            wrong.bias = wrong.bias.cpu()
        elif bad == "tokens of two dimensions":
            idx = toks[2][:, None]
        wrong.tokens, wrong.lengths, wrong.prompt = rules.tokens, rules.lengths, rules.prompt
        if bad == "history of another type":
            wrong.tokens = rules.tokens.int()
        with pytest.raises(ValueError):
            m.step(idx, state, wrong)
        assert state.pos == 2 and all(torch.equal(a, b) for a, b in zip(before, _tensors(state, rules)))
        for t in range(2, 4):
            assert torch.equal(m.step(toks[t], state, rules), m.step(toks[t], s2, r2))


def test_a_vocabulary_past_the_kernels_limits_is_refused_before_the_state_moves():
    big = (1 << 21) + 32
    m = _model(mem=False, ffn="none", layers=1, d=16, heads=4, d_a=4, tie=False)
    m.head = torch.nn.Linear(16, big, bias=False).cuda()
    state = m.decode_state(B, "cuda")
    with torch.no_grad(), pytest.raises(ValueError, match="limits"):
        m.step(torch.zeros(B, dtype=torch.long, device="cuda"), state, _rules(bias=None, mask=None))
    assert state.pos == 0


def test_a_projection_of_another_width():
    """A subclass whose logits are not one to a row of the embedding: the rules are checked against its own logits."""
    class Wider(OneSdmLM):
        def project(self, h):
            return torch.nn.functional.pad(super().project(h), (0, 21), value=1.0)
    torch.manual_seed(0)
    m = Wider(V, d=64, layers=1, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4).cuda().eval()
    rules = _rules(bias=torch.zeros(V + 21, device="cuda"), mask=None)
    idx = torch.arange(B, device="cuda")
    with torch.no_grad():
        raw = m.step(idx, m.decode_state(B, "cuda"))
        got = m.step(idx, m.decode_state(B, "cuda"), rules)
    check(dict(logits=raw.cpu(), tokens=idx.cpu()[:, None], lengths=torch.ones(B, dtype=torch.long), repetition=rules.repetition.cpu(),
               frequency=0.3, presence=0.2, bias=rules.bias.cpu()), got)


def test_float16_logits_of_an_autocast_step():
    """Under float16 autocast the logits are float16: the rules are applied in float32 and rounded to it."""
    m = _model(mem=False, layers=1)
    rules = _rules(mask=None)
    idx = torch.arange(B, device="cuda")
    with torch.no_grad(), torch.autocast("cuda", torch.float16):
        raw = m.step(idx, m.decode_state(B, "cuda"))
        got = m.step(idx, m.decode_state(B, "cuda"), rules)
    assert raw.dtype == got.dtype == torch.float16
    check(dict(logits=raw.cpu(), tokens=idx.cpu()[:, None], lengths=torch.ones(B, dtype=torch.long), repetition=rules.repetition.cpu(),
               frequency=0.3, presence=0.2, bias=rules.bias.cpu()), got)


def test_rules_of_a_class_of_ones_own():
    """append and apply of a subclass, or of any object with them, are the ones that step calls."""
    class Loud(TokenRules):
        def append(self, idx_t):
            super().append(idx_t + 1)

        def apply(self, logits, out=None):
            return super().apply(logits, out=out).neg_()

    class Other:
        tokens = torch.zeros(B, 1)

        def append(self, idx_t):
            self.seen = idx_t

        def apply(self, logits, out=None):
            return logits + 1
    m, idx = _model(), torch.arange(B, device="cuda")
    with torch.no_grad():
        raw = m.step(idx, m.decode_state(B, "cuda"))
        rules = Loud(B, 4, "cuda", bias=torch.ones(V, device="cuda"))
        assert torch.equal(m.step(idx, m.decode_state(B, "cuda"), rules), -(raw + 1)) and rules.tokens[:, 0].tolist() == [1, 2, 3]
        other = Other()
        assert torch.equal(m.step(idx, m.decode_state(B, "cuda"), other), raw + 1) and other.seen is idx
