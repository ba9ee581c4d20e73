"""core.process_logits, core.append_tokens, TokenRules and their place in OneSdmLM.step and DecodeGraph, on the GPU against
plain float64.

Tolerance: the rules are at most five float32 operations on a value (divide or multiply, count times frequency plus presence
with one rounding, subtract, add), each off by 2^-24 of its result, and one rounding to the logits' type (eps / 2)."""
import pytest
import torch

from sdmchat_amd import DecodeGraph, OneSdmLM, TokenRules, core
from tests._gpu_util import say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def make(B, V, L, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(B, V, generator=g) * scale).to(dtype)
    tokens = torch.randint(0, max(1, min(V, 3 * L)), (B, L), generator=g)
    lengths = torch.randint(0, L + 1, (B,), generator=g)
    lengths[0] = L
    prompt = (lengths * torch.rand(B, generator=g)).long()
    rep = 1 + torch.rand(B, generator=g)
    rep[0] = 0.7
    return dict(logits=z, tokens=tokens, lengths=lengths, prompt=prompt, repetition=rep, frequency=torch.randn(B, generator=g),
                presence=torch.randn(B, generator=g), bias=torch.randn(V, generator=g) * 2,
                mask=core.pack_mask(torch.rand(B, V, generator=g) < 0.6))


def history(a, b):
    """The tokens of stream b with their positions."""
    L, n = a["tokens"].shape[1], int(a["lengths"][b])
    return [(p, int(a["tokens"][b, p % L])) for p in range(max(0, n - L), n)]


def reference(a):
    z = a["logits"].double()
    B, V = z.shape
    mag = z.abs()

    def per_row(name, default, b):
        v = a.get(name, default)
        return float(v) if not torch.is_tensor(v) else float(v.double().expand(B)[b] if v.dim() else v)
    for b in range(B):
        r, f, pr = per_row("repetition", 1.0, b), per_row("frequency", 0.0, b), per_row("presence", 0.0, b)
        seen, count = torch.zeros(V, dtype=torch.bool), torch.zeros(V, dtype=torch.float64)
        if a.get("tokens") is not None:
            start = 0 if a.get("prompt") is None else int(a["prompt"][b])
            for p, t in history(a, b):
                if 0 <= t < V:
                    seen[t] = True
                    count[t] += p >= start
        x = z[b]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        mag[b] = torch.maximum(mag[b], x.abs())
        minus = torch.where(count > 0, count * f + pr, 0.0)
        x = x - minus
        mag[b] += (count * f).abs() + abs(pr) * (count > 0) + minus.abs()
        if a.get("bias") is not None:
            bias = a["bias"].double() if a["bias"].dim() == 1 else a["bias"][b].double()
            x = x + bias
            mag[b] += bias.abs()
        if a.get("mask") is not None:
            words = (a["mask"] if a["mask"].dim() == 1 else a["mask"][b]).long()
            v = torch.arange(V)
            x = torch.where(((words[v // 32] >> (v % 32)) & 1).bool(), x, -INF)
        z[b] = x
    return z, mag


def check(a, got):
    want, mag = reference(a)
    got = got.double().cpu()
    fin = want.isfinite()
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    assert torch.equal(got.isnan(), want.isnan())
    half = torch.finfo(a["logits"].dtype).eps / 2
    err, tol = (got - want).abs()[fin], (6 * U * mag * (1 + half) + half * want.abs())[fin]
    assert bool((err <= tol).all()), float((err - tol).max())


def call(a, **over):
    kw = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in {**a, **over}.items()}
    return core.process_logits(kw.pop("logits"), kw.pop("tokens", None), kw.pop("lengths", None), **kw)


@pytest.mark.parametrize("B,V,L", [
    (1, 1, 1), (2, 31, 5), (3, 32, 40), (5, 33, 64), (4, 1000, 100), (1, 2048, 300), (2, 2049, 513), (64, 4096, 200), (7, 32003, 1500),
    (1, 32768, 9000), (40, 32768, 700), (9, 131071, 3000), (300, 5001, 50),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rules(B, V, L, dtype):
    say(f"[rules] B={B} V={V} L={L} {dtype}")
    a = make(B, V, L, dtype, B + V + L)
    check(a, call(a))


@pytest.mark.parametrize("rules", [(), ("tokens",), ("tokens", "repetition"), ("tokens", "prompt", "frequency"), ("tokens", "presence"),
                                   ("bias",), ("mask",), ("bias", "mask")])
def test_rules_apart(rules):
    a = make(6, 777, 90, torch.float32, 3)
    keep = {"logits", *rules} | ({"lengths"} if "tokens" in rules else set())
    a = {k: v for k, v in a.items() if k in keep}
    got = call(a)
    check(a, got)
    if rules in ((), ("tokens",)):
        assert torch.equal(got.cpu(), a["logits"])


def test_numbers_and_shared_rows():
    a = make(5, 300, 40, torch.bfloat16, 4)
    a.update(repetition=1.3, frequency=0.25, presence=torch.tensor(0.5), mask=a["mask"][1])
    check(a, call(a))
    a["bias"] = torch.randn(5, 300, generator=torch.Generator().manual_seed(1))
    check(a, call(a))


def test_empty_histories_and_batches():
    a = make(4, 100, 8, torch.float32, 5)
    a["lengths"].zero_()
    check(a, call(a))
    a["lengths"].fill_(-3)   # nothing of the history counts
    assert torch.equal(call(a), call(a, lengths=torch.zeros(4, dtype=torch.long)))
    a["tokens"] = torch.zeros(4, 0, dtype=torch.long)
    check(dict(a, lengths=torch.zeros(4, dtype=torch.long)), call(a))
    none = torch.zeros(0, 100, device="cuda")
    assert tuple(core.process_logits(none, torch.zeros(0, 3, dtype=torch.long, device="cuda"),
                                     torch.zeros(0, dtype=torch.long, device="cuda"), repetition=2.0).shape) == (0, 100)


def test_ids_outside_the_vocabulary_count_nowhere():
    a = make(3, 50, 30, torch.float32, 6)
    a["tokens"][:, ::3] = -1
    a["tokens"][:, 1::3] = 50
    a["tokens"][0, 2] = 2 ** 62
    a["tokens"][1, 2] = -2 ** 62
    a["tokens"][2, 2] = 2 ** 32 + 7   # not token 7
    check(a, call(a))


def test_ring_of_the_last_tokens():
    a = make(6, 60, 16, torch.float32, 7)
    a["lengths"] = torch.tensor([16, 17, 31, 32, 1000, 5])
    a["prompt"] = torch.tensor([3, 17, 20, 16, 990, 2])
    check(a, call(a))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_nan_and_rows_that_allow_nothing(dtype):
    a = make(5, 200, 30, dtype, 8)
    z = a["logits"]
    z[0, :50] = -INF
    z[1, :50] = torch.finfo(dtype).min
    z[2, 10], z[2, 11] = INF, float("nan")
    z[3, :50] = float("nan")
    a["bias"][5] = -INF
    a["bias"][6] = INF
    z[4, 6] = 1.0
    allowed = torch.rand(5, 200, generator=torch.Generator().manual_seed(2)) < 0.5
    allowed[3, :50] = False   # NaN where nothing is allowed
    allowed[4] = False        # a row that allows nothing
    a["mask"] = core.pack_mask(allowed)
    a["repetition"], a["frequency"], a["presence"] = 1.5, 0.5, 0.25
    got = call(a)
    want, _ = reference(a)
    want = want.to(dtype).double()
    assert torch.equal(got.cpu().isnan(), want.isnan())
    assert torch.equal(got.double().cpu() == -INF, want == -INF) and torch.equal(got.double().cpu() == INF, want == INF)
    assert bool((got[4] == -INF).all()) and not got[3].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_alignment_and_in_place(dtype):
    a = make(6, 501, 33, dtype, 9)
    want = call(a)
    wide = torch.zeros(6, 1600, dtype=dtype, device="cuda")
    z = wide[:, 3:504]
    z.copy_(a["logits"])
    got = call(a, logits=z)
    assert torch.equal(got, want)
    before = wide.clone()
    out = wide[:, 1001:1502]   # other columns of the same buffer
    assert call(a, logits=z, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want) and torch.equal(wide[:, :1001], before[:, :1001]) and torch.equal(wide[:, 1502:], before[:, 1502:])
    call(a, logits=z, out=z)
    assert torch.equal(z, want) and torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 504:1001], before[:, 504:1001])
    assert torch.equal(call(a, logits=a["logits"].t().contiguous().cuda().t()), want)
    assert torch.equal(call(a, tokens=a["tokens"].t().contiguous().cuda().t(), mask=a["mask"].t().contiguous().cuda().t()), want)
    row = a["logits"][:1].cuda().expand(6, 501)
    assert torch.equal(call(a, logits=row), call(a, logits=row.contiguous()))
    one = a["tokens"][:1].expand(6, 33)
    assert torch.equal(call(a, tokens=one.cuda()), call(a, tokens=one.contiguous()))


def test_refusals():
    a = {k: v.cuda() for k, v in make(4, 100, 8, torch.float32, 10).items()}
    z = a["logits"]
    for over, text in ((dict(logits=z.half()), "float32 or bfloat16"), (dict(logits=z[0]), "vocab"), (dict(tokens=a["tokens"].int()), "int64"),
                       (dict(tokens=a["tokens"][:3]), "tokens"), (dict(lengths=None), "lengths"), (dict(lengths=a["lengths"][:3]), "lengths"),
                       (dict(prompt=a["prompt"].float()), "prompt"), (dict(repetition=0.0), "repetition"), (dict(repetition=INF), "finite"),
                       (dict(frequency=float("nan")), "finite"), (dict(presence=a["presence"][:3]), "presence"),
                       (dict(presence=a["prompt"]), "presence"), (dict(bias=a["bias"][:99]), "bias"), (dict(bias=a["bias"].double()), "bias"),
                       (dict(mask=a["mask"][:, :3]), "mask"), (dict(mask=a["mask"].long()), "mask"), (dict(out=z[:3]), "out"),
                       (dict(out=z.bfloat16()), "out"), (dict(tokens=None, prompt=None), "need tokens")):
        with pytest.raises(ValueError, match=text):
            call(a, **over)
    with pytest.raises(ValueError, match="cpu"):
        core.process_logits(z, bias=a["bias"].cpu())
    with pytest.raises(RuntimeError, match="inference"):
        core.process_logits(z.clone().requires_grad_(True))
    buf = torch.zeros(5, 100, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        core.process_logits(buf[:4], out=buf[1:])
    with pytest.raises(ValueError, match="int64"):
        core.append_tokens(a["tokens"], a["lengths"], a["lengths"].int())
    with pytest.raises(ValueError, match="int64"):
        core.append_tokens(a["tokens"], a["lengths"], a["lengths"][:3])
    with pytest.raises(ValueError, match="contiguous"):
        core.append_tokens(a["tokens"].t().contiguous().t(), a["lengths"], a["lengths"])


def test_a_vocabulary_past_32_bits_is_refused():
    with pytest.raises(ValueError, match="limits"):
        core.process_logits(torch.zeros(1, 1, device="cuda").expand(2, 2 ** 32 + 1))


def test_append_tokens():
    B, width = 300, 5
    g = torch.Generator().manual_seed(11)
    wide = torch.full((B, width + 3), -7)
    tokens, lengths = wide.cuda()[:, 1:1 + width], torch.randint(0, 9, (B,), generator=g).cuda()
    want, n = wide.clone()[:, 1:1 + width], lengths.cpu().clone()
    for s in range(7):
        new = torch.randint(0, 99, (B,), generator=g)
        core.append_tokens(tokens, lengths, new.cuda())
        want[torch.arange(B), n % width] = new
        n += 1
    assert torch.equal(tokens.cpu(), want) and torch.equal(lengths.cpu(), n)
    assert bool((tokens._base[:, 0] == -7).all()) and bool((tokens._base[:, 1 + width:] == -7).all())


def _model(V=211):
    torch.manual_seed(0)
    return OneSdmLM(V, d=64, layers=2, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4).cuda().eval()


def _rules(B, V, window=6):
    g = torch.Generator().manual_seed(4)
    return TokenRules(B, window, "cuda", repetition=1.0 + torch.rand(B, generator=g).cuda(), frequency=0.3, presence=0.2,
                      bias=torch.randn(V, generator=g).cuda(), mask=core.pack_mask(torch.rand(B, V, generator=g) < 0.7).cuda())


def test_decode_loop_with_rules():
    """prefill, start, then steps: every step's logits are the plain step's with the rules of the tokens so far."""
    B, V, T, steps = 3, 211, 9, 12
    m, rules = _model(V), _rules(B, V)
    idx = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(5)).cuda()
    with torch.no_grad():
        logits, state = m.prefill(idx)
        _, plain = m.prefill(idx)
        rules.start(idx)
        last = logits[:, -1].clone()
        nxt = rules.apply(logits[:, -1]).argmax(-1)
        assert torch.equal(last, logits[:, -1])   # a new tensor unless asked
        said = idx.cpu()
        for _ in range(steps):
            raw = m.step(nxt, plain)
            got = m.step(nxt, state, rules)
            said = torch.cat([said, nxt.cpu()[:, None]], 1)
            L = said.shape[1]
            a = dict(logits=raw.cpu(), tokens=said[:, -6:], lengths=torch.full((B,), min(L, 6)), prompt=torch.full((B,), T - (L - 6)),
                     repetition=rules.repetition.cpu(), frequency=0.3, presence=0.2, bias=rules.bias.cpu(), mask=rules.mask.cpu())
            check(a, got)
            nxt = got.argmax(-1)
            allowed = (rules.mask.cpu().long()[torch.arange(B), nxt.cpu() // 32] >> (nxt.cpu() % 32)) & 1
            assert bool(allowed.all())
    assert rules.lengths.tolist() == [T + steps] * B and state.pos == T + steps


def test_step_with_rules_of_another_batch_or_outside_no_grad():
    """Rules of another batch are refused before the streams' state moves, and so is a step of the mixers outside no_grad;
    a model without mixers steps there too, to logits without a gradient."""
    m, B, V = _model(211), 3, 211
    toks = torch.arange(B).cuda()
    state, rules = m.decode_state(B, "cuda"), _rules(B, V)
    with torch.no_grad(), pytest.raises(ValueError, match="streams"):
        m.step(toks, state, _rules(B + 1, V))
    with pytest.raises(RuntimeError, match="inference"):
        m.step(toks, state, rules)
    assert state.pos == 0 and rules.lengths.tolist() == [0] * B
    torch.manual_seed(1)
    m = OneSdmLM(V, d=64, layers=1, mlp_f=64, mem=False).cuda().eval()
    got = m.step(toks, m.decode_state(B, "cuda"), rules)
    with torch.no_grad():
        want = m.step(toks, m.decode_state(B, "cuda"), _rules(B, V))
    assert torch.equal(got, want) and not got.requires_grad


@pytest.mark.parametrize("steps", [1, 3])
def test_decode_graph_with_rules(steps):
    """The captured steps with rules equal the eager ones bit for bit, and read a mask that changes between replays."""
    B, V = 4, 211
    m = _model(V)
    g = torch.Generator().manual_seed(6)
    with torch.no_grad():
        s1, s2 = m.decode_state(B, "cuda"), m.decode_state(B, "cuda")
        r1, r2 = _rules(B, V), _rules(B, V)
        graph = DecodeGraph(m, s1, steps=steps, rules=r1)
        assert r1.lengths.tolist() == [0] * B   # capture appended nothing
        for rep in range(4):
            toks = torch.randint(0, V, (steps, B), generator=g).cuda()
            mask = core.pack_mask(torch.rand(B, V, generator=g) < 0.7).cuda()
            r1.mask.copy_(mask)
            r2.mask.copy_(mask)
            got = graph.run(toks if steps > 1 else toks[0])
            want = [m.step(toks[t], s2, r2) for t in range(steps)]
            torch.cuda.synchronize()
            assert torch.equal(got, torch.stack(want) if steps > 1 else want[0]), rep
        assert torch.equal(r1.tokens, r2.tokens) and torch.equal(r1.lengths, r2.lengths)


def test_training_step_and_decode_together():
    """The three operators in one program: a distillation step through embedding and loss, then a decode with rules."""
    V, B = 211, 2
    torch.manual_seed(1)
    m = OneSdmLM(V, d=64, layers=1, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4, emb_scale=8.0).cuda()
    g = torch.Generator().manual_seed(7)
    idx = torch.randint(0, V, (B, 30), generator=g).cuda()
    with torch.no_grad():
        teacher = torch.randn(B, 30, V, generator=g).cuda()
    top, ids = teacher.topk(8)
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    for _ in range(2):
        opt.zero_grad()
        m.distill_loss(idx, ids, top, labels=ids[..., 0], alpha=0.5, temperature=2.0).backward()
        assert all(p.grad is None or bool(p.grad.isfinite().all()) for p in m.parameters())
        assert bool(m.emb.weight.grad.any())
        opt.step()
    m.eval()
    rules = _rules(B, V)
    with torch.no_grad():
        logits, state = m.prefill(idx)
        rules.start(idx)
        nxt = rules.apply(logits[:, -1]).argmax(-1)
        for _ in range(3):
            nxt = m.step(nxt, state, rules).argmax(-1)
    assert rules.lengths.tolist() == [33] * B
