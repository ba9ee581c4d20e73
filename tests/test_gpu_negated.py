"""Lazily negated tensors (a bit that says that the values stand with the other sign; autograd hands such gradients over where a
real tensor became the imaginary part of a complex one that was conjugated): what is read has its sign, what would be written is
refused.  Everything here is exact, except for the training losses' gradients, which are compared with the call's own for the
same values in plain memory."""
import pytest
import torch

from sdmchat_amd import AdamW, core

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def negated(t):
    """t's values, lazily negated in memory."""
    n = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert n.is_neg() and torch.equal(n, t)
    return n


def dense_negated(t):
    """The same without gaps between the values."""
    n = torch._neg_view(-t)
    assert n.is_neg() and n.is_contiguous() and torch.equal(n, t)
    return n


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("what", ["logprob", "entropy", "both"])
def test_gradients_of_log_probabilities(rows, what):
    g = torch.Generator().manual_seed(rows)
    z, y = torch.randn(rows, 203, generator=g).cuda(), torch.randint(0, 203, (rows,), generator=g).cuda()
    w = [torch.randn(rows, generator=g).cuda() for _ in range(2)]
    got = []
    for through in (lambda t: t, lambda t: torch.complex(torch.zeros_like(t), t).conj().imag.neg()):
        x = z.clone().requires_grad_(True)
        r = core.token_logprobs(x, y, entropy=True)
        loss = sum((through(o) * v).sum() for o, v, name in zip((r.logprobs, r.entropy), w, ("logprob", "entropy"))
                   if what in (name, "both"))
        got.append(torch.autograd.grad(loss, x)[0])
    assert torch.equal(*got) and bool(got[0].any())
    for wrap in (negated, dense_negated):
        x = z.clone().requires_grad_(True)
        r = core.token_logprobs(x, y, entropy=True)
        outs = [(o, wrap(v)) for o, v, name in zip((r.logprobs, r.entropy), w, ("logprob", "entropy")) if what in (name, "both")]
        assert torch.equal(torch.autograd.grad([o for o, _ in outs], x, [v for _, v in outs])[0], got[0])


@pytest.mark.parametrize("lead", [(5,), (2, 3)])
def test_logits_of_log_probabilities(lead):
    z = torch.randn(*lead, 300, device="cuda")
    y = torch.randint(0, 300, lead, device="cuda")
    want = core.token_logprobs(z, y, entropy=True, top=4)
    for wrap in (negated, dense_negated):
        assert all(torch.equal(a, b) for a, b in zip(core.token_logprobs(wrap(z), y, entropy=True, top=4), want))
        grads = []
        for x in (z.clone().requires_grad_(True), wrap(z).detach().requires_grad_(True)):
            grads.append(torch.autograd.grad(core.token_logprobs(x, y).logprobs.sum(), x)[0])
        assert torch.equal(*grads)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 300])
def test_gradients_of_a_step(bits, n):
    gen = torch.Generator().manual_seed(n)
    p, g = torch.randn(n, generator=gen).cuda(), torch.randn(n, generator=gen).cuda()
    states = []
    for grad in (g, negated(g), dense_negated(g)):
        q = p.clone()
        st = ([torch.zeros_like(q)], [torch.zeros_like(q)]) if bits == 32 else ([core.new_moments(q)],)
        norm = core.adamw([q], [grad], *st, step=1, max_norm=0.5, **HYPER)
        states.append([q, norm, *(t for ts in st for t in ts)])
    for other in states[1:]:
        assert all(torch.equal(a, b) for a, b in zip(states[0], other))


def test_a_gradient_that_autograd_leaves_negated():
    """One value whose .grad keeps the bit: the optimiser moves it against its gradient."""
    out = []
    for through in (False, True):
        p = torch.nn.Parameter(torch.tensor([0.5], device="cuda"))
        loss = (torch.complex(torch.zeros_like(p), p).conj() * 1.25).sum().imag if through else (p * -1.25).sum()
        loss.backward()
        assert float(p.grad) == -1.25 and p.grad.is_neg() == through
        AdamW([p], lr=1e-2).step()
        out.append(p.detach())
    assert torch.equal(*out) and float(out[0]) > 0.5


def test_norms_and_rates():
    g = torch.randn(300, device="cuda")
    assert torch.equal(core.grad_norm([g]), core.grad_norm([negated(g)]))
    out = []
    for wrap in (lambda t: t, dense_negated):
        p = torch.ones(300, device="cuda")
        core.adamw([p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)], step=torch.zeros((), dtype=torch.int64, device="cuda"),
                   lr=wrap(torch.full((1,), 1e-2, device="cuda")), max_norm=1.0, norm=wrap(torch.full((1,), 3.0, device="cuda")))
        out.append(p)
    assert torch.equal(*out)


def test_what_would_be_written_is_refused():
    g = torch.randn(300, device="cuda")
    z = lambda: torch.zeros(300, device="cuda")  # noqa: E731
    n = lambda: dense_negated(torch.zeros(300, device="cuda"))  # noqa: E731
    s = core.new_moments(g)
    for call in (lambda: core.adamw([n()], [g], [z()], [z()], step=1), lambda: core.adamw([z()], [g], [n()], [z()], step=1),
                 lambda: core.adamw([z()], [g], [z()], [n()], step=1), lambda: core.adamw([n()], [g], [s], step=1),
                 lambda: core.read_moments([s], [n()], [z()]), lambda: core.read_moments([s], [z()], [n()])):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert not s.any()


def test_losses_and_embeddings():
    """The operators on token ids and vocabulary rows."""
    g = torch.Generator().manual_seed(1)
    table, dy = torch.randn(50, 16, generator=g).cuda(), torch.randn(7, 16, generator=g).cuda()
    idx = torch.randint(0, 50, (7,), generator=g).cuda()
    logits, ids, top = torch.randn(7, 50, generator=g).cuda(), torch.arange(21).view(7, 3).cuda(), torch.randn(7, 3, generator=g).cuda()
    bias = torch.randn(50, generator=g).cuda()
    for wrap in (negated, dense_negated):
        assert torch.equal(core.embedding(idx, wrap(table)), core.embedding(idx, table))
        assert torch.equal(core.embedding_backward(idx, wrap(dy), 50), core.embedding_backward(idx, dy, 50))
        assert torch.equal(core.distill_loss(wrap(logits), ids, wrap(top)), core.distill_loss(logits, ids, top))
        assert torch.equal(core.process_logits(wrap(logits), bias=wrap(bias)), core.process_logits(logits, bias=bias))
        grads = []
        for w in (lambda t: t, wrap):
            for reduction in ("mean", "none"):
                x = logits.clone().requires_grad_(True)
                loss = core.distill_loss(x, ids, top, reduction=reduction)
                grads.append(torch.autograd.grad(loss, x, w(torch.full(loss.shape, 0.7, device="cuda")))[0])
        assert torch.equal(grads[0], grads[2]) and torch.equal(grads[1], grads[3])
        with pytest.raises(ValueError, match="negated"):
            core.process_logits(logits, bias=bias, out=dense_negated(logits.clone()))


@pytest.mark.parametrize("wrap", [negated, dense_negated])
def test_norms_mixers_and_tables(wrap):
    """Their inputs and the gradients that come into them."""
    g = torch.Generator().manual_seed(2)
    x, w, dy = torch.randn(2, 5, 64, generator=g).cuda(), torch.rand(64, generator=g).cuda(), torch.randn(2, 5, 64, generator=g).cuda()
    assert torch.equal(core.rms_norm(wrap(x), w), core.rms_norm(x, w))
    assert all(torch.equal(a, b) for a, b in zip(core.rms_norm_backward(wrap(x), w, wrap(dy), 1e-6),
                                                 core.rms_norm_backward(x, w, dy, 1e-6)))
    H, dh, d_a, n = 2, 32, 16, 8
    kz, qz = (torch.randn(2, 5, H * d_a, generator=g).cuda() for _ in range(2))
    v, gate = torch.randn(2, 5, H * dh, generator=g).cuda(), torch.randn(2, 5, H, generator=g).cuda()
    k1, k2 = (torch.randn(H, n, d_a // 2, generator=g).cuda() for _ in range(2))
    scale, decay = torch.full((H,), 2.0).cuda(), torch.full((H,), 0.9).cuda()
    cfg = dict(k=4, read_mode="mean", out_norm=False, read_eps=1e-3, out_norm_eps=1e-2)
    table = torch.randn(H, n * n, dh, generator=g).cuda()
    grads = []
    for wr in (lambda t: t, wrap):
        ins = [t.clone().requires_grad_(True) for t in (kz, qz, v, gate, k1, k2)]
        r = core.SdmCoreFunction.apply(*ins, None, scale, decay, None, None, dict(cfg))
        one = torch.autograd.grad(r, ins, wr(dy))
        ins = [t.clone().requires_grad_(True) for t in (qz, k1, k2, scale, table)]
        r = core.TableSdmFunction.apply(*ins, dict(k=4))
        grads.append(one + torch.autograd.grad(r, ins, wr(dy)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    with pytest.raises(ValueError, match="negated"):
        core.core_forward(wrap(kz) if wrap is dense_negated else dense_negated(kz), qz, v, gate, keys1=k1, keys2=k2, log_scale=scale,
                          decay=decay, out_norm=False, k=4)
