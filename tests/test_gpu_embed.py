"""core.embedding and its gradient on the GPU against plain float64 sums, over sizes, types, strides and id streams, with
refusals, graphs and the model's training path.

Tolerances: the lookup is one float32 product and one rounding, equal bit for bit to torch's.  A gradient row of c terms is
a float32 sum in some order times the scale: at most (c + 2) 2^-24 of the sum of the terms' absolute values, plus the final
rounding of half a step (2^-9 or 2^-24 of twice the value: eps / 2)."""
import pytest
import torch

from sdmchat_amd import OneSdmLM, core
from tests._gpu_util import say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _ids(kind, n, V, g):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "zipf":
        r = torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * torch.log(torch.tensor(V + 1.0, dtype=torch.float64)))
        return r.long().clamp(1, V) - 1
    if kind == "one":   # one token all along
        return torch.full((n,), V // 2, dtype=torch.long)
    if kind == "bytes":   # few different ids
        return torch.randint(0, min(V, 256), (n,), generator=g)
    return torch.arange(n) % V   # "all": every row


def _want_grad(ids, dy, V, scale, pad):
    """The float64 gradient and the per-element bound of the kernel's error before its last rounding."""
    ids = ids.reshape(-1).clamp(0, V - 1)
    d64 = dy.double().cpu().reshape(ids.numel(), -1)
    if pad is not None:
        d64 = d64 * (ids != pad)[:, None]
    want = torch.zeros(V, d64.shape[1], dtype=torch.float64).index_add_(0, ids, d64) * scale
    mag = torch.zeros_like(want).index_add_(0, ids, d64.abs()) * abs(scale)
    c = torch.bincount(ids, minlength=V)[:, None]
    return want, (c + 2) * U * mag


def _check_grad(got, ids, dy, V, scale, pad=None):
    want, bound = _want_grad(ids, dy, V, scale, pad)
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double().cpu() - want).abs()
    tol = bound * (1 + half) + half * want.abs() + 1e-42
    assert bool((err <= tol).all()), f"{float((err - tol).max())} over the bound"


@pytest.mark.parametrize("N,V,d,kind", [
    (1, 1, 1, "one"), (1, 1000, 768, "uniform"), (63, 50, 7, "uniform"), (64, 32768, 768, "zipf"), (65, 513, 330, "zipf"),
    (777, 255, 64, "all"), (1000, 256, 100, "uniform"), (2048, 257, 768, "one"), (5003, 32003, 130, "zipf"),
    (4096, 5000, 1030, "bytes"), (16384, 32768, 768, "zipf"), (40000, 70000, 96, "zipf"), (3000, 600000, 8, "uniform"),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lookup_and_gradient(N, V, d, kind, dtype):
    g = torch.Generator().manual_seed(N + V + d)
    ids = _ids(kind, N, V, g)
    table = torch.randn(V, d, generator=g).to(dtype).cuda().requires_grad_(True)
    dy = torch.randn(N, d, generator=g).to(dtype).cuda()
    scale = 3.7
    say(f"[embed] N={N} V={V} d={d} {kind} {dtype}")
    y = core.embedding(ids.cuda(), table, scale)
    assert torch.equal(y, (table.detach()[ids.cuda()].float() * scale).to(dtype))
    y.backward(dy)
    _check_grad(table.grad, ids, dy, V, scale)
    again = core.embedding_backward(ids.cuda(), dy, V, scale)
    assert torch.equal(again, table.grad)   # deterministic


@pytest.mark.parametrize("pad", [0, 3, -1])
def test_padding_row_gets_no_gradient(pad):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 40, (6, 33), generator=g)
    ids[:, 20:] = pad % 40
    table = torch.randn(40, 24, generator=g).cuda().requires_grad_(True)
    dy = torch.randn(6, 33, 24, generator=g).cuda()
    y = core.embedding(ids.cuda(), table, 2.0, padding_idx=pad)
    assert torch.equal(y, table.detach()[ids.cuda()] * 2.0)
    y.backward(dy)
    assert not table.grad[pad].any()
    _check_grad(table.grad, ids, dy, 40, 2.0, pad % 40)


def test_padding_alone_gives_zeros():
    ids = torch.full((500,), 7, device="cuda")
    got = core.embedding_backward(ids, torch.randn(500, 16, device="cuda"), 9, 1.0, 7)
    assert not got.any()


@pytest.mark.parametrize("shape", [(0,), (2, 0), ()])
def test_no_tokens_and_one_token(shape):
    table = torch.randn(10, 12, device="cuda", requires_grad=True)
    ids = torch.zeros(shape, dtype=torch.long, device="cuda")
    y = core.embedding(ids, table)
    assert tuple(y.shape) == shape + (12,)
    y.sum().backward()
    want = torch.zeros(10, 12)
    want[0] = ids.numel()
    assert torch.equal(table.grad.cpu(), want)


def test_ids_outside_are_clamped():
    table = torch.randn(10, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([-1, -2 ** 62, 10, 2 ** 62, 4], device="cuda")
    y = core.embedding(ids, table)
    assert torch.equal(y, table.detach()[[0, 0, 9, 9, 4]])
    dy = torch.randn(5, 8, device="cuda")
    y.backward(dy)
    _check_grad(table.grad, ids.cpu(), dy, 10, 1.0)
    assert torch.equal(core.embedding(ids[-1:].int(), table.detach()), table.detach()[4:5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """Tables and gradients that are slices, transposed, repeated or start at an odd element."""
    g = torch.Generator().manual_seed(2)
    V, d, N = 50, 37, 200
    ids = torch.randint(0, V, (N,), generator=g)
    base = torch.randn(V, 64, generator=g).to(dtype).cuda()
    for table in (base[:, 3:3 + d], base.t()[:d, :V].t(), base[:1, 1:1 + d].expand(V, d), base[::2, 5:5 + d]):
        at = ids % table.shape[0]
        assert torch.equal(core.embedding(at.cuda(), table, 0.5), (table[at.cuda()].float() * 0.5).to(dtype))
    dbase = torch.randn(N, 64, generator=g).to(dtype).cuda()
    for dy in (dbase[:, 1:1 + d], dbase[:1, 3:3 + d].expand(N, d), torch.ones(1, 1, device="cuda", dtype=dtype).expand(N, d),
               torch.randn(64, N, generator=g).to(dtype).cuda()[:d].t()):
        _check_grad(core.embedding_backward(ids.cuda(), dy, V, 1.5), ids, dy, V, 1.5)
    assert torch.equal(core.embedding(ids.cuda()[::2], base), base[ids.cuda()[::2]])


def test_infinities_and_nan_stay_in_their_rows():
    ids = torch.tensor([1, 2, 2, 3, 2], device="cuda")
    dy = torch.ones(5, 40, device="cuda")
    dy[0] = float("inf")
    dy[3, 5] = float("nan")
    got = core.embedding_backward(ids, dy, 6).cpu()
    assert bool((got[1] == float("inf")).all()) and bool((got[2] == 3).all()) and not got[[0, 4, 5]].any()
    assert bool(got[3, 5].isnan()) and bool((got[3, 6:] == 1).all())


def test_twice_differentiable():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 9, (20,), generator=g).cuda()
    table = torch.randn(9, 5, generator=g).cuda().requires_grad_(True)
    w = torch.randn(20, 5, generator=g).cuda()
    for f in (lambda t: core.embedding(ids, t, 1.5, 4), lambda t: torch.nn.functional.embedding(ids, t, 4) * 1.5):
        gr, = torch.autograd.grad((f(table) ** 3 * w).sum(), table, create_graph=True)
        g2, = torch.autograd.grad((gr ** 2).sum(), table)
        if "first" not in locals():
            first = (gr.detach(), g2)
    # the same few float32 products and sums in another order: 20 terms of 2^-24 each, three times over
    for a, b in zip(first, (gr.detach(), g2)):
        assert float((a - b).abs().max()) <= 60 * U * float(b.abs().max())


@pytest.mark.parametrize("again", [False, True])
def test_nan_in_the_gradient_of_padding_is_not_read(again):
    ids = torch.tensor([1, 2, 2, 0, 2], device="cuda")
    table = torch.ones(4, 40, device="cuda", requires_grad=True)
    dy = torch.ones(5, 40, device="cuda")
    dy[[1, 2, 4]] = float("nan")
    got, = torch.autograd.grad(core.embedding(ids, table, 1.0, padding_idx=2), table, dy, create_graph=again)
    assert torch.equal(got.detach().cpu()[:, 0], torch.tensor([1.0, 1.0, 0.0, 0.0]))
    assert torch.equal(core.embedding_backward(ids, dy, 4, padding_idx=-2), got.detach())


@pytest.mark.parametrize("dtype,N,d", [(torch.bfloat16, 70001, 1024), (torch.float32, 66000, 514)])
def test_streams_larger_than_the_caches(dtype, N, d):
    """Outputs and gradients past 128 MiB take the kernels that pass the caches by."""
    V = 3001
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(0, V, (N,), generator=g, device="cuda")
    ids[: N // 3] = 17
    table = torch.randn(V, d, generator=g, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn(N, d, generator=g, device="cuda", dtype=dtype)
    y = core.embedding(ids, table, 0.5)
    assert torch.equal(y, (table.detach()[ids].float() * 0.5).to(dtype))
    y.backward(dy)
    want = torch.zeros(V, d, dtype=torch.float64, device="cuda").index_add_(0, ids, dy.double()) * 0.5
    mag = torch.zeros_like(want).index_add_(0, ids, dy.double().abs()) * 0.5
    c = torch.bincount(ids, minlength=V)[:, None]
    half = torch.finfo(dtype).eps / 2
    tol = (c + 2) * U * mag * (1 + half) + half * want.abs() + 1e-42
    assert bool(((table.grad.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("N", [255, 256, 257, 1023, 1024, 1025, 2049])
@pytest.mark.parametrize("d", [64, 65, 128, 129, 256, 257])
def test_sizes_around_tiles_and_slices(N, d):
    g = torch.Generator().manual_seed(N * d)
    for kind, V in (("zipf", 300), ("one", 9), ("bytes", 70000)):
        ids = _ids(kind, N, V, g)
        dy = torch.randn(N, d, generator=g)
        _check_grad(core.embedding_backward(ids.cuda(), dy.cuda(), V, 1.0), ids, dy, V, 1.0)


@pytest.mark.parametrize("N,V,d", [
    (5119, 300, 257), (5120, 9, 65), (5120, 300, 1028), (5121, 9, 65), (5121, 300, 257), (5121, 300, 3), (9217, 20000, 1),
    (10240, 257, 130), (5000, 262144, 9), (5000, 262145, 9), (255, 262145, 65), (1025, 300000, 2), (1, 300000, 64),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_around_one_launch(N, V, d, dtype):
    """Tokens and vocabularies on both sides of what one launch takes, with padding."""
    g = torch.Generator().manual_seed(N + V + d)
    for kind in ("zipf", "one"):
        ids = _ids(kind, N, V, g)
        pad = int(ids[0]) if kind == "zipf" else (int(ids[0]) + 1) % V
        dy = torch.randn(N, d, generator=g).to(dtype)
        _check_grad(core.embedding_backward(ids.cuda(), dy.cuda(), V, 1.3, pad), ids, dy, V, 1.3, pad)


@pytest.mark.parametrize("m", [1, 31, 32, 33, 64, 500])
@pytest.mark.parametrize("d", [1, 2, 5, 255, 256, 260, 4100, 5000])
def test_rows_of_few_and_many_tokens(m, d):
    """Rows of m tokens each, summed by one wave or by all of them, of fewer and more column slices than those."""
    g = torch.Generator().manual_seed(m + d)
    V = 1030
    rows = torch.tensor([0, 1, 255, 256, 257, 511, 512, 768, 1024])[:max(1, 4096 // m)]   # several of one bucket
    ids = rows.repeat(m)[torch.randperm(len(rows) * m, generator=g)]
    dy = torch.randn(len(ids), d, generator=g)
    _check_grad(core.embedding_backward(ids.cuda(), dy.cuda(), V, 1.0), ids, dy, V, 1.0)


def test_refusals():
    table = torch.randn(10, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    for args, text in (((ids.float(), table), "int64"), ((ids, table.half()), "float32 or bfloat16"), ((ids, table[0]), "vocab"),
                       ((ids.cpu(), table), "cpu"), ((ids, table, 1.0, 10), "padding_idx"), ((ids, table, 1.0, -11), "padding"),
                       ((ids, table[:0]), "vocab")):
        with pytest.raises(ValueError, match=text):
            core.embedding(*args)
    with pytest.raises(ValueError, match="padding_idx"):
        core.embedding_backward(ids, table[:3], 10, padding_idx=10)
    with pytest.raises(ValueError, match="dy"):
        core.embedding_backward(ids, table, 10)
    with pytest.raises(ValueError, match="float32"):
        core.embedding_backward(ids, table[:3].half(), 10)


def test_widths_past_32_bits_are_refused():
    """A width that 32 bits would cut to a small one is refused, not taken as that."""
    wide = torch.zeros(1, 1, device="cuda").expand(3, 2 ** 32 + 1)
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="limits"):
        core.embedding(ids, wide)
    with pytest.raises(ValueError, match="limits"):
        core.embedding_backward(ids, wide, 4)


def test_captured_training_step_replays():
    """Lookup and gradient in a captured graph, replayed on other tokens with eager work in between."""
    g = torch.Generator().manual_seed(5)
    V, d, N = 3000, 96, 2500
    table = torch.randn(V, d, generator=g).cuda().bfloat16()
    ids = torch.randint(0, V, (N,), generator=g).cuda()
    dy = torch.randn(N, d, generator=g).cuda().bfloat16()

    def step():
        t = table.detach().requires_grad_(True)
        y = core.embedding(ids, t, 2.0)
        return y.detach(), torch.autograd.grad(y, t, dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dt = step()
    for r in range(4):
        ids.copy_(torch.randint(0, V if r % 2 else 40, (N,), generator=g))
        dy.copy_(torch.randn(N, d, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        wy, wdt = step()
        assert torch.equal(y, wy) and torch.equal(dt, wdt), r


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(6)
    V, d, N = 20000, 256, 8000
    work = [(torch.randint(0, V, (N,), generator=g).cuda(), torch.randn(N, d, generator=g).cuda()) for _ in range(2)]
    want = [core.embedding_backward(i, dy, V) for i, dy in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [None, None]
    for _ in range(3):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[s] = core.embedding_backward(*work[s], V)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _model(**kw):
    torch.manual_seed(0)
    return OneSdmLM(97, d=64, layers=1, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4, **kw).cuda()


@pytest.mark.parametrize("scale", [1.0, 8.0])
def test_model_embeds_and_trains_on_it(scale):
    """OneSdmLM.enfold: the same embedded tokens as the module's, and the same gradients up to the order of their sums."""
    idx = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(7)).cuda()
    m, plain = _model(emb_scale=scale), _model(emb_scale=scale)
    plain.emb.register_forward_hook(lambda *a: None)   # a hooked embedding runs as the module it is
    with torch.no_grad():
        assert torch.equal(m.enfold(idx), m.emb(idx) * scale)
        assert torch.equal(m(idx), plain(idx))
    for mod in (m, plain):
        torch.nn.functional.cross_entropy(mod(idx)[:, :-1].flatten(0, 1), idx[:, 1:].flatten()).backward()
    assert type(m.enfold(idx).grad_fn).__name__.startswith("EmbeddingFunction")
    for (n, a), (_, b) in zip(m.named_parameters(), plain.named_parameters()):
        if n != "emb.weight":
            assert torch.equal(a.grad, b.grad), n
    # the embedding's part of the gradient: at most 80 terms of 2^-24 of a sum of magnitudes below 80 of the largest
    d = float((m.emb.weight.grad - plain.emb.weight.grad).abs().max())
    assert d <= 80 * U * 80 * float(plain.emb.weight.grad.abs().max())


def test_model_decode_with_a_scaled_embedding():
    idx = torch.randint(0, 97, (3, 6), generator=torch.Generator().manual_seed(8)).cuda()
    m = _model(emb_scale=4.0).eval()
    with torch.no_grad():
        want = m(idx)
        st = m.decode_state(3, "cuda")
        got = torch.stack([m.step(idx[:, t], st) for t in range(6)], 1)
    assert float((got - want).abs().max()) <= 1e-4 * max(1.0, float(want.abs().max()))
