"""core.token_logprobs and its gradient on the GPU against the definitions in float64.

Tolerances, with U = 2^-24, a_j = (max - z_j) / temperature and c the length of a chain of sums (a thread's part of a row and
the joins after it): a difference z_j - max is rounded once, its product with the constant of the temperature once, the constant
carries three roundings more, and the exponential is off by its last place, so 2^e is off by U (5 a_j + 4) relative; a sum of
them over S by s = U (sum_j p_j (5 a_j + 4) + c).  A log probability is a_target (3 U relative) and the logarithm of S (s, and 4 U
of its size), rounded; the entropy the logarithm and sum_j p_j a_j, whose terms are off by U (5 a_j + 8 + 2 c) relative.  p_j =
2^(e_j - log2 S) is off by r_j = U (5 a_j + 8) + 4 U log S + s relative, and a gradient by that and 6 U of each of its terms,
the entropy's part by its l_j + H too, and its last rounding (eps / 2)."""
import math

import pytest
import torch

from sdmchat_amd import OneSdmLM, core
from tests._gpu_util import say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FAR = 200.0   # from here on exp(-a) is nothing


def chain(V):
    return V / 64 + 24


def reference(z, y, tau, k, ignore=-100):
    """The definitions on the CPU in float64 with their bounds; rows hold no NaN or +inf."""
    N, V = z.shape
    z = z.double()
    m = z.amax(1, keepdim=True)
    empty = (m == -math.inf)[:, 0]
    a = torch.where(z > -math.inf, (torch.where(m > -math.inf, m, 0.0) - z) / tau, math.inf)
    p = torch.exp(-a)
    S = torch.where(empty, 1.0, p.sum(1))
    p = p / S[:, None]
    log_s = torch.log(S)
    af = a.clamp(max=FAR)
    l = -a - log_s[:, None]
    s = U * ((p * (5 * af + 4)).sum(1) + chain(V))
    out = dict(p=p, l=l, a=af, log_s=log_s, s=s, empty=empty)
    given = torch.zeros(N, dtype=torch.bool) if y is None else (y >= 0) & (y < V) & (y != ignore)
    out["given"] = given
    if y is not None:
        at = torch.where(given, y, 0)[:, None]
        lp = torch.where(empty, -math.inf, l.gather(1, at)[:, 0])
        out["logprobs"] = torch.where(given, lp, 0.0)
        size = torch.where(lp > -math.inf, -lp, 0.0)
        out["logprobs_b"] = 3 * U * a.gather(1, at)[:, 0].clamp(max=3e38) + s + 4 * U * log_s + 2 * U * size
    fl = torch.where(p > 0, l, 0.0)
    out["entropy"] = torch.where(empty, 0.0, -(p * fl).sum(1))
    out["entropy_b"] = s + 4 * U * log_s + U * (p * af * (5 * af + 8 + 2 * chain(V))).sum(1) + 2 * U * out["entropy"]
    if k:
        v, ids = torch.sort(z, dim=1, descending=True, stable=True)
        v, ids = v[:, :k], ids[:, :k]
        there = v > -math.inf
        lt = l.gather(1, ids)
        b = 3 * U * torch.where(there, a.gather(1, ids), 0.0) + (s + 4 * U * log_s)[:, None] + 2 * U * torch.where(there, -lt, 0.0)
        fill = k - v.shape[1]
        pad = torch.nn.functional.pad
        out["top_ids"] = pad(torch.where(there, ids, -1), (0, fill), value=-1)
        out["top_logprobs"] = pad(torch.where(there, lt, -math.inf), (0, fill), value=-math.inf)
        out["top_logprobs_b"] = pad(b, (0, fill))
    return out


def near(got, want, bound, what):
    got = got.double().cpu()
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and not got.isnan().any(), what
    d = torch.where(inf, 0.0, (got - want).abs())
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert bool((d <= bound).all()), (what, worst)
    return worst


def check(z, y, tau=1.0, k=0, entropy=True, ignore=-100):
    with torch.no_grad():
        r = core.token_logprobs(z.cuda(), None if y is None else y.cuda(), temperature=tau, entropy=entropy, top=k,
                                ignore_index=ignore)
    w = reference(z, y, tau, k, ignore)
    worst = []
    if y is not None:
        worst.append(near(r.logprobs, w["logprobs"], w["logprobs_b"], "logprobs"))
    if entropy:
        worst.append(near(r.entropy, w["entropy"], w["entropy_b"], "entropy"))
    if k:
        assert torch.equal(r.top_ids.cpu(), w["top_ids"])
        worst.append(near(r.top_logprobs, w["top_logprobs"], w["top_logprobs_b"], "top_logprobs"))
    return r, w, worst


def check_grad(z, y, tau, dlp, dh, ignore=-100):
    x = z.cuda().requires_grad_(True)
    r = core.token_logprobs(x, None if y is None else y.cuda(), temperature=tau, entropy=dh is not None, ignore_index=ignore)
    outs = [(o, g.cuda()) for o, g in ((r.logprobs, dlp), (r.entropy, dh)) if g is not None]
    got, = torch.autograd.grad([o for o, _ in outs], x, [g for _, g in outs])
    assert got.dtype == z.dtype and got.shape == z.shape
    w = reference(z, y, tau, 0, ignore)
    zero = torch.zeros(z.shape[0], dtype=torch.float64)
    gl = zero if dlp is None else torch.where(w["given"], dlp.double(), 0.0)
    ge = zero if dh is None else dh.double()
    hot = torch.zeros_like(w["p"])
    if y is not None:
        hot[torch.arange(z.shape[0]), torch.where(w["given"], y, 0)] = w["given"].double()
    lh = torch.where(w["p"] > 0, w["l"] + w["entropy"][:, None], 0.0)
    want = (gl[:, None] * (hot - w["p"]) - ge[:, None] * w["p"] * lh) / tau
    want[w["empty"]] = 0.0
    rel = U * (5 * w["a"] + 8) + (4 * U * w["log_s"] + w["s"])[:, None]
    l_err = 3 * U * w["a"] + (4 * U * w["log_s"] + w["s"] + w["entropy_b"])[:, None]
    size = w["p"] * (gl.abs()[:, None] + ge.abs()[:, None] * (w["l"].abs().clamp(max=FAR + 50) + w["entropy"][:, None]))
    bound = ((rel + 6 * U) * size + w["p"] * ge.abs()[:, None] * l_err + 6 * U * gl.abs()[:, None] * hot) / tau
    bound = bound + torch.finfo(z.dtype).eps / 2 * want.abs() + 1e-37
    return near(got, want, bound, "grad"), got


def make(N, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V, generator=g) * spread).to(dtype)
    y = torch.randint(0, V, (N,), generator=g)
    if N > 2:
        y[1] = -100
        y[2] = V
    return z, y, g


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 64, 65, 511, 1000, 1024, 1025, 2049, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 1, 5, 256])
def test_small_vocabularies(V, dtype, k):
    z, y, _ = make(5, V, dtype, V + k)
    say(V, dtype, k, check(z, y, 0.8, k)[2])


@pytest.mark.parametrize("N,V", [(3, 8192), (2, 16385), (3, 32767), (3, 32768), (3, 32769), (2, 50257), (2, 65536), (2, 65543),
                                 (2, 151936), (1, 300001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 20, 200])
def test_wide_rows(N, V, dtype, k):
    z, y, _ = make(N, V, dtype, V + k, 1.5)
    say(V, dtype, k, check(z, y, 1.3, k)[2])


@pytest.mark.parametrize("N", [1, 17, 300, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(N, dtype):
    z, y, _ = make(N, 1003, dtype, N)
    check(z, y, 1.0, 7)


@pytest.mark.parametrize("V", [777, 5000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [3, 64, 256])
def test_ties_and_crowded_alternatives(V, dtype, k):
    """Equal logits in any number, the best ones next to each other, rising and falling rows, zeros of both signs."""
    rows = [torch.zeros(V), torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), torch.arange(V).float() / 64,
            -torch.arange(V).float() / 64, torch.full((V,), -3.0), (torch.arange(V) % 3).float(), (torch.arange(V) % 97).float() / 8]
    rows[4][V // 2:V // 2 + 300] = torch.arange(300)[:V - V // 2].float() / 16
    a = torch.randn(V, generator=torch.Generator().manual_seed(V))
    a[V - 290:] = a[V - 290:].abs() + 8
    rows.append(a)
    b = torch.full((V,), 1.0)
    b[::5] = 2.0
    rows.append(b)
    z = torch.stack(rows).to(dtype)
    y = torch.arange(len(rows)) * 11
    say(check(z, y, 1.0, k)[2])


@pytest.mark.parametrize("V,k", [(300001, 256), (1 << 21, 100), (1 << 21, 256), (1 << 21, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_widest_rows(V, k, dtype):
    """As many slices as there can be, with more keys in them than the join holds in LDS."""
    z, y, _ = make(2, V, dtype, V + k, 1.5)
    say(V, dtype, k, check(z, y, 1.1, k)[2])


@pytest.mark.parametrize("V", [130, 900, 1500, 6000, 33000, 70000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [20, 100, 256])
def test_coarse_logits_and_counts_around_k(V, dtype, k):
    """Few different values, in any order; rows that leave k - 1, k and k + 1 tokens, spread or side by side; all but a few values
    of one size."""
    g = torch.Generator().manual_seed(V + k)
    rows = [(torch.randn(V, generator=g) * 1.5).round(), (torch.randn(V, generator=g) * 3).round() / 2 - 9,
            torch.randint(0, 2, (V,), generator=g).float(), torch.randn(V, generator=g) * 0.02 + 5, torch.randn(V, generator=g) * 0.02 - 5]
    for left in (k - 1, k, k + 1):
        for spread in (True, False):
            x = torch.full((V,), -math.inf)
            at = torch.randperm(V, generator=g)[:left] if spread else torch.arange(V)[V // 3:V // 3 + left]
            x[at] = torch.randn(len(at), generator=g)
            rows.append(x)
    x = torch.zeros(V)
    x[torch.randperm(V, generator=g)[:max(1, k // 2)]] = 1.0
    rows += [x, -x]
    z = torch.stack(rows).to(dtype)
    y = torch.arange(len(rows)) * 7
    say(check(z, y, 1.0, k)[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [10, 2100, 40001])
def test_masked_rows(dtype, V):
    """-inf anywhere: fewer tokens left than alternatives asked, one, none; the type's lowest value beside them."""
    z, y, g = make(7, V, dtype, V)
    low = torch.finfo(dtype).min
    z[0, torch.rand(V, generator=g) < 0.7] = -math.inf
    z[0, 3] = 1.0
    z[1] = -math.inf
    z[2] = -math.inf
    z[2, V // 2] = -5.0
    z[3] = low
    z[4] = low
    z[4, V - 1] = low / 2
    z[5] = -math.inf
    z[5, V - 3:] = torch.tensor([1.0, 2.0, 2.0]).to(dtype)
    y = torch.tensor([3, 4, V // 2, 0, V - 1, 0, 5])
    r, w, _ = check(z, y, 1.0, 9)
    assert r.logprobs[1] == -math.inf and r.logprobs[2] == 0 and r.logprobs[5] == -math.inf and r.entropy[1] == 0
    assert r.top_ids[1].tolist() == [-1] * 9 and r.top_ids[5].tolist() == [V - 2, V - 1, V - 3] + [-1] * 6
    dlp, dh = torch.randn(7, generator=g), torch.randn(7, generator=g)
    dh[3:5] = 0   # l_j itself is -1e38 there
    _, grad = check_grad(z, y, 1.0, dlp, dh)
    assert not grad[1].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50, 40001])
def test_nan_and_infinity(dtype, V):
    z, y, g = make(6, V, dtype, 3)
    clean = z.clone()
    z[0, V // 3] = math.nan
    z[2, 0] = math.inf
    z[4] = math.nan
    y = torch.tensor([1, 2, 0, 3, 4, -100])
    with torch.no_grad():
        r = core.token_logprobs(z.cuda(), y.cuda(), entropy=True, top=4)
    bad = torch.tensor([True, False, True, False, True, False])
    assert torch.equal(r.logprobs.isnan().cpu(), bad) and torch.equal(r.entropy.isnan().cpu(), bad)
    assert torch.equal(r.top_logprobs.isnan().all(1).cpu(), bad) and bool((r.top_ids[bad.cuda()] == -1).all())
    w = reference(clean, y, 1.0, 4)
    assert torch.equal(r.top_ids.cpu()[~bad], w["top_ids"][~bad])
    assert bool(((r.logprobs.cpu().double() - w["logprobs"]).abs() <= w["logprobs_b"])[~bad].all())
    # a row that counts for nothing has gradient 0 whatever it holds
    x = z.cuda().requires_grad_(True)
    r = core.token_logprobs(x, y.cuda(), entropy=True)
    keep = (~bad).float().cuda()
    keep[5] = 0
    grad, = torch.autograd.grad([r.logprobs, r.entropy], x, [keep, keep])
    assert not grad[bad.cuda()].any() and not grad[5].any() and bool(grad[1].any()) and not grad.isnan().any()


@pytest.mark.parametrize("dtype,patterns", [(torch.float32, [0x7fc00000, 0xffc00000, 0x7f800001, 0x7fffffff, 0xffffffff, 0xfff00001]),
                                            (torch.bfloat16, [0x7fc0, 0xffc0, 0x7f81, 0x7fff, 0xffff, 0xfff0])])
@pytest.mark.parametrize("V", [7, 5000, 40001])
def test_nan_of_any_bits(dtype, patterns, V):
    """A NaN is one whatever its sign and payload: among logits, negative logits, masked ones and in a row of its own kind, in the
    first place, the middle and the last."""
    whole = torch.int32 if dtype == torch.float32 else torch.int16
    for bits in patterns:
        nan = bits - (1 << whole.itemsize * 8) if bits >> (whole.itemsize * 8 - 1) else bits
        z = torch.randn(10, V, generator=torch.Generator().manual_seed(5)).to(dtype)
        z[3:6] = -z[3:6].abs() - 1.0
        z[6:9] = -math.inf
        w = z.view(whole)
        for r in range(9):
            w[r, (0, V // 2, V - 1)[r % 3]] = nan
        w[9] = nan
        assert z.isnan().any(1).all()
        for top, entropy in ((0, False), (0, True), (3, True)):
            with torch.no_grad():
                r = core.token_logprobs(z.cuda(), torch.full((10,), 1).cuda(), entropy=entropy, top=top)
            assert bool(r.logprobs.isnan().all()), hex(bits)
            if entropy:
                assert bool(r.entropy.isnan().all()), hex(bits)
            if top:
                assert bool(r.top_logprobs.isnan().all()) and bool((r.top_ids == -1).all()), hex(bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 70001])
@pytest.mark.parametrize("tau", [1.0, 1e6, 1e18])
def test_the_types_largest_values(V, dtype, tau):
    """Logits at both ends of the type: a difference past float32's range whose quotient by the temperature is not.  Off by the
    two roundings of the difference and the temperature's reciprocal and the product, 4 U, and the sum's (at most 2^-20)."""
    big = torch.finfo(dtype).max
    z = torch.full((3, V), -big, dtype=dtype)
    z[0, 1] = z[1, V - 1] = big
    z[2] = torch.linspace(-big / 2, big, V, dtype=torch.float64).to(dtype)
    y = torch.tensor([0, 2, 0])
    with torch.no_grad():
        r = core.token_logprobs(z.cuda(), y.cuda(), temperature=tau, entropy=True, top=3)
    t = (z.double() - z.double().max(1, keepdim=True).values) / tau
    l = t - t.exp().sum(1, keepdim=True).log()
    want = torch.cat([l.gather(1, y[:, None]), l.gather(1, r.top_ids.cpu())], 1)
    got = torch.cat([r.logprobs[:, None], r.top_logprobs], 1).cpu().double()
    past = want < -float(torch.finfo(torch.float32).max)
    assert torch.equal(got == -math.inf, past) and bool((past.any() if tau == 1.0 else ~past.any()))
    assert bool(((got - want).abs() <= 4 * U * want.abs() + 2.0 ** -20)[~past].all())
    p = l.exp()
    h = -torch.where(p > 0, p * l, torch.zeros_like(p)).sum(1)
    assert bool(((r.entropy.cpu().double() - h).abs() <= 2.0 ** -20 * (1 + h)).all())


def test_nearly_certain_rows_keep_their_digits():
    """A token of probability 1 - q, q down to 1e-12: log probability -q and entropy of about q (1 + log 1 / q), to relative
    precision: log1p of the others' sum, which is off by U (5 a + 4 + c)."""
    V = 1000
    for gap in (5.0, 15.0, 25.0, 35.0):
        z = torch.zeros(2, V)
        z[:, 123] = gap
        y = torch.tensor([123, 7])
        with torch.no_grad():
            r = core.token_logprobs(z.cuda(), y.cuda(), entropy=True)
        w = reference(z, y, 1.0, 0)
        q = (V - 1) * math.exp(-gap)
        lp, h = -math.log1p(q), math.log1p(q) + gap * q / (1 + q)
        rel = U * (5 * gap + 16 + 3 * chain(V))
        assert abs(float(r.logprobs[0]) - lp) <= rel * abs(lp), gap
        assert abs(float(r.entropy[0]) - h) <= 2 * rel * h, gap
        assert abs(float(r.logprobs[1]) - float(w["logprobs"][1])) <= float(w["logprobs_b"][1])


@pytest.mark.parametrize("N,V", [(4, 1), (5, 13), (4, 64), (6, 1000), (3, 4099), (2, 32768), (2, 32771), (2, 70001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("what", ["logprob", "entropy", "both"])
def test_gradient(N, V, dtype, what):
    z, y, g = make(N, V, dtype, V)
    dlp = torch.randn(N, generator=g) if what != "entropy" else None
    dh = torch.randn(N, generator=g) if what != "logprob" else None
    if N > 3 and dlp is not None:
        dlp[3] = 0
    say(V, dtype, what, check_grad(z, y, 0.7, dlp, dh)[0])


def test_gradient_by_differences():
    """(f(z + h d) - f(z - h d)) / 2 h for a few directions: off by h^2 / 6 of the third derivative (below 8 / tau^3 |d|^3 for
    both functions) and by the outputs' own error over h."""
    z, y, g = make(4, 300, torch.float32, 5)
    tau, h = 0.9, 2.0 ** -7
    x = z.cuda().requires_grad_(True)
    r = core.token_logprobs(x, y.cuda(), temperature=tau, entropy=True)
    wl, wh = torch.randn(4, generator=g), torch.randn(4, generator=g)
    grad, = torch.autograd.grad([r.logprobs, r.entropy], x, [wl.cuda(), wh.cuda()])
    w = reference(z, y, tau, 0)
    for _ in range(3):
        d = torch.randn(z.shape, generator=g).clamp(-1, 1)
        up, down = ((z + s * h * d) for s in (1, -1))
        with torch.no_grad():
            f = [core.token_logprobs(t.cuda(), y.cuda(), temperature=tau, entropy=True) for t in (up, down)]
        f = [(wl.double() * t.logprobs.cpu().double() + wh.double() * t.entropy.cpu().double()).sum() for t in f]
        got = float((grad.double().cpu() * d.double()).sum())
        err = float((wl.abs() * w["logprobs_b"] + wh.abs() * w["entropy_b"]).sum()) * 2 / h
        err += h * h / 6 * 8 / tau ** 3 * float((wl.abs() + wh.abs() * 8).sum()) + 1e-5 * abs(got)
        # z + h d is rounded: half a step of values below 16, in every direction
        err += 2.0 ** -21 / h * float(grad.abs().sum())
        assert abs(float(f[0] - f[1]) / (2 * h) - got) <= err


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_strides_and_alignment(dtype):
    """Leading dimensions, row strides, rows that start at any element, one row for all, expanded gradients, int32 targets."""
    V = 203
    z, y, g = make(24, V + 6, dtype, 9)
    wide = z.cuda()
    for off in (0, 1, 3):
        part = wide[:, off:off + V]
        r = core.token_logprobs(part, y.cuda().clamp(0, V - 1).int(), entropy=True, top=6)
        w = reference(z[:, off:off + V], y.clamp(0, V - 1), 1.0, 6)
        near(r.logprobs, w["logprobs"], w["logprobs_b"], off)
        assert torch.equal(r.top_ids.cpu(), w["top_ids"])
        x = wide.clone().requires_grad_(True)
        core.token_logprobs(x[:, off:off + V], y.cuda(), ignore_index=-100).logprobs.sum().backward()   # an expanded gradient
        want = (torch.where(w["p"] >= 0, -w["p"], 0.0))
        given = (y >= 0) & (y < V)
        want[~given] = 0.0
        want[torch.arange(24)[given], y[given]] += 1.0
        assert float((x.grad[:, off:off + V].double().cpu() - want).abs().max()) < torch.finfo(dtype).eps
        assert not x.grad[:, :off].any() and not x.grad[:, off + V:].any()
    r3 = core.token_logprobs(wide.view(2, 3, 4, V + 6), y.cuda().view(2, 3, 4), entropy=True, top=6)
    r2 = core.token_logprobs(wide, y.cuda(), entropy=True, top=6)
    assert r3.logprobs.shape == (2, 3, 4) and r3.top_ids.shape == (2, 3, 4, 6)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(r3, r2))
    t = core.token_logprobs(wide[:8].t(), None, top=2)   # a transposed view
    assert torch.equal(t.top_ids, core.token_logprobs(wide[:8].t().contiguous(), None, top=2).top_ids)
    one = core.token_logprobs(wide[:1].expand(5, -1), y[:1].cuda().expand(5), top=3)
    assert torch.equal(one.logprobs, r2.logprobs[:1].expand(5)) and torch.equal(one.top_ids, r2.top_ids[:1, :3].expand(5, -1))
    v = core.token_logprobs(wide[0], y[0].cuda(), top=3)
    assert v.logprobs.shape == () and torch.equal(v.top_ids, r2.top_ids[0, :3])
    e = core.token_logprobs(wide[:0], y[:0].cuda(), entropy=True, top=3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)
    x = wide[:0].clone().requires_grad_(True)
    core.token_logprobs(x, y[:0].cuda()).logprobs.sum().backward()
    assert x.grad.shape == x.shape
    back = core.token_logprobs(wide.clone().requires_grad_(True), y.cuda(), entropy=True, top=6)
    assert all(torch.equal(a, b) for a, b in zip(back, r2)) and not back.top_logprobs.requires_grad


def test_offsets_past_32_bits():
    """The last rows of a tensor of more than 2^31 logits, at a row stride that only 64 bits hold."""
    V, stride, N = 1000, (1 << 28) + 8, 9
    buf = torch.empty((N - 1) * stride + V, dtype=torch.bfloat16, device="cuda")
    z = buf.as_strided((N, V), (stride, 1))
    small, y, _ = make(N, V, torch.bfloat16, 4)
    z.copy_(small)
    r = core.token_logprobs(z, y.cuda(), entropy=True, top=5)
    s = core.token_logprobs(small.cuda(), y.cuda(), entropy=True, top=5)
    assert all(torch.equal(a, b) for a, b in zip(r, s))
    x = z.detach().requires_grad_(True)
    g, = torch.autograd.grad(core.token_logprobs(x, y.cuda()).logprobs.sum(), x)
    x = small.cuda().requires_grad_(True)
    h, = torch.autograd.grad(core.token_logprobs(x, y.cuda()).logprobs.sum(), x)
    assert torch.equal(g, h)


def test_streams_graphs_and_repeats():
    """The same bits from call to call, on another stream, and from replays of two graphs that hold the call, between eager
    calls of their own; a training step captured along with its gradient."""
    z, y, g = make(40, 33000, torch.bfloat16, 8)
    a, b = z.cuda(), z.flip(0).contiguous().cuda()
    yd = y.cuda()
    want = core.token_logprobs(a, yd, entropy=True, top=20)
    want_b = core.token_logprobs(b, yd, entropy=True, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = core.token_logprobs(a, yd, entropy=True, top=20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    held = a.clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = core.token_logprobs(held, yd, entropy=True, top=20)
        graphs.append((gr, out))
    train = torch.cuda.CUDAGraph()
    x = held.clone().requires_grad_(True)
    torch.autograd.grad(core.token_logprobs(x, yd, entropy=True).logprobs.sum(), x)
    torch.cuda.synchronize()
    with torch.cuda.graph(train):
        r = core.token_logprobs(x, yd, entropy=True)
        dx, = torch.autograd.grad([r.logprobs, r.entropy], x, [torch.ones_like(r.logprobs), torch.ones_like(r.entropy)])
    for i in range(4):
        src, w = ((a, want), (b, want_b))[i % 2]
        held.copy_(src)
        for gr, out in graphs:
            gr.replay()
        eager = core.token_logprobs(src, yd, entropy=True, top=20)
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, w)) and all(torch.equal(p, q) for p, q in zip(eager, w))
        with torch.no_grad():
            x.copy_(src)
        train.replay()
        e = src.clone().requires_grad_(True)
        r2 = core.token_logprobs(e, yd, entropy=True)
        de, = torch.autograd.grad([r2.logprobs, r2.entropy], e, [torch.ones_like(r.logprobs), torch.ones_like(r.entropy)])
        torch.cuda.synchronize()
        assert torch.equal(dx, de)


def test_model_scores_and_teaches():
    """OneSdmLM.token_logprobs is the operator on its logits; a teacher's alternatives go straight into a student's distillation
    loss; the loss on given tokens trains."""
    torch.manual_seed(0)
    kw = dict(d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4)
    teacher, student = OneSdmLM(211, **kw, seed=1).cuda(), OneSdmLM(211, **kw, seed=2).cuda()
    idx = torch.randint(0, 211, (3, 40), device="cuda")
    with torch.no_grad():
        r = teacher.token_logprobs(idx, entropy=True, top=12)
        logits = teacher(idx)
        want = core.token_logprobs(logits[:, :-1].contiguous(), idx[:, 1:], entropy=True, top=12)
    assert r.logprobs.shape == (3, 40) and not r.logprobs[:, -1].any()
    assert all(torch.equal(p[:, :-1], q) for p, q in zip(r, want))
    # the loss knows the teacher by differences of its entries alone: its logits at the ids, or their log probabilities
    loss = student.distill_loss(idx, r.top_ids, r.top_logprobs, temperature=2.0)
    same = student.distill_loss(idx, r.top_ids, logits.gather(-1, r.top_ids), temperature=2.0)
    assert abs(float(loss.detach()) - float(same.detach())) <= 1e-5 * float(loss.detach())
    s = student.token_logprobs(idx, entropy=True)
    (-s.logprobs.sum() - 0.01 * s.entropy.sum()).backward()
    ref = [p.grad.clone() for p in student.parameters() if p.grad is not None]
    student.zero_grad()
    logits = student(idx)
    lp = torch.log_softmax(logits.float(), -1)
    ce = -lp[:, :-1].gather(-1, idx[:, 1:, None]).sum() - 0.01 * -(lp.exp() * lp).sum()
    ce.backward()
    for a, p in zip(ref, (p for p in student.parameters() if p.grad is not None)):
        assert float((a - p.grad).abs().max()) <= 1e-3 * float(p.grad.abs().max()) + 1e-6


def test_in_a_decode_loop():
    """Each token's log probability and alternatives beside the step that samples it."""
    model = OneSdmLM(307, d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4, seed=3).cuda()
    state = model.decode_state(5)
    tok = torch.arange(5, device="cuda")
    seq, lps = [tok], []
    with torch.no_grad():
        for _ in range(6):
            logits = model.step(tok, state)
            tok = logits.argmax(-1)
            r = core.token_logprobs(logits, tok, top=3)
            assert torch.equal(r.top_ids[:, 0], tok) and torch.equal(r.top_logprobs[:, 0], r.logprobs)
            seq.append(tok)
            lps.append(r.logprobs)
        idx = torch.stack(seq, 1)
        full = model.token_logprobs(idx).logprobs[:, :-1]
    assert float((full - torch.stack(lps, 1)).abs().max()) < 1e-3


def test_refusals_on_the_gpu():
    z, y = torch.randn(4, 50, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    for call, text in [
            (lambda: core.token_logprobs(z.double(), y), "float32 or bfloat16"),
            (lambda: core.token_logprobs(z, y[:3]), "targets"),
            (lambda: core.token_logprobs(z, y.float()), "int64 or int32"),
            (lambda: core.token_logprobs(z, y.cpu()), "is on cpu"),
            (lambda: core.token_logprobs(z), "neither"),
            (lambda: core.token_logprobs(z[:, :0], y), "vocab"),
            (lambda: core.token_logprobs(z, y, top=257), "256"),
            (lambda: core.token_logprobs(z, y, top=-1), "top"),
            (lambda: core.token_logprobs(z, y, temperature=0.0), "temperature"),
            (lambda: core.token_logprobs(z, y, temperature=math.nan), "temperature")]:
        with pytest.raises((ValueError, RuntimeError), match=text):
            call()
    x = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(core.token_logprobs(x, y).logprobs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
