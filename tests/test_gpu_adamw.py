"""core.adamw, core.grad_norm, core.read_moments and the AdamW optimiser on the GPU.

The moments' arithmetic is the formula's, every product and sum rounded to float32, so float32 on the CPU gives the same bits, and
the codes of the 8-bit moments follow from the format by exact arithmetic in float64.  A parameter in float32 is off by U = 2^-24
of its size for its own product and sum (3 U), and its change by the roundings of a division and a square root (16 U); in
bfloat16 by half a step (2^-9... of its size, eps / 2) more."""
import copy
import io
import math

import numpy as np
import pytest
import torch

from sdmchat_amd import AdamW, OneSdmLM, core

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (127,), (128,), (129,), (5, 77), (4096,), (4097,), (16385,), (3, 8, 11), (0,), (200, 130)]


def mix(x):
    x = ((x ^ (x >> 16)) * 2654435761) & 0xffffffff
    x = ((x ^ (x >> 15)) * 3144134277) & 0xffffffff
    return x ^ (x >> 16)


def rounded(x, r, low):
    """float32 [blocks, 128] to the values of the 8-bit format, in float64, with whole numbers r < 2^16; low: 14 or 30."""
    x = x.astype(np.float64)
    big = np.abs(x).max(1, keepdims=True)
    frac, e = np.frexp(big)
    top = e - 1 + (frac > 0.9375)
    y = np.abs(x) * np.exp2(-top.astype(np.float64))
    q = np.exp2(np.floor(np.log2(np.maximum(y, 2.0 ** -low))) - 3.0)
    # 20 bits of a value lie below its code's last place: all that float32 has of a normal one, rounded to them below
    n = np.floor(np.rint(y / q * 2.0 ** 20) / 2.0 ** 20 + r / 65536.0)
    if low == 30:
        n = np.where((y > 0) & (n < 1), 1.0, n)
    return np.where(big < 2.0 ** -126, 0.0, np.sign(x) * n * q * np.exp2(top.astype(np.float64)))


class Twin:
    """The formula on the CPU for one list of tensors."""

    def __init__(self, ps, bits, seed=0):
        self.bits, self.seed, self.t = bits, seed, 0
        self.p = [p.detach().float().cpu().numpy().reshape(-1) for p in ps]
        self.dtype = [p.dtype for p in ps]
        self.m = [np.zeros(p.size, np.float32) for p in self.p]
        self.v = [np.zeros(p.size, np.float32) for p in self.p]

    def step(self, grads, max_norm=None, norm=None, lr=None, betas=None, eps=None, weight_decay=None):
        f = np.float32
        lr, betas = HYPER["lr"] if lr is None else lr, betas or HYPER["betas"]
        eps, wd = HYPER["eps"] if eps is None else eps, HYPER["weight_decay"] if weight_decay is None else weight_decay
        self.t += 1
        gs = [g.detach().float().cpu().numpy().reshape(-1) for g in grads]
        if max_norm is not None:
            if norm is None:
                norm = f(math.sqrt(sum(float(np.square(g.astype(np.float64)).sum()) for g in gs)))
            c = f(max_norm) / (f(norm) + f(1e-6))
            gs = [g * min(f(1.0), c) for g in gs]
        b1, b2, c1, c2 = f(betas[0]), f(betas[1]), f(1 - betas[0]), f(1 - betas[1])
        first = 0
        self.bound = []
        for i, g in enumerate(gs):
            m = self.m[i] * b1 + g * c1
            v = self.v[i] * b2 + g * g * c2
            den = np.sqrt(v.astype(np.float64)) / math.sqrt(1 - betas[1] ** self.t) + eps
            with np.errstate(invalid="ignore", divide="ignore"):
                move = lr / (1 - betas[0] ** self.t) * m.astype(np.float64) / den
            p = self.p[i] * (1 - lr * wd) - move
            b = 3 * U * np.abs(self.p[i]) + 16 * U * np.abs(move) + 1e-37
            if self.dtype[i] == torch.bfloat16:
                b = b + 2.0 ** -8 * np.abs(p)
            self.bound.append(b)
            self.p[i] = p
            n = m.size
            if self.bits == 8 and n:
                blocks = -(-n // 128)
                key = mix((self.seed + self.t * 2654435761) & 0xffffffff)
                u = mix((np.arange(blocks * 128, dtype=np.int64) + first * 128 + key) & 0xffffffff).reshape(-1, 128)
                pad = lambda a: np.pad(a, (0, blocks * 128 - n)).reshape(-1, 128)  # noqa: E731
                m = rounded(pad(m), u >> 16, 14).reshape(-1)[:n].astype(np.float32)
                v = rounded(pad(v), u & 0xffff, 30).reshape(-1)[:n].astype(np.float32)
                first += blocks
            self.m[i], self.v[i] = m, v

    def compare(self, ps, ms, vs):
        for i, (p, m, v) in enumerate(zip(ps, ms, vs)):
            got = p.detach().float().cpu().numpy().reshape(-1)
            assert np.array_equal(m.detach().float().cpu().numpy().reshape(-1), self.m[i]), ("exp_avg", i)
            assert np.array_equal(v.detach().float().cpu().numpy().reshape(-1), self.v[i]), ("exp_avg_sq", i)
            d = np.abs(got - self.p[i])
            assert (d <= self.bound[i]).all(), ("param", i, float((d / self.bound[i]).max()))
            self.p[i] = got   # the next step starts where the kernel is


def tensors(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for i, s in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        ps.append(torch.randn(s, generator=g).to(dt).cuda())
        gs.append((torch.randn(s, generator=g) * scale * 10.0 ** float(torch.randint(-4, 1, (1,), generator=g))).to(dt).cuda())
    return ps, gs


def regrad(gs, seed):
    g = torch.Generator().manual_seed(seed)
    return [(x.float().cpu() * torch.randn(x.shape, generator=g)).to(x.dtype).cuda() for x in gs]


def read(states, ps, dtype=torch.float32):
    ms, vs = ([torch.full(p.shape, 7.0, dtype=dtype, device="cuda") for p in ps] for _ in range(2))
    core.read_moments(states, ms, vs)
    return ms, vs


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
def test_steps_in_32_bits(dtypes, clip):
    ps, gs = tensors(SIZES, dtypes, 1)
    ms, vs = ([torch.zeros(p.shape, device="cuda") for p in ps] for _ in range(2))
    twin = Twin(ps, 32)
    for t in range(1, 5):
        gs = regrad(gs, t)
        norm = core.adamw(ps, gs, ms, vs, step=t, max_norm=clip, **HYPER)
        twin.step(gs, clip)
        twin.compare(ps, ms, vs)
        if clip is None:
            assert norm is None
        else:
            want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
            assert abs(float(norm) - want) <= 2 * U * want


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_steps_in_8_bits(dtypes, clip):
    """Every code is the format's for the formula's value and the hash, at all sizes of tensors around blocks and chunks."""
    ps, gs = tensors(SIZES, dtypes, 2)
    st = [core.new_moments(p) for p in ps]
    twin = Twin(ps, 8, seed=99)
    for t in range(1, 6):
        gs = regrad(gs, t)
        if t == 4:
            gs = [g * 0 for g in gs]   # moments fade without gradients
        core.adamw(ps, gs, st, step=t, max_norm=clip, seed=99, **HYPER)
        twin.step(gs, clip)
        ms, vs = read(st, ps)
        twin.compare(ps, ms, vs)
        mb, vb = read(st, ps, torch.bfloat16)
        assert all(torch.equal(a.float(), b) for a, b in zip(mb + vb, ms + vs))


def test_values_of_every_size_in_8_bits():
    """Blocks whose values span what float32 holds: zeros, values below the format's least, single values, powers of two, and
    just below and above a mantissa of 1.875."""
    rows = [np.zeros(128), np.exp2(-np.arange(128.0) / 2), np.exp2(-np.arange(128.0)), np.full(128, 1.875), np.full(128, 1.8750001),
            np.full(128, 1.9999999), np.exp2(np.linspace(-60, 60, 128)), np.where(np.arange(128) == 5, 3e-20, 0.0),
            np.full(128, 1e-22), np.linspace(-1, 1, 128), np.full(128, 2.0 ** -60), np.linspace(1e-12, 1e12, 128)]
    g = torch.from_numpy(np.stack(rows).astype(np.float32).reshape(-1)).cuda()
    p = torch.zeros_like(g)
    st, twin = [core.new_moments(p)], Twin([p], 8)
    for t in range(1, 4):
        core.adamw([p], [g], st, step=t, **HYPER)
        twin.step([g])
        ms, vs = read(st, [p])
        assert np.array_equal(ms[0].cpu().numpy(), twin.m[0]) and np.array_equal(vs[0].cpu().numpy(), twin.v[0])
        seen = g.cpu().numpy()
        squares = np.float32(1 - 0.999) * seen * seen
        blocks = squares.reshape(-1, 128).max(1).repeat(128)
        assert (vs[0].cpu().numpy()[(squares > 0) & (blocks > 1e-37)] > 0).all()
        assert np.isfinite(p.cpu().numpy()).all()


def test_rounding_is_fair():
    """The mean of the stored moments over many seeds is the value itself: n of them are off by a step q at most, so their mean
    by 6 q / sqrt(n) but for a chance of 1e-8; and 2^-16 q of the hash's 16 bits."""
    n, value = 1 << 16, 0.731
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), value, device="cuda")
    g[::128] = 5.0   # the block's largest
    st = [core.new_moments(p)]
    core.adamw([p], [g], st, step=1, seed=5, **HYPER)
    ms, vs = read(st, [p])
    keep = torch.arange(n, device="cuda") % 128 != 0
    for got, want in ((ms[0][keep], np.float32(value) * np.float32(1 - 0.9)),
                      (vs[0][keep], np.float32(value) * np.float32(value) * np.float32(1 - 0.999))):
        q = 2.0 ** (math.floor(math.log2(want)) - 3)
        values = got.double().unique()
        assert len(values) == 2 and float(values[1] - values[0]) == q
        assert abs(float(got.double().mean()) - float(want)) <= 6 * q / math.sqrt(got.numel()) + 2.0 ** -16 * q


def test_fading_is_not_stuck():
    """Without gradients a second moment falls by 0.1% a step: less than a code's step, so only chance rounding follows it.  After
    2,000 steps it is at exp(-2) of its start on the mean (here within 10%: the mean of 2^14 walks, each of a spread of about a
    third of its mean)."""
    n = 1 << 14
    p = torch.zeros(n, device="cuda")
    g = torch.ones(n, device="cuda")
    st = [core.new_moments(p)]
    core.adamw([p], [g], st, step=1, seed=1, **HYPER)
    start = float(read(st, [p])[1][0].double().mean())
    zero = torch.zeros_like(g)
    for t in range(2, 2002):
        core.adamw([p], [zero], st, step=t, seed=1, **HYPER)
    assert abs(float(read(st, [p])[1][0].double().mean()) / start / math.exp(-2.0) - 1) < 0.1


def test_norm():
    ps, gs = tensors(SIZES, [torch.float32, torch.bfloat16], 3)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    got = core.grad_norm(gs)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - want) <= U * want * 1.01
    assert torch.equal(got, core.grad_norm(gs))
    big = [torch.full((100000,), 1e30, device="cuda"), torch.full((5,), 1e-30, device="cuda")]
    assert abs(float(core.grad_norm(big)) / (1e30 * math.sqrt(1e5)) - 1) < 2.0 ** -22
    assert abs(float(core.grad_norm(big[1:])) / (1e-30 * math.sqrt(5)) - 1) < 2.0 ** -22
    assert math.isnan(float(core.grad_norm([torch.tensor([1.0, math.nan], device="cuda")])))
    assert float(core.grad_norm([torch.tensor([1.0, -math.inf], device="cuda")])) == math.inf
    assert float(core.grad_norm([torch.empty(0, device="cuda")])) == 0.0
    t = torch.randn(60, 50, device="cuda")
    many = [t[:, ::2], t.t(), t[:1].expand(7, -1)]   # any strides
    want = math.sqrt(sum(float(x.double().square().sum()) for x in many))
    assert abs(float(core.grad_norm(many)) - want) <= 2 * U * want


@pytest.mark.parametrize("count", [1, 67, 68, 69, 137, 300])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(count, bits):
    """Lists longer than a launch takes."""
    g = torch.Generator().manual_seed(count)
    sizes = [(int(n),) for n in torch.randint(1, 6000, (count,), generator=g)]
    ps, gs = tensors(sizes, [torch.float32, torch.bfloat16, torch.bfloat16], 4)
    twin = Twin(ps, bits, 3)
    ms, vs = ([torch.zeros(p.shape, device="cuda") for p in ps] for _ in range(2))
    st = [core.new_moments(p) for p in ps]
    for t in (1, 2):
        core.adamw(ps, gs, *((ms, vs) if bits == 32 else (st,)), step=t, max_norm=1.0, seed=3, **HYPER)
        twin.step(gs, 1.0)
        if bits == 8:
            ms, vs = read(st, ps)
        twin.compare(ps, ms, vs)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alignment_and_neighbours(bits, dtype):
    """Parameters and gradients that begin at any element of a buffer; what lies beside them stays."""
    n = [1, 5, 131, 2049, 4103]
    for off in (0, 1, 3, 7):
        at, spans = off, []
        for k in n:
            spans.append((at, at + k))
            at += k + 3
        g = torch.Generator().manual_seed(off)
        buf, gbuf = ((torch.randn(at + 9, generator=g)).to(dtype).cuda() for _ in range(2))
        before = buf.clone()
        ps, gs = ([b[i:j] for i, j in spans] for b in (buf, gbuf))
        fm, fv = torch.full((at + 9,), 3.0, device="cuda"), torch.full((at + 9,), 3.0, device="cuda")
        ms, vs = ([b[i:j] for i, j in spans] for b in (fm, fv))
        for t in ms + vs:
            t.zero_()
        st = [core.new_moments(p) for p in ps]
        twin = Twin(ps, bits)
        core.adamw(ps, gs, *((ms, vs) if bits == 32 else (st,)), step=1, **HYPER)
        twin.step(gs)
        twin.compare(ps, *((ms, vs) if bits == 32 else read(st, ps)))
        gaps = torch.ones(at + 9, dtype=torch.bool)
        for i, j in spans:
            gaps[i:j] = False
        gaps = gaps.cuda()
        assert torch.equal(buf[gaps], before[gaps]) and bool((fm[gaps] == 3).all()) and bool((fv[gaps] == 3).all())


def test_orders_of_dimensions():
    """Dense parameters of any order of dimensions, gradients of another."""
    p0 = torch.randn(12, 10, device="cuda").t()
    p1 = torch.randn(2, 3, 4, 5, device="cuda").to(memory_format=torch.channels_last)
    gs = [torch.randn(10, 12, device="cuda"), torch.randn(2, 3, 4, 5, device="cuda")]
    a = [p0.clone(memory_format=torch.preserve_format), p1.clone(memory_format=torch.preserve_format)]
    b = [p0.contiguous(), p1.contiguous()]
    assert a[0].stride() == p0.stride() and a[1].stride() == p1.stride()
    za, zb = ([[torch.zeros_like(p) for p in x] for _ in range(2)] for x in (a, b))
    for t in (1, 2):
        core.adamw(a, gs, *za, step=t, **HYPER)
        core.adamw(b, gs, *zb, step=t, **HYPER)
    assert all(torch.equal(x, y) for x, y in zip(a + za[0] + za[1], b + zb[0] + zb[1]))


def test_non_finite_gradients():
    """In 32 bits a NaN stays with its value; in 8 bits with its block of 128; through a clip it reaches everything."""
    for bits in (32, 8):
        p = torch.ones(300, device="cuda")
        g = torch.ones(300, device="cuda")
        g[140] = math.nan
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        st = [core.new_moments(p)]
        for t in (1, 2):
            core.adamw([p], [g], *(([m], [v]) if bits == 32 else (st,)), step=t, **HYPER)
        bad = p.isnan().cpu()
        want = torch.zeros(300, dtype=torch.bool)
        if bits == 32:
            want[140] = True
        else:
            want[128:256] = True
        assert torch.equal(bad, want)
        q = torch.ones(300, device="cuda")
        core.adamw([q], [g], *(([torch.zeros_like(q)], [torch.zeros_like(q)]) if bits == 32 else ([core.new_moments(q)],)),
                   step=1, max_norm=1.0, **HYPER)
        assert bool(q.isnan().all())
    p, g = torch.ones(4, device="cuda"), torch.tensor([1.0, math.inf, 0.0, 1.0], device="cuda")
    core.adamw([p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)], step=1, max_norm=1.0, **HYPER)
    assert p.isnan().cpu().tolist() == [False, True, False, False]   # 1 / inf: the others' gradients are 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-30, 1e-15, 1e-12, 1e-8, 1e3])
def test_gradients_and_eps_of_every_size(bits, eps):
    """One value alone in its block, from 1e-38 (v underflows: as the formula does in float32) to 1e18: the parameter is the formula's
    from float32 moments to the roundings of a root, a quotient and their products (16 U of the move)."""
    for e in range(-38, 19, 2):
        g = torch.zeros(4 * 128)
        g[::128] = torch.tensor([1.0, -1.3, 1.7, 2.0]) * 10.0 ** e
        p = torch.randn(g.shape, generator=torch.Generator().manual_seed(e + 50))
        f = np.float32
        m, v = g.numpy() * f(1 - 0.9), g.numpy() * g.numpy() * f(1 - 0.999)
        for device in (False, True):
            q = p.cuda()
            st = ([torch.zeros_like(q)], [torch.zeros_like(q)]) if bits == 32 else ([core.new_moments(q)],)
            core.adamw([q], [g.cuda()], *st, step=torch.zeros((), dtype=torch.int64, device="cuda") if device else 1,
                       **dict(HYPER, eps=eps))
            with np.errstate(invalid="ignore", divide="ignore"):
                move = HYPER["lr"] / (1 - 0.9) * (m.astype(np.float64) / (np.sqrt(v.astype(np.float64) / (1 - 0.999)) + eps))
            old = p.numpy().astype(np.float64)
            want = old * (1 - HYPER["lr"] * HYPER["weight_decay"]) - move
            got = q.cpu().numpy().astype(np.float64)
            with np.errstate(invalid="ignore"):
                near = np.abs(got - want) <= 3 * U * np.abs(old) + 16 * U * np.abs(move)
            same = (np.isnan(got) & np.isnan(want)) | (got == want)   # 0 / 0 and m / 0
            assert (near | same).all(), (e, device, got[::128], want[::128])


@pytest.mark.parametrize("dtype,patterns", [(torch.float32, [0x7fc00000, 0xffc00000, 0x7f800001, 0x7fffffff, 0xffffffff, 0xfff00001]),
                                            (torch.bfloat16, [0x7fc0, 0xffc0, 0x7f81, 0x7fff, 0xffff, 0xfff0])])
def test_nan_of_any_bits(dtype, patterns):
    """A NaN is one whatever its sign and payload: for its block's exponents, its parameter and the norm."""
    whole = torch.int32 if dtype == torch.float32 else torch.int16
    for bits in patterns:
        g = torch.ones(300, device="cuda", dtype=dtype)
        g.view(whole)[140] = bits - (1 << whole.itemsize * 8) if bits >> (whole.itemsize * 8 - 1) else bits
        assert g.isnan().cpu().nonzero().flatten().tolist() == [140]
        assert math.isnan(float(core.grad_norm([g])))
        p = torch.ones_like(g)
        st = [core.new_moments(p)]
        core.adamw([p], [g], st, step=1, **HYPER)
        assert p.isnan().cpu().nonzero().flatten().tolist() == [140], hex(bits)
        block = torch.zeros(300, dtype=torch.bool)
        block[128:256] = True
        for moment in read(st, [p]):
            assert torch.equal(moment[0].isnan().cpu(), block), hex(bits)
        m, v = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
        core.adamw([p], [g], [m], [v], step=1, **HYPER)
        for moment in (m, v, p):
            assert moment.isnan().cpu().nonzero().flatten().tolist() == [140], hex(bits)


def test_step_and_lr_on_the_device():
    ps, gs = tensors([(300,), (77,)], [torch.float32], 6)
    for bits in (32, 8):
        a, b = ([p.clone() for p in ps] for _ in range(2))
        sa, sb = ((([torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]) if bits == 32 else
                   ([core.new_moments(p) for p in ps],)) for _ in range(2))
        count, lr = torch.zeros((), dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
        for t in range(1, 5):
            rate = 1e-3 * t
            lr.fill_(rate)
            core.adamw(a, gs, *sa, step=t, lr=float(lr), betas=(0.8, 0.95), seed=4, weight_decay=0.2)
            core.adamw(b, gs, *sb, step=count, lr=lr, betas=(0.8, 0.95), seed=4, weight_decay=0.2)
            assert int(count) == t
        assert all(torch.equal(x, y) for x, y in zip(sa[0], sb[0]))
        # the two hosts' and device's corrections may differ by their last places
        assert all(float((x - y).abs().max()) <= 16 * U for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Two graphs that hold the same optimiser's step, replayed in turn with eager work between them, against an eager twin; a
    schedule writes the learning rate.  The moments are the twin's to the bit; a parameter may differ by the last places of the
    corrections and rates that the device computes (16 U of five moves of at most 2e-2)."""
    ps, gs = tensors(SIZES, [torch.float32, torch.bfloat16], 12)
    a, b = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    lr = torch.full((), 1e-3, device="cuda")
    oa = AdamW(a, lr=1e-3, state_bits=bits, max_norm=1.0)
    ob = AdamW(b, lr=lr, state_bits=bits, max_norm=1.0, capturable=True)
    for p, g in zip(b, gs):
        p.grad = g.clone()
    with pytest.raises(RuntimeError, match="run a step before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ob.step()

    def write(t, rate):
        new = regrad(gs, t)
        for p, q, g in zip(a, b, new):
            p.grad = g
            q.grad.copy_(g)
        lr.fill_(rate)
        for group in oa.param_groups:
            group["lr"] = float(lr)

    def same():
        torch.cuda.synchronize()
        assert torch.equal(oa.norm, ob.norm)
        for p, q in zip(a, b):
            step = 2.0 ** -8 * p.detach().float().abs() if p.dtype == torch.bfloat16 else U * p.detach().abs()
            assert bool(((p - q).detach().float().abs() <= 2 * step + 16 * U * 5 * 2e-2).all())
            assert all(torch.equal(v, ob.state[q][k]) for k, v in oa.state[p].items() if k != "step")
            with torch.no_grad():
                q.copy_(p)
    write(0, 1e-3)
    oa.step()
    ob.step()
    same()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ob.step()
        norm = ob.norm
        graphs[-1].norm_of_step = norm
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step()
    for t in range(1, 7):
        write(t, 1e-3 * t)
        oa.step()
        g = graphs[t % 2]
        g.replay()
        ob.norm = g.norm_of_step
        core.grad_norm(gs)
        same()
    assert {int(st["step"]) for st in ob.state.values()} == {7} == {st["step"] for st in oa.state.values()}


def test_optimizer_follows_torch():
    """The optimiser's steps on a model are those of torch's AdamW behind clip_grad_norm_ on the same gradients."""
    ps, gs = tensors([(64, 64), (300,), (7, 9)], [torch.float32], 8)
    a, b = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    mine = AdamW([dict(params=a[:1], weight_decay=0.3), dict(params=a[1:], lr=5e-4, betas=(0.8, 0.9))], lr=1e-3, max_norm=0.7)
    ref = torch.optim.AdamW([dict(params=b[:1], weight_decay=0.3), dict(params=b[1:], lr=5e-4, betas=(0.8, 0.9))], lr=1e-3,
                            foreach=False)
    for t in range(5):
        new = regrad(gs, t)
        for x, y, g in zip(a, b, new):
            x.grad, y.grad = g.clone(), g.clone()
        if t == 2:
            a[1].grad = b[1].grad = None   # a parameter that sits a step out keeps its count
        mine.step()
        torch.nn.utils.clip_grad_norm_(b, 0.7)
        ref.step()
        assert abs(float(mine.norm) - math.sqrt(sum(float(g.double().square().sum()) for x, g in zip(a, new) if x.grad is not None))) \
            <= 4 * U * float(mine.norm)
        for x, y in zip(a, b):
            # five steps of roundings of float32 products in another order
            assert float((x - y).detach().abs().max()) <= (t + 1) * 64 * U * float(y.detach().abs().max())
    assert [mine.state[p]["step"] for p in a] == [5, 4, 5]
    assert all(torch.equal(x.grad, g) for x, g in zip(a, new))   # the gradients themselves are not clipped


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.float32), (8, torch.bfloat16), (32, torch.bfloat16)])
def test_optimizer_state_travels(bits, dtype):
    """state_dict through torch.save and load_state_dict, and a deepcopy, continue with the same bits."""
    ps, gs = tensors([(64, 33), (129,)], [dtype], 9)

    def fresh(capturable=False):
        qs = [torch.nn.Parameter(p.clone()) for p in ps]
        return qs, AdamW([dict(params=qs[:1]), dict(params=qs[1:], state_bits=32)], lr=1e-2, state_bits=bits, seed=6,
                         capturable=capturable)

    def go(qs, opt, seeds):
        for s in seeds:
            for q, g in zip(qs, regrad(gs, s)):
                q.grad = g
            opt.step()
    for capturable in (False, True):
        a, oa = fresh(capturable)
        go(a, oa, range(3))
        f = io.BytesIO()
        torch.save(dict(p=[q.detach() for q in a], o=oa.state_dict()), f)
        f.seek(0)
        blob = torch.load(f, weights_only=True, map_location="cpu")
        b, ob = fresh(capturable)
        with torch.no_grad():
            for q, v in zip(b, blob["p"]):
                q.copy_(v)
        ob.load_state_dict(blob["o"])
        c = copy.deepcopy(a)
        oc = AdamW([dict(params=c[:1]), dict(params=c[1:], state_bits=32)], lr=1e-2, state_bits=bits, seed=6, capturable=capturable)
        oc.load_state_dict(oa.state_dict())
        for qs, o in ((a, oa), (b, ob), (c, oc)):
            go(qs, o, range(3, 6))
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
        for x, y in zip(a, b):
            assert {k: str(v.dtype) for k, v in oa.state[x].items() if k != "step"} == {
                k: str(v.dtype) for k, v in ob.state[y].items() if k != "step"}
            assert all(torch.equal(v, ob.state[y][k]) for k, v in oa.state[x].items() if k != "step")
        wrong = AdamW(b, lr=1e-2, state_bits=8 if bits == 32 else 32, capturable=capturable)
        sd = oa.state_dict()
        sd["param_groups"] = [dict(sd["param_groups"][0], params=[0, 1], state_bits=8 if bits == 32 else 32)]
        with pytest.raises(ValueError, match="state of a parameter"):
            wrong.load_state_dict(sd)


def test_a_model_trains_and_serves_its_new_weights():
    """Caches of prepared weights see the step; every arm's parameters move; in float32 and under bfloat16 autocast."""
    torch.manual_seed(2)
    kw = dict(d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4)
    for ffn, autocast, bits in (("mlp", False, 32), ("sdm", False, 8), ("mlp", True, 8)):
        model = OneSdmLM(211, **kw, ffn=ffn, sdm_n_sub=8, sdm_heads=2, sdm_d_a=16, sdm_k=8, seed=4).cuda()
        opt = model.optimizer(1e-2, state_bits=bits, max_norm=1.0)
        idx = torch.randint(0, 211, (2, 24), device="cuda")
        with torch.no_grad():
            before = model(idx)
        old = {n: p.detach().clone() for n, p in model.named_parameters()}
        versions = {n: p._version for n, p in model.named_parameters()}
        for _ in range(2):
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
                loss = -model.token_logprobs(idx).logprobs.mean()
            loss.backward()
            opt.step()
        for n, p in model.named_parameters():
            if p.grad is not None and bool(p.grad.any()):
                assert not torch.equal(p, old[n]), n
                assert p._version > versions[n]
        twin = OneSdmLM(211, **kw, ffn=ffn, sdm_n_sub=8, sdm_heads=2, sdm_d_a=16, sdm_k=8, seed=5).cuda()
        twin.load_state_dict(model.state_dict())
        with torch.no_grad():
            now = model(idx)
            assert torch.equal(now, twin(idx)) and not torch.equal(now, before)


def test_a_saved_parameter_is_not_read_again():
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_another_stream():
    ps, gs = tensors([(70000,), (300,)], [torch.float32], 7)
    a, b = ([p.clone() for p in ps] for _ in range(2))
    za, zb = ([[torch.zeros_like(p) for p in ps] for _ in range(2)] for _ in range(2))
    side = torch.cuda.Stream()
    for t in (1, 2, 3):
        core.adamw(a, gs, *za, step=t, max_norm=1.0, **HYPER)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (1, 2, 3):
            core.adamw(b, gs, *zb, step=t, max_norm=1.0, **HYPER)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals_on_the_gpu():
    p, g = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    s = core.new_moments(p)
    keep = p.clone()
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    for call, text in [
            (lambda: core.adamw([], [], [], [], step=1), "no tensors"),
            (lambda: core.adamw([p], [g, g], [m], [v], step=1), "2 grads for 1"),
            (lambda: core.adamw([p], [g.bfloat16()], [m], [v], step=1), "grad of"),
            (lambda: core.adamw([p], [g[:299]], [m], [v], step=1), "grad of"),
            (lambda: core.adamw([p.double()], [g.double()], [m], [v], step=1), "float32 or bfloat16"),
            (lambda: core.adamw([p[::2]], [g[::2]], [m[::2]], [v[::2]], step=1), "dense"),
            (lambda: core.adamw([p], [g], [m.bfloat16()], [v], step=1), "moments must be float32"),
            (lambda: core.adamw([p], [g], [m[:299]], [v], step=1), "moments must be float32"),
            (lambda: core.adamw([p], [g], [m], step=1), "8-bit moments"),
            (lambda: core.adamw([p], [g], [s[:2]], step=1), "8-bit moments"),
            (lambda: core.adamw([p, p], [g, g], [m, v], [m.clone(), v.clone()], step=1), "overlap"),
            (lambda: core.adamw([p], [g], [m], [m], step=1), "overlap"),
            (lambda: core.adamw([p], [p], [m], [v], step=1), "overlap"),
            (lambda: core.adamw([p], [g.cpu()], [m], [v], step=1), "is on cpu"),
            (lambda: core.adamw([p], [g.to_sparse()], [m], [v], step=1), "layout"),
            (lambda: core.adamw([p], [g], [m], [v], step=0), "t must be"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, lr=-1.0), "lr"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, lr=torch.ones((), device="cuda")), "beside a step"),
            (lambda: core.adamw([p], [g], [m], [v], step=count.float()), "int64"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, betas=(1.0, 0.9)), "beta1"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, eps=math.inf), "eps"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, max_norm=0.0), "max_norm"),
            (lambda: core.adamw([p], [g], [m], [v], step=1, norm=torch.ones((), device="cuda")), "needs max_norm"),
            (lambda: core.read_moments([s], [m], [v[:299]]), "alike"),
            (lambda: core.read_moments([s], [m[:100]], [v[:100]]), "contiguous uint8"),
            (lambda: core.grad_norm([]), "no tensors"),
            (lambda: core.grad_norm([g.half()]), "float32 or bfloat16")]:
        with pytest.raises((ValueError, RuntimeError), match=text):
            call()
    assert torch.equal(p, keep) and not m.any() and int(count) == 0


def test_overlaps():
    """What overlaps a tensor that is written is refused, in the plain case and where a tensor's strides are not; grads may be one
    tensor for several params, params may lie next to each other."""
    buf = torch.randn(1000, device="cuda")
    z = lambda n=300: torch.zeros(n, device="cuda")  # noqa: E731
    g = torch.randn(300, device="cuda")
    keep = buf.clone()
    for strided in (False, True):
        more = ([torch.randn(20, 10, device="cuda").t()] if strided else [])
        extra = [torch.randn(10, 20, device="cuda") for _ in more]
        zs = lambda: [torch.zeros_like(t) for t in more]  # noqa: E731
        for ps, gs, ms, vs in [
                ([buf[:300], buf[299:599]], [g, g], [z(), z()], [z(), z()]),
                ([buf[:300]], [buf[100:400]], [z()], [z()]),
                ([buf[:300]], [g], [buf[200:500]], [z()]),
                ([buf[:300]], [g], [z()], [buf[200:500]])]:
            with pytest.raises(ValueError, match="overlap"):
                core.adamw(ps + more, gs + extra, ms + zs(), vs + zs(), step=1)
        assert torch.equal(buf, keep)
        a = [buf[:300], buf[300:600]]
        ms, vs = [z(), z()], [z(), z()]
        core.adamw(a + more, [g, g] + extra, ms + zs(), vs + zs(), step=1, **HYPER)
        b = [t.clone() for t in (keep[:300], keep[300:600])]
        core.adamw(b, [g.clone(), g.clone()], [z(), z()], [z(), z()], step=1, **HYPER)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(buf[600:], keep[600:])
        buf.copy_(keep)
    s = [core.new_moments(g)]
    with pytest.raises(ValueError, match="overlap"):
        core.read_moments(s, [buf[:300]], [buf[299:599]])


class Named(torch.Tensor):
    pass


def test_other_kinds_of_tensors():
    """Subclasses, inference tensors, tuples and iterators in place of lists."""
    g0 = torch.randn(300, device="cuda")
    want = torch.ones(300, device="cuda")
    core.adamw([want], [g0], [torch.zeros_like(want)], [torch.zeros_like(want)], step=1, max_norm=0.1, **HYPER)
    for wrap in (lambda t: t.as_subclass(Named), lambda t: torch.nn.Parameter(t)):
        p, g, m, v = (wrap(t) for t in (torch.ones(300, device="cuda"), g0.clone(), torch.zeros_like(g0), torch.zeros_like(g0)))
        with torch.no_grad():
            core.adamw((p,), iter([g]), (m,), [v], step=1, max_norm=0.1, **HYPER)
        assert torch.equal(p.detach().as_subclass(torch.Tensor), want)
    with torch.inference_mode():
        p, m, v = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
        core.adamw([p], [g0], [m], [v], step=1, max_norm=0.1, **HYPER)
        assert torch.equal(p, want)


def test_the_largest_steps_stream():
    """More values than the last-level cache keeps take other loads and stores: the same bits as in parts."""
    n = (1 << 25) + 77
    for bits in (32, 8):
        for dtype in (torch.float32, torch.bfloat16):
            gen = torch.Generator(device="cuda").manual_seed(1)
            p = torch.randn(n, device="cuda", generator=gen).to(dtype)
            g = torch.randn(n, device="cuda", generator=gen).to(dtype)
            q = p.clone()
            cut = 1 << 18   # a whole number of blocks
            parts = [t.split(cut) for t in (q, g)]
            if bits == 32:
                m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
                m2, v2 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
                core.adamw([p], [g], [m], [v], step=1, **HYPER)
                for a, b, c, d in zip(*parts, m2.split(cut), v2.split(cut)):
                    core.adamw([a], [b], [c], [d], step=1, **HYPER)
                assert torch.equal(m, m2) and torch.equal(v, v2)
            else:
                s = core.new_moments(p)
                core.adamw([p], [g], [s], step=1, seed=3, **HYPER)
                m, v = torch.empty(n, dtype=dtype, device="cuda"), torch.empty(n, dtype=dtype, device="cuda")
                core.read_moments([s], [m], [v])
                # the parts in one list have the positions that the whole has
                small = [core.new_moments(t) for t in parts[0]]
                core.adamw(list(parts[0]), list(parts[1]), small, step=1, seed=3, **HYPER)
                assert torch.equal(torch.cat(small), s)
                m2, v2 = torch.empty_like(m), torch.empty_like(v)
                for t, a, b in zip(small, m2.split(cut), v2.split(cut)):
                    core.read_moments([t], [a], [b])
                assert torch.equal(m, m2) and torch.equal(v, v2)
            assert torch.equal(p, q)
            del p, q, g, m, v, m2, v2, parts


def test_a_training_run_and_its_decoding():
    """The operators together, as a program uses them: a loss on given tokens with an entropy bonus, its gradient, the clipped
    step, the new weights in a captured decode step beside the log probabilities of what it chose."""
    torch.manual_seed(5)
    kw = dict(d=64, layers=2, mlp_f=96, heads=4, n_sub=8, d_a=16, k=4)
    model = OneSdmLM(211, **kw, seed=6).cuda()
    opt = model.optimizer(3e-3, state_bits=8, max_norm=1.0)
    idx = torch.randint(0, 211, (4, 33), device="cuda")
    for _ in range(3):
        opt.zero_grad()
        r = model.token_logprobs(idx, entropy=True)
        (-r.logprobs.sum() / (4 * 32) - 0.01 * r.entropy.mean()).backward()
        opt.step()
        assert math.isfinite(float(opt.norm)) and float(opt.norm) > 0
    with torch.no_grad():
        state, eager = model.decode_state(4), model.decode_state(4)
        tok = idx[:, 0].clone()
        warm = model.decode_state(4)
        for _ in range(2):
            r = core.token_logprobs(model.step(tok, warm), tok, top=5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.step(tok, state)
            nxt = logits.argmax(-1)
            r = core.token_logprobs(logits, nxt, entropy=True, top=5)
        t = idx[:, 0].clone()
        for i in range(5):
            tok.copy_(t)
            graph.replay()
            want = model.step(t, eager)
            w = core.token_logprobs(want, want.argmax(-1), entropy=True, top=5)
            torch.cuda.synchronize()
            assert torch.equal(nxt, want.argmax(-1)) and all(torch.equal(a, b) for a, b in zip(r, w))
            assert torch.equal(r.top_ids[:, 0], nxt)
            t = want.argmax(-1)
