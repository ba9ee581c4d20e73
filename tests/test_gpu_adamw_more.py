"""More of core.adamw and the AdamW optimiser on the GPU (test_gpu_adamw.py has the formula's twin and the bounds)."""
import io

import numpy as np
import pytest
import torch

from sdmchat_amd import AdamW, core
from tests.test_gpu_adamw import HYPER, SIZES, Twin, mix, read, regrad, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_read_on_the_cpu_with_a_rate_on_the_device(bits):
    """The optimiser goes on where the saved one was, its schedule's tensor reaches it, also in a step captured after."""
    ps, gs = tensors(SIZES, [torch.float32, torch.bfloat16], 21)

    def fresh():
        qs = [torch.nn.Parameter(p.clone()) for p in ps]
        rate = torch.full((), 1e-3, device="cuda")
        return qs, rate, AdamW([dict(params=qs[:4]), dict(params=qs[4:])], lr=rate, state_bits=bits, capturable=True, seed=3)

    def give(qs, seed):
        for q, g in zip(qs, regrad(gs, seed)):
            if q.grad is None:
                q.grad = g
            else:
                q.grad.copy_(g)
    a, rate_a, oa = fresh()
    for s in range(3):
        give(a, s)
        rate_a.fill_(1e-3 * (s + 1))
        oa.step()
    f = io.BytesIO()
    torch.save(dict(p=[q.detach() for q in a], o=oa.state_dict()), f)
    f.seek(0)
    blob = torch.load(f, weights_only=True, map_location="cpu")
    b, rate_b, ob = fresh()
    with torch.no_grad():
        for q, v in zip(b, blob["p"]):
            q.copy_(v)
    ob.load_state_dict(blob["o"])
    assert torch.equal(rate_a, rate_b) and all(g["lr"] is rate_b for g in ob.param_groups)

    def same():
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(v, ob.state[y][k]) for x, y in zip(a, b) for k, v in oa.state[x].items())
    for s in range(3, 5):
        for qs, rate, opt in ((a, rate_a, oa), (b, rate_b, ob)):
            give(qs, s)
            rate.fill_(2e-3 * s)
            opt.step()
        same()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for s in range(5, 8):
        for qs, rate in ((a, rate_a), (b, rate_b)):
            give(qs, s)
            rate.fill_(1e-3 * s)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        same()


def stored(x, r, low):
    """What a block's values x (float32 [128]) read as: the format's codes for random whole numbers r < 2^16, in float64; low: 14
    for m, 30 for v."""
    big = float(np.abs(x).max())
    if big > 1.875 * 2.0 ** 126:
        return np.full(128, np.nan)
    if big <= 0.875 * 2.0 ** -126:
        return np.zeros(128)
    frac, e = np.frexp(big)
    top = 2.0 ** max(e - 1 + (frac > 0.9375), -126)
    y = np.abs(x.astype(np.float64)) / top
    q = np.exp2(np.floor(np.log2(np.maximum(y, 2.0 ** -low))) - 3.0)
    n = np.floor(np.rint(y / q * 2.0 ** 20) / 2.0 ** 20 + r / 65536.0)
    if low == 30:
        n = np.where((y > 0) & (n < 1), 1.0, n)
    return np.sign(x) * n * q * top


def test_the_ends_of_the_8_bit_range():
    """Blocks whose largest moment is next to the least and to the largest that have codes (beta 0: m = g, v = g^2, which are exact
    here or rounded as on the CPU): zeros up to 0.875 2^-126, NaN above 1.875 2^126, the format's codes from one to the other."""
    ends = [np.array([bits], np.uint32).view(np.float32)[0] for bits in (0x6fffff, 0x700000, 0x700001, 0x700010, 0x7fffff, 0x800000,
                                                                         0x800001, 0xf00000, 0xf00001)]
    ends += [np.float32(k * 2.0 ** -75) for k in (3831, 3832, 4095, 4096, 5608, 5609, 5792)]   # their squares: 0.8748 2^-126 and on
    ends += [np.float32(k * 2.0 ** 51) for k in (4096, 5000, 5608)]      # up to 1.8746 2^126 ...
    past = [np.float32(k * 2.0 ** 51) for k in (5609, 5700, 5792, 6000)] + [np.float32(3e38)]   # ... and from 1.8752 2^126 on
    rng = np.random.default_rng(1)
    rows = []
    for end in ends + past:
        row = np.zeros(128, np.float32)
        row[::2] = end * rng.uniform(-1, 1, 64).astype(np.float32)
        row[17] = end
        rows.append(row)
    g = np.stack(rows)
    p = torch.zeros(g.size, device="cuda")
    st = [core.new_moments(p)]
    core.adamw([p], [torch.from_numpy(g.reshape(-1)).cuda()], st, step=1, lr=0.0, betas=(0.0, 0.0), seed=3)
    ms, vs = (x[0].cpu().numpy().reshape(g.shape) for x in read(st, [p]))
    u = mix((np.arange(g.size, dtype=np.int64) + mix((3 + 2654435761) & 0xffffffff)) & 0xffffffff).reshape(g.shape)
    with np.errstate(over="ignore", under="ignore"):
        squares = g * g
    for i, row in enumerate(g):
        m, v = stored(row, u[i] >> 16, 14), stored(squares[i], u[i] & 0xffff, 30)
        if np.isnan(v).any():
            m = v
        assert np.isnan(v).all() == (i >= len(ends)), i
        for got, want in ((ms[i], m), (vs[i], v)):
            assert np.array_equal(got, want.astype(np.float32), equal_nan=True), (i, row[17])


@pytest.mark.parametrize("full", [96, 108, 120, 191])
@pytest.mark.parametrize("more", [-1, 0, 1])
@pytest.mark.parametrize("copies", [1, 2])
def test_lists_at_the_edges_of_a_launch(full, more, copies):
    """Lists of as many tensors as a launch of the 32-bit step takes (96), of the 8-bit step (108), of read_moments (120), of the
    norm (191), one fewer and one more, and twice that; tensors without values among them, at the ends and at the edge."""
    count = full * copies + more
    gen = torch.Generator().manual_seed(count)
    sizes = [(int(n),) for n in torch.randint(1, 5000, (count,), generator=gen)]
    for at in (0, full - 1, full, count):   # which no launch's table holds
        sizes.insert(at, (0,))
    ps, gs = tensors(sizes, [torch.float32, torch.bfloat16, torch.bfloat16], count)
    want = sum(float(g.double().square().sum()) for g in gs) ** 0.5
    assert abs(float(core.grad_norm(gs)) - want) <= 2.0 ** -24 * 1.01 * want
    for bits in (32, 8):
        qs = [p.clone() for p in ps]
        twin = Twin(qs, bits, 5)
        if bits == 32:
            ms, vs = ([torch.zeros(p.shape, device="cuda") for p in qs] for _ in range(2))
            core.adamw(qs, gs, ms, vs, step=1, max_norm=1.0, **HYPER)
        else:
            st = [core.new_moments(p) for p in qs]
            core.adamw(qs, gs, st, step=1, max_norm=1.0, seed=5, **HYPER)
            ms, vs = read(st, qs)
        twin.step(gs, 1.0)
        twin.compare(qs, ms, vs)
