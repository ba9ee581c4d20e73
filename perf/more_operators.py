"""Workloads of the operators at the end of a training step, and of a token that is scored: the log probabilities of given
tokens with entropy, top alternatives and their gradient, the norm of a model's gradients, and the AdamW step over all of a
model's tensors with its moments in 32 or in 8 bits.

``run`` computes a case's operator in elementary torch ops (float32, sums of squares in float64, one rounding at the end) or,
with ``own`` set, through the framework's entry points; ``exact`` restates the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
# the sizes of the full-width models: vocabulary, and the benchmark's batch of 8 x 2,048 tokens
VOCAB, TOKENS = 32768, 8 * 2048
# the full-width model's layers: 12 heads of 64, addresses of 64, 32 sub-keys, a gated map of 2,048
FULL = dict(layers=12, heads=12, dh=64, d_a=64, n_sub=32, f=2048, V=VOCAB)


def listed():
    return [
        # a token of one user's stream: float32 logits, the five best alternatives shown beside it
        dict(name="logprob_decode_1", kind="logprob", N=1, V=VOCAB, dtype="f32", top=5, entropy=False, train=False, tau=1.0,
             mask=False),
        # a token of each of 64 streams behind a grammar's mask, some of which leaves fewer tokens than are asked for
        dict(name="logprob_decode_64", kind="logprob", N=64, V=VOCAB, dtype="bf16", top=20, entropy=True, train=False,
             tau=0.8, mask=True),
        # a packed float32 batch of an odd length over an odd vocabulary in a training step
        dict(name="logprob_train_odd_f32", kind="logprob", N=1537, V=32003, dtype="f32", top=0, entropy=True, train=True,
             tau=0.7, mask=False),
        # a teacher's best tokens over a large vocabulary, for a distillation loss
        dict(name="logprob_teacher_wide", kind="logprob", N=2048, V=151936, dtype="bf16", top=64, entropy=False, train=False,
             tau=1.0, mask=False),
        # the benchmark's batch in a training step with an entropy bonus
        dict(name="logprob_train_b8_t2048", kind="logprob", N=TOKENS, V=VOCAB, dtype="bf16", top=0, entropy=True, train=True,
             tau=1.0, mask=False),
        # the gradients of one layer of odd sizes
        dict(name="norm_one_layer_odd", kind="norm", layers=1, heads=5, dh=66, d_a=32, n_sub=16, f=881, V=1003, dtype="f32"),
        # the gradients of the full-width model, before they are clipped
        dict(name="norm_full_bf16", kind="norm", dtype="bf16", **FULL),
        # a test model's step
        dict(name="adamw_small", kind="adamw", layers=2, heads=4, dh=32, d_a=32, n_sub=16, f=344, V=2048, dtype="f32", bits=32,
             clip=False),
        # odd sizes, moments in 8 bits with blocks that end inside the tensors' rows and at their ends
        dict(name="adamw8_odd_f32", kind="adamw", layers=3, heads=5, dh=66, d_a=32, n_sub=16, f=881, V=32003, dtype="f32",
             bits=8, clip=True),
        # the full-width model trained under autocast: float32 weights and moments, clipped gradients
        dict(name="adamw_full_f32", kind="adamw", dtype="f32", bits=32, clip=True, **FULL),
        # the same in bfloat16 with moments in 8 bits
        dict(name="adamw8_full_bf16", kind="adamw", dtype="bf16", bits=8, clip=True, **FULL),
        # a wider model with a large vocabulary: bfloat16 weights, moments in float32
        dict(name="adamw_wide_bf16", kind="adamw", layers=12, heads=16, dh=64, d_a=64, n_sub=32, f=2752, V=131072,
             dtype="bf16", bits=32, clip=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("logprob", "logprob", "norm", "adamw", "adamw"))
    dtype = rng.choice(("bf16", "f32"))
    if kind == "logprob":
        V = _log_int(rng, 500, 151936)
        if rng.random() < 0.5:
            V = (V + 127) // 128 * 128
        train = rng.random() < 0.5
        N = _log_int(rng, 1, min(TOKENS, (TOKENS * VOCAB // (2 if train else 1) // (1 if dtype == "bf16" else 2)) // V))
        top = 0 if rng.random() < (0.7 if train else 0.1) else _log_int(rng, 1, 128)
        return dict(kind=kind, N=N, V=V, dtype=dtype, top=top, entropy=rng.random() < 0.6, train=train,
                    tau=rng.choice((1.0, 1.0, 0.6, 1.5)), mask=rng.random() < 0.3)
    dh = rng.choice((8, 16, 32, 33, 64, 66))
    heads = rng.randint(2, 1024 // dh if dh > 32 else 16)
    sizes = dict(layers=_log_int(rng, 1, 12), heads=heads, dh=dh, d_a=rng.choice((16, 32, 64)), n_sub=rng.choice((8, 16, 32)),
                 f=_log_int(rng, 50, 2752), V=_log_int(rng, 500, 65536))
    if kind == "norm":
        return dict(kind=kind, dtype=dtype, **sizes)
    return dict(kind=kind, dtype=dtype, bits=rng.choice((32, 8)), clip=rng.random() < 0.6, **sizes)


def _shapes(case):
    """The parameters of a model: embedding, per layer the mixer's and the gated map's, the last norm's."""
    H, dh, a, n, f, V = (case[k] for k in ("heads", "dh", "d_a", "n_sub", "f", "V"))
    d = H * dh
    layer = [(d,), (H * a, d), (H * a, d), (d, d), (H, d), (H,), (d, d), (H, n, a // 2), (H, n, a // 2), (H,), (H, dh),
             (d,), (f, d), (f, d), (d, f)]
    return [(V, d)] + layer * case["layers"] + [(d,)]


# -- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 29)
    return (_prepare_logprob if case["kind"] == "logprob" else _prepare_step)(case, g)


def _prepare_logprob(case, g):
    N, V, dt = case["N"], case["V"], DT[case["dtype"]]
    z = torch.randn((N, V), generator=g, device=DEV, dtype=dt).mul_(1.5)
    # targets that repeat as text repeats them, most of them among the tokens that the model finds likely
    u = torch.rand((N,), generator=g, device=DEV, dtype=torch.float64)
    y = torch.exp(u * math.log(V)).long().clamp_(0, V - 1)
    z[torch.arange(N, device=DEV), y] += (torch.rand((N,), generator=g, device=DEV) * 12.0).to(dt)
    if case["mask"]:   # half of a grammar's tokens; the last row is left three of them, its target among them
        z.masked_fill_(torch.rand((N, V), generator=g, device=DEV) < 0.5, -math.inf)
        z[N - 1] = -math.inf
        z[N - 1, torch.stack([y[N - 1], (y[N - 1] + V // 3) % V, (y[N - 1] + V // 2) % V])] = torch.tensor(
            [0.5, 1.0, 1.0], device=DEV, dtype=dt)
    st = dict(case=case, logits=z.requires_grad_(case["train"]))
    if N > 16:   # the padded end of a batch
        y[N - N // 16:N - 1] = -100
    st["targets"] = y
    if case["train"]:
        there = (y != -100).float()
        st["g_logprob"] = torch.randn((N,), generator=g, device=DEV) * there / N
        st["g_entropy"] = torch.rand((N,), generator=g, device=DEV) * there * (0.1 / N) if case["entropy"] else None
    return st


BLOCK = 128   # values that share an exponent in the 8-bit moments
PITCH = 264   # a block's bytes there: 128 codes of the first moment, 128 of the second, their exponents, 6 unused


def _prepare_step(case, g):
    dt = DT[case["dtype"]]
    shapes = _shapes(case)
    blocks = [-(-math.prod(s) // BLOCK) for s in shapes]
    total = sum(blocks)
    at, starts = 0, []
    for b in blocks:
        starts.append(at)
        at += b

    def normal():
        return torch.randn((total * BLOCK,), generator=g, device=DEV)

    def views(flat):   # each tensor begins a block of its own, as an allocator's tensors begin where they are aligned
        return [flat[s * BLOCK:s * BLOCK + math.prod(sh)].view(sh) for s, sh in zip(starts, shapes)]

    st = dict(case=case, t=100)
    there = torch.zeros(total * BLOCK, device=DEV)   # zero in the gaps between tensors
    scale = torch.ones(total * BLOCK, device=DEV)
    for v, s, size in zip(views(there), views(scale), (10.0 ** (-2.0 - 3.0 * torch.rand((len(shapes),), generator=g,
                                                                                         device=DEV))).tolist()):
        v.fill_(1.0)
        s.fill_(size)   # gradients of a tensor are alike in size, those of different tensors are not
    emb = views(there)[0]
    rows = emb.shape[0]
    seldom = torch.rand((rows,), generator=g, device=DEV)
    emb[seldom < 0.4] = 0.0   # tokens that have not come up
    grad = normal() * (0.3 + torch.rand((total * BLOCK,), generator=g, device=DEV)) * scale * there
    st["grad"] = grad.to(dt)
    st["grads"] = views(st["grad"])
    if case["kind"] == "norm":
        return st
    st["param"] = (normal() * 0.02 * there).to(dt)
    st["params"] = views(st["param"])
    m = normal().mul_(0.3).mul_(scale).mul_(there)
    v = torch.rand((total * BLOCK,), generator=g, device=DEV).add_(0.2).mul_(scale).mul_(scale).mul_(there)
    if case["bits"] == 32:
        st["m"], st["v"] = m, v
        st["ms"], st["vs"] = views(m), views(v)
    else:
        st["moments"] = _encode(m, v, 0, 0)
        st["states"] = [st["moments"][s:s + b] for s, b in zip(starts, blocks)]
        # where the values that the codes stand for are read to
        st["m"], st["v"] = torch.zeros(2, total * BLOCK, dtype=torch.bfloat16, device=DEV)
        st["ms"], st["vs"] = views(st["m"]), views(st["v"])
    return st


# the constants of a training step
STEP = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
MAX_NORM, SEED = 1.0, 12345


# -- one pass ----------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if case["kind"] == "adamw":
        st["t"] += 1
    if own:
        return _run_own(st, case)
    return {"logprob": _logprob_plain, "norm": _norm_plain, "adamw": _adamw_plain}[case["kind"]](st, case)


def _run_own(st, case):
    from sdmchat_amd import core

    if case["kind"] == "logprob":
        r = core.token_logprobs(st["logits"], st["targets"], temperature=case["tau"], entropy=case["entropy"],
                                top=case["top"])
        out = dict(logprobs=r.logprobs.detach())
        if case["entropy"]:
            out["entropy"] = r.entropy.detach()
        if case["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        if case["train"]:
            outs, grads = ([r.logprobs, r.entropy], [st["g_logprob"], st["g_entropy"]]) if case["entropy"] else (
                [r.logprobs], [st["g_logprob"]])
            out["grad"] = torch.autograd.grad(outs, st["logits"], grads)[0]
        return out
    if case["kind"] == "norm":
        return core.grad_norm(st["grads"])
    out = dict(param=st["param"], m=st["m"], v=st["v"])
    if case["bits"] == 32:
        norm = core.adamw(st["params"], st["grads"], st["ms"], st["vs"], step=st["t"],
                          max_norm=MAX_NORM if case["clip"] else None, **STEP)
    else:
        norm = core.adamw(st["params"], st["grads"], st["states"], step=st["t"], seed=SEED,
                          max_norm=MAX_NORM if case["clip"] else None, **STEP)
        core.read_moments(st["states"], st["ms"], st["vs"])
    if case["clip"]:
        out["norm"] = norm
    return out


def _logprob_plain(st, case):
    z, y, V, tau = st["logits"].detach(), st["targets"], case["V"], case["tau"]
    x = z.float()
    given = y >= 0
    at = torch.where(given, y, 0)[:, None]
    x = (x - x.amax(1, keepdim=True)) / tau
    e = torch.exp(x)
    s = e.sum(1, keepdim=True)
    x = x - torch.log(s)
    e = e / s
    out = dict(logprobs=torch.where(given, torch.gather(x, 1, at)[:, 0], 0.0))
    if case["entropy"]:
        xf = torch.where(e > 0, x, 0.0)
        h = -(e * xf).sum(1)
        out["entropy"] = h
    if case["top"]:
        # one whole number a token, greater for a greater logit and, at equal logits, for a lower id
        bits = z.float().add(0.0).view(torch.int32)   # -0 as 0
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
        key = (order << 32) + (V - 1 - torch.arange(V, device=z.device))
        key = torch.topk(key, min(case["top"], V), dim=1).values
        ids = V - 1 - (key & 0xffffffff)
        best = torch.gather(x, 1, ids)
        pad = (0, case["top"] - ids.shape[1])
        out["top_ids"] = torch.nn.functional.pad(torch.where(best == -math.inf, -1, ids), pad, value=-1)
        out["top_logprobs"] = torch.nn.functional.pad(best, pad, value=-math.inf)
    if case["train"]:
        grad = e * -st["g_logprob"][:, None]
        if case["entropy"]:
            grad = grad - e * (xf + h[:, None]) * st["g_entropy"][:, None]
        grad.scatter_add_(1, at, torch.where(given, st["g_logprob"], 0.0)[:, None])
        out["grad"] = (grad / tau).to(z.dtype)
    return out


def _norm_plain(st, case):
    return torch.sqrt(st["grad"].double().square().sum()).float()


def _adamw_plain(st, case):
    lr, (b1, b2), eps, wd = STEP["lr"], STEP["betas"], STEP["eps"], STEP["weight_decay"]
    t = st["t"]
    g = st["grad"].float()
    out = {}
    if case["clip"]:
        out["norm"] = norm = _norm_plain(st, case)
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    if case["bits"] == 32:
        m, v = st["m"], st["v"]
    else:
        m, v = _decode(st["moments"])
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g * g * (1.0 - b2)
    p = st["param"].float()
    p = p * (1.0 - lr * wd) - m / (torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2 ** t)) + eps) * (lr / (1.0 - b1 ** t))
    st["param"].copy_(p)
    if case["bits"] == 32:
        st["m"].copy_(m)
        st["v"].copy_(v)
    else:
        st["moments"].copy_(_encode(m, v, SEED, t))
        m, v = _decode(st["moments"])
        st["m"].copy_(m)   # 4 bits of a value: bfloat16 holds them
        st["v"].copy_(v)
    out.update(param=st["param"], m=st["m"], v=st["v"])
    return out


# The moments in 8 bits.  A block's exponent E is that of its largest magnitude a, one more where a's mantissa is over 1.875:
# then all its values over 2^(E - 127) are at most 1.875.  Those of the first moment have a sign, 4 bits of exponent and 3 of
# mantissa, those of the second 5 and 3, and 2^-14 and 2^-30 are the least that are normal.  A value between two codes takes
# the upper one with the probability that its place between them says, by 16 bits of a hash of its position; a second moment
# above zero has no code 0.
_A, _B, _MASK = 2654435761, 3144134277, 0xffffffff   # of the golden ratio and of the square root of 3


def _mix(x):
    x = ((x ^ (x >> 16)) * _A) & _MASK
    x = ((x ^ (x >> 15)) * _B) & _MASK
    return x ^ (x >> 16)


def _encode_one(x, u, top):
    """Magnitude codes and exponents of x [blocks, 128] with random whole numbers u < 2^16; top: the largest code's exponent
    field."""
    bits = x.abs().amax(1, keepdim=True).view(torch.int32)
    E = (bits + 0xfffff) >> 23
    y = x.abs() * ((254 - E) << 23).view(torch.float32)
    # where the least normal value of the code is the least of float32, the code is its first bits
    y = y * 2.0 ** (top - 127)
    code = (y.view(torch.int32) + (u << 4)) >> 20
    return torch.where(E > 0, code, 0), E


def _encode(m, v, seed, t):
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    key = _mix((torch.tensor(seed) + t * _A) & _MASK).item()
    u = _mix((torch.arange(m.numel(), device=m.device) + key) & _MASK).view(-1, BLOCK)
    cm, em = _encode_one(m, (u >> 16).int(), 15)
    cv, ev = _encode_one(v, (u & 0xffff).int(), 31)
    cv = torch.where((v > 0) & (ev > 0), cv.clamp(min=1), cv)
    cm = cm + (m < 0) * 128
    none = torch.zeros(m.shape[0], PITCH - 2 * BLOCK - 2, dtype=torch.int32, device=m.device)
    return torch.cat([cm, cv, em, ev, none], 1).to(torch.uint8)


def _decode(moments):
    cm, cv, em, ev = (x.int() for x in moments[:, :2 * BLOCK + 2].split([BLOCK, BLOCK, 1, 1], 1))
    m = ((cm & 127) << 20).view(torch.float32) * 2.0 ** 112 * (em << 23).view(torch.float32)
    v = (cv << 20).view(torch.float32) * 2.0 ** 96 * (ev << 23).view(torch.float32)
    return torch.where(cm > 127, -m, m).view(-1), v.view(-1)


# -- the least that a pass reads, writes and computes ------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "logprob":
        N, V, K = case["N"], case["V"], case["top"]
        nbytes = N * V * es + N * 12 + N * K * 12 + N * 4 * case["entropy"]
        flops = N * V * (5 + 2 * case["entropy"])
        if case["train"]:
            nbytes += N * V * es + N * 4 * (1 + case["entropy"])
            flops += N * V * (3 + 3 * case["entropy"])
        return {"bytes": nbytes, "flops": flops}
    n = sum(math.prod(s) for s in _shapes(case))
    if case["kind"] == "norm":
        return {"bytes": n * es + 4, "flops": 2 * n}
    blocks = sum(-(-math.prod(s) // BLOCK) for s in _shapes(case))
    # parameter and gradient in, parameter out; both moments in and out, in 8 bits the values that they stand for out too
    state = 16 * n if case["bits"] == 32 else 4 * BLOCK * blocks + 4 * blocks + 4 * n
    return {"bytes": 3 * n * es + state, "flops": n * (14 + 2 * case["clip"] + 24 * (case["bits"] == 8))}


# -- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"logprob": _logprob_exact, "norm": _norm_exact, "adamw": _adamw_exact}[case["kind"]](st, case)


def _logprob_exact(st, case):
    N, V, K = case["N"], case["V"], case["top"]
    z, y = st["logits"].detach(), st["targets"]
    parts = []
    rows = max(1, (1 << 26) // V)
    for a in range(0, N, rows):
        zi = z[a:a + rows].double() / case["tau"]
        yi = y[a:a + rows]
        lp = torch.log_softmax(zi, 1)
        hot = torch.zeros_like(lp)
        real = torch.nonzero(yi >= 0)[:, 0]
        hot[real, yi[real]] = 1.0
        part = dict(logprobs=torch.where(hot > 0, lp, 0.0).sum(1))
        p = torch.exp(lp)
        h = torch.special.entr(p).sum(1)
        if case["entropy"]:
            part["entropy"] = h
        if K:
            best = lp.sort(1, descending=True).values[:, :K]
            part["top_logprobs"] = torch.cat([best, torch.full((best.shape[0], K - best.shape[1]), -math.inf,
                                                               device=DEV, dtype=torch.float64)], 1)
        if case["train"]:
            gl = st["g_logprob"][a:a + rows, None].double()
            d = hot * gl - p * gl
            if case["entropy"]:
                ge = st["g_entropy"][a:a + rows, None].double()
                d += ge * (torch.special.entr(p) - p * h[:, None])
            part["grad"] = d / case["tau"]
        parts.append(part)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _norm_exact(st, case):
    return sum(torch.linalg.vector_norm(g.double()) ** 2 for g in st["grads"]) ** 0.5


def _adamw_exact(st, case):
    lr, (b1, b2), eps, wd = STEP["lr"], STEP["betas"], STEP["eps"], STEP["weight_decay"]
    t = st["t"] + 1
    g, p = st["grad"].double(), st["param"].double()
    out = {}
    if case["clip"]:
        out["norm"] = norm = _norm_exact(st, case)
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m, v = (st["m"].double(), st["v"].double()) if case["bits"] == 32 else _values_exact(st["moments"])
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    step = m / (1.0 - b1 ** t) / (torch.sqrt(v / (1.0 - b2 ** t)) + eps)
    out["param"] = p - lr * (wd * p + step)
    if case["bits"] == 8:
        m, v = _round_exact(m, v, SEED, t)
    out["m"], out["v"] = m, v
    return out


def _values_exact(moments):
    cm, cv = moments[:, :BLOCK].long(), moments[:, BLOCK:2 * BLOCK].long()
    em, ev = (moments[:, 2 * BLOCK + k:2 * BLOCK + k + 1].double() - 127.0 for k in (0, 1))
    both = []
    for sign, mag, e, low in ((1.0 - 2.0 * (cm // 128), cm % 128, em, 14), (1.0, cv, ev, 30)):
        field, frac = mag // 8, (mag % 8).double()
        x = torch.where(field > 0, (8.0 + frac) * torch.exp2(field.double() - low - 4.0), frac * 2.0 ** (-low - 3))
        both.append((sign * x * torch.exp2(e)).reshape(-1))
    return both


def _round_exact(m, v, seed, t):
    """The values between codes put up or down by the hash, from the quantum of each value."""
    A, B = 2654435761, 3144134277

    def mixed(x):
        x = (x ^ (x >> 16)) * A & 0xffffffff
        x = (x ^ (x >> 15)) * B & 0xffffffff
        return x ^ (x >> 16)
    u = mixed((torch.arange(m.numel(), device=DEV) + mixed((seed + t * A) & 0xffffffff)) & 0xffffffff)
    both = []
    for x, r, low in ((m, u >> 16, 14), (v, u & 0xffff, 30)):
        size = x.view(-1, BLOCK).abs().amax(1)
        frac, e = torch.frexp(size)
        top = torch.exp2((e - 1 + (frac > 0.9375)).double()).repeat_interleave(BLOCK)   # 2^(E - 127)
        tiny = top < 2.0 ** -126
        y = x.abs() / torch.where(size.repeat_interleave(BLOCK) > 0, top, 1.0)
        quantum = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -low))) - 3.0)
        n = torch.floor(y / quantum + r.double() / 65536.0)
        if low == 30:
            n = torch.where((y > 0) & (n < 1), 1.0, n)
        both.append(torch.where(tiny, 0.0, torch.sign(x) * n * quantum * top))
    return both
