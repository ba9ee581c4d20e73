"""Workloads of the operators at the two ends of the vocabulary: the scaled embedding lookup with its gradient, the
distillation loss from a teacher's top logits with its gradient, and the rules of a decode step on its logits (penalties
for repeated tokens, a bias, a grammar mask).

``run`` computes a case's operator in elementary torch ops (float32, one rounding at the end) or, with ``own`` set,
through the framework's entry points; ``exact`` restates the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
# the sizes of the full-width models: vocabulary, layer width, and the benchmark's batch of 8 x 2,048 tokens
VOCAB, WIDTH, TOKENS = 32768, 768, 8 * 2048


def listed():
    return [
        # the tokens of 64 decode streams looked up
        dict(name="embed_decode_64", kind="embed", N=64, V=VOCAB, d=WIDTH, dtype="bf16", train=False, pad=False),
        # the benchmark's batch in a training step: lookup and the whole table's gradient
        dict(name="embed_train_b8_t2048", kind="embed", N=TOKENS, V=VOCAB, d=WIDTH, dtype="bf16", train=True, pad=False),
        # a packed batch of an odd length, padded, on float32 weights of a width that is no multiple of 4
        dict(name="embed_train_odd_f32", kind="embed", N=5003, V=32003, d=330, dtype="f32", train=True, pad=True),
        # long documents on a wide model with a large vocabulary
        dict(name="embed_train_131072", kind="embed", N=131072, V=131072, d=1024, dtype="bf16", train=True, pad=True),
        # one short sequence of a fine-tuning step
        dict(name="distill_64", kind="distill", N=64, V=VOCAB, K=16, dtype="bf16", tau=1.0, alpha=1.0),
        # the float32 validation shape with labels
        dict(name="distill_f32_b1_t1024", kind="distill", N=1024, V=VOCAB, K=8, dtype="f32", tau=1.0, alpha=0.5),
        # a batch of an odd length over an odd vocabulary, some positions without a target
        dict(name="distill_odd", kind="distill", N=1537, V=32003, K=50, dtype="bf16", tau=1.5, alpha=0.7),
        # a few rows over a large vocabulary
        dict(name="distill_wide", kind="distill", N=512, V=151936, K=100, dtype="bf16", tau=2.0, alpha=0.9),
        # the benchmark's batch in a training step
        dict(name="distill_b8_t2048", kind="distill", N=TOKENS, V=VOCAB, K=32, dtype="bf16", tau=2.0, alpha=0.5),
        # a token of one user's stream, float32 logits, all rules
        dict(name="rules_1", kind="rules", B=1, V=VOCAB, L=300, dtype="f32", bias=True, mask=True),
        # a token of each of 64 streams, all rules
        dict(name="rules_64", kind="rules", B=64, V=VOCAB, L=2048, dtype="bf16", bias=True, mask=True),
        # a serving batch over a large odd vocabulary with long histories, penalties alone
        dict(name="rules_256_wide", kind="rules", B=256, V=131071, L=8192, dtype="bf16", bias=False, mask=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("embed", "distill", "rules"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind == "embed":
        d = _log_int(rng, 48, 1536)
        if rng.random() < 0.6:
            d = (d + 63) // 64 * 64
        V = _log_int(rng, 1000, 131072)
        N = _log_int(rng, 1, min(131072, (1 << 27) // d))
        return dict(kind=kind, N=N, V=V, d=d, dtype=dtype, train=rng.random() < 0.75, pad=rng.random() < 0.5)
    if kind == "distill":
        V = _log_int(rng, 500, 151936)
        if rng.random() < 0.5:
            V = (V + 127) // 128 * 128
        N = _log_int(rng, 1, min(TOKENS, (TOKENS * VOCAB // 4) // V))
        labels = rng.random() < 0.6
        return dict(kind=kind, N=N, V=V, K=_log_int(rng, 1, 128), dtype=dtype, tau=rng.choice((1.0, 1.0, 1.5, 2.0, 4.0)),
                    alpha=rng.choice((0.3, 0.5, 0.9)) if labels else 1.0)
    V = _log_int(rng, 500, 151936)
    if rng.random() < 0.5:
        V = (V + 63) // 64 * 64
    return dict(kind=kind, B=_log_int(rng, 1, 256), V=V, L=_log_int(rng, 1, 8192), dtype=dtype,
                bias=rng.random() < 0.6, mask=rng.random() < 0.6)


# -- inputs ------------------------------------------------------------------------------------------------------------
def _zipf(g, shape, V):
    """Token ids that repeat as text repeats them: the r-th most frequent one has a share of about 1 / (r ln V)."""
    u = torch.rand(shape, generator=g, device=DEV, dtype=torch.float64)
    r = torch.exp(u * math.log(V + 1)).long().clamp_(1, V) - 1
    return (r * 7919 + 11) % V if V % 7919 else r


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    dt = DT[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    st = dict(case=case)
    if case["kind"] == "embed":
        N, V, d = case["N"], case["V"], case["d"]
        st["table"] = (normal(V, d) * 0.02).to(dt).requires_grad_(case["train"])
        st["ids"] = _zipf(g, (N,), V)
        st["scale"] = math.sqrt(d)
        st["pad"] = 0 if case["pad"] else None
        if case["pad"]:   # the padded end of a batch
            st["ids"][N - N // 16:] = 0
        if case["train"]:
            st["dy"] = normal(N, d, dtype=dt)
    elif case["kind"] == "distill":
        N, V, K = case["N"], case["V"], case["K"]
        # a teacher's K best tokens, distinct, their logits falling from the best on; the student roughly agrees
        K = min(K, V)
        first = _zipf(g, (N, 1), V)
        stride = torch.randint(1, max(2, V // K), (N, 1), generator=g, device=DEV)
        ids = (first + stride * torch.arange(K, device=DEV)) % V
        top = 9.0 - torch.cumsum(torch.rand((N, K), generator=g, device=DEV) * (8.0 / K), 1) + normal(N, 1) * 0.5
        z = normal(N, V, dtype=dt).mul_(1.5)
        z.scatter_(1, ids, (top + normal(N, K)).to(dt))
        live = torch.randint(1, K + 1, (N, 1), generator=g, device=DEV)   # entries of a row that the teacher kept
        live = torch.where(torch.rand((N, 1), generator=g, device=DEV) < 0.25, live, K)
        st["labels"] = None
        if case["alpha"] < 1.0:
            labels = torch.where(torch.rand((N,), generator=g, device=DEV) < 0.7, ids[:, 0], _zipf(g, (N,), V))
            st["labels"] = torch.where(torch.rand((N,), generator=g, device=DEV) < 0.05, -100, labels)
        if N > 16:   # the padded end of a batch: no target at all
            live[N - N // 16:] = 0
            if st["labels"] is not None:
                st["labels"][N - N // 16:] = -100
        st["ids"] = torch.where(torch.arange(K, device=DEV) < live, ids, -1)
        st["top"] = top
        st["logits"] = z.requires_grad_(True)
    else:
        B, V, L = case["B"], case["V"], case["L"]
        st["logits"] = normal(B, V).mul_(3.0).to(dt)
        st["tokens"] = _zipf(g, (B, L), V)
        st["lengths"] = torch.randint(L // 2, L + 1, (B,), generator=g, device=DEV)   # ragged histories
        st["prompt"] = (st["lengths"].double() * torch.rand((B,), generator=g, device=DEV, dtype=torch.float64)).long()
        st["repetition"] = 1.0 + 0.5 * torch.rand((B,), generator=g, device=DEV)
        st["frequency"] = 0.4 * torch.rand((B,), generator=g, device=DEV)
        st["presence"] = 0.6 * torch.rand((B,), generator=g, device=DEV)
        st["bias"] = st["mask"] = None
        if case["bias"]:   # a few tokens raised, lowered or banned
            b = torch.zeros(V, device=DEV)
            at = torch.randint(0, V, (max(1, V // 200),), generator=g, device=DEV)
            b[at] = normal(at.numel()) * 2.0
            b[at[:1]] = -math.inf
            st["bias"] = b
        if case["mask"]:   # a grammar allows about half the words of 32 tokens, each in part
            W = (V + 31) // 32
            bits = torch.randint(-2**31, 2**31, (B, W), generator=g, device=DEV)
            st["mask"] = torch.where(torch.rand((B, W), generator=g, device=DEV) < 0.5, bits, 0).to(torch.int32)
    return st


# -- one pass ----------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    return {"embed": _embed_plain, "distill": _distill_plain, "rules": _rules_plain}[case["kind"]](st, case)


def _run_own(st, case):
    from sdmchat_amd import core

    if case["kind"] == "embed":
        y = core.embedding(st["ids"], st["table"], scale=st["scale"], padding_idx=st["pad"])
        if not case["train"]:
            return y
        return [y.detach(), torch.autograd.grad(y, st["table"], st["dy"])[0]]
    if case["kind"] == "distill":
        loss = core.distill_loss(st["logits"], st["ids"], st["top"], temperature=case["tau"], labels=st["labels"],
                                 alpha=case["alpha"])
        return [loss.detach(), torch.autograd.grad(loss, st["logits"])[0]]
    return core.process_logits(st["logits"], st["tokens"], st["lengths"], prompt=st["prompt"],
                               repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                               bias=st["bias"], mask=st["mask"])


def _embed_plain(st, case):
    table, ids = st["table"].detach(), st["ids"]
    y = (table[ids].float() * st["scale"]).to(table.dtype)
    if not case["train"]:
        return y
    dt = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    dt.index_add_(0, ids, st["dy"].float())
    if st["pad"] is not None:
        dt[st["pad"]] = 0.0
    return [y, (dt * st["scale"]).to(table.dtype)]


def _distill_plain(st, case):
    logits, ids, top, labels = st["logits"].detach(), st["ids"], st["top"], st["labels"]
    tau, alpha = case["tau"], case["alpha"]
    z = logits.float()
    live = ids >= 0
    at = ids.clamp(min=0)
    taught = live.any(1)
    # the teacher's distribution over its live entries (zeros where a row has none)
    t = torch.where(live, top / tau, -math.inf)
    tm = torch.where(taught, t.amax(1), 0.0)[:, None]
    te = torch.exp(t - tm)
    ts = te.sum(1, keepdim=True).clamp(min=1e-30)
    q = te / ts
    logq = torch.where(live, t - tm - torch.log(ts), 0.0)
    # the student's
    m = z.amax(1, keepdim=True)
    zc = z - m
    e = torch.exp(zc / tau)
    s = e.sum(1, keepdim=True)
    logp = torch.gather(zc, 1, at) / tau - torch.log(s)
    target = taught
    loss = alpha * tau * tau * (q * (logq - logp)).sum(1)
    grad = (e / s * taught[:, None] * (alpha * tau)).scatter_add_(1, at, q * (-alpha * tau))
    if labels is not None:
        has = labels != -100
        lab = torch.where(has, labels, 0)[:, None]
        target = taught | has
        e1 = torch.exp(zc)
        s1 = e1.sum(1, keepdim=True)
        ce = torch.log(s1) - torch.gather(zc, 1, lab)
        loss = loss + torch.where(has, (1.0 - alpha) * ce[:, 0], 0.0)
        e1 = e1 / s1 * has[:, None] * (1.0 - alpha)
        grad = grad + e1.scatter_add_(1, lab, has[:, None] * -(1.0 - alpha))
    w = 1.0 / target.sum().clamp(min=1)
    return [loss.sum() * w, (grad * w).to(logits.dtype)]


def _rules_plain(st, case):
    logits, tokens, V = st["logits"], st["tokens"], case["V"]
    x = logits.float()
    at = torch.arange(tokens.shape[1], device=tokens.device)
    there = at < st["lengths"][:, None]
    said = there & (at >= st["prompt"][:, None])
    zeros = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    seen = zeros.scatter_add(1, tokens, there.float()) > 0
    count = zeros.scatter_add(1, tokens, said.float())
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (count * st["frequency"][:, None] + (count > 0) * st["presence"][:, None])
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["mask"] is not None:
        v = torch.arange(V, device=x.device)
        allowed = (st["mask"][:, v // 32] >> (v % 32).int()) & 1
        x = torch.where(allowed != 0, x, -math.inf)
    return x.to(logits.dtype)


# -- the least that a pass reads, writes and computes ------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "embed":
        N, V, d = case["N"], case["V"], case["d"]
        rows = min(N, V)
        nbytes, flops = N * 8 + rows * d * es + N * d * es, N * d
        if case["train"]:
            nbytes += N * d * es + V * d * es
            flops += N * d + rows * d
        return {"bytes": nbytes, "flops": flops}
    if case["kind"] == "distill":
        N, V, K = case["N"], case["V"], case["K"]
        sums = 1 if case["alpha"] == 1.0 or case["tau"] == 1.0 else 2   # softmaxes of a row
        return {"bytes": 2 * N * V * es + N * K * 12 + N * 8 * (case["alpha"] < 1.0), "flops": N * V * 8 * sums}
    B, V, L = case["B"], case["V"], case["L"]
    nbytes = 2 * B * V * es + B * L * 8 + (V * 4 if case["bias"] else 0) + (B * ((V + 31) // 32) * 4 if case["mask"] else 0)
    return {"bytes": nbytes, "flops": B * V * 6}


# -- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"embed": _embed_exact, "distill": _distill_exact, "rules": _rules_exact}[case["kind"]](st, case)


def _embed_exact(st, case):
    table, ids = st["table"].detach().double(), st["ids"]
    y = torch.index_select(table, 0, ids) * st["scale"]
    if not case["train"]:
        return y
    dy = st["dy"].double() * st["scale"]
    if st["pad"] is not None:
        dy[ids == st["pad"]] = 0.0
    return [y, torch.zeros_like(table).index_put_((ids,), dy, accumulate=True)]


def _distill_exact(st, case):
    N, V, K = case["N"], case["V"], case["K"]
    tau, alpha = case["tau"], case["alpha"]
    logits, labels = st["logits"].detach(), st["labels"]
    grad = torch.empty(N, V, dtype=torch.float64, device=DEV)
    loss = torch.zeros((), dtype=torch.float64, device=DEV)
    rows = max(1, (1 << 26) // V)
    n_target = 0
    for a in range(0, N, rows):
        z = logits[a:a + rows].double()
        ids, top = st["ids"][a:a + rows], st["top"][a:a + rows].double()
        kept = (ids >= 0).double()
        has_t = kept.amax(1)
        w = torch.exp((top - 9.0) / tau) * kept
        q = w / w.sum(1).clamp(min=1e-300)[:, None]
        logp = torch.log_softmax(z / tau, 1)
        dense = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
        cross = -(q * logp.gather(1, ids.clamp(min=0))).sum(1)
        entropy = -torch.special.xlogy(q, q).sum(1)
        loss += (alpha * tau ** 2 * (cross - entropy)).sum()
        g = alpha * tau * (torch.exp(logp) * has_t[:, None] - dense)
        target = has_t > 0
        if labels is not None:
            y = labels[a:a + rows]
            has = y >= 0
            logp = torch.log_softmax(z, 1)
            pick = logp.gather(1, y.clamp(min=0)[:, None])[:, 0]
            loss -= (1 - alpha) * (pick * has).sum()
            one = torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], 1.0)
            g += (1 - alpha) * has[:, None] * (torch.exp(logp) - one)
            target = target | has
        n_target += int(target.sum())
        grad[a:a + rows] = g
    return [loss / max(n_target, 1), grad.div_(max(n_target, 1))]


def _rules_exact(st, case):
    B, V = case["B"], case["V"]
    out = st["logits"].double()
    for b in range(B):
        n, p = int(st["lengths"][b]), int(st["prompt"][b])
        r, f, pr = (float(st[k][b]) for k in ("repetition", "frequency", "presence"))
        ever = torch.bincount(st["tokens"][b, :n], minlength=V) > 0
        count = torch.bincount(st["tokens"][b, p:n], minlength=V)
        x = out[b]
        x = torch.where(ever & (x > 0), x / r, torch.where(ever, x * r, x))
        x = x - f * count - pr * (count > 0)
        if st["bias"] is not None:
            x = x + st["bias"].double()
        if st["mask"] is not None:
            shifts = torch.arange(32, device=DEV, dtype=torch.int64)
            bits = ((st["mask"][b].long()[:, None] >> shifts) & 1).reshape(-1)[:V]
            x = x.masked_fill(bits == 0, -math.inf)
        out[b] = x
    return out
