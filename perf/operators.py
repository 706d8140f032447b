"""Measured workloads of the token-distribution operators: the teacher's top-k log-probs, the
distillation losses and the cross entropies, each on logits in memory and (the losses) through the
LM head without logits.

`listed()` gives the cases, `draw(rng)` more of the same ranges; `prepare(case, seed)` makes a
case's inputs on the GPU, `run(state)` is one pass: the framework's operators where `own` is true,
otherwise their formulas in elementary torch operations.  `exact(case, seed)` is the same pass
from the definitions in 64 bits, and `work(case)` the bytes and operations no pass can avoid.

Formulas (z = x / temperature, p = softmax(z), a row's teacher entries (i_k, l_k), q_k = exp(l_k)):
an entry counts if i_k >= 0 and l_k > -inf, and a repeated id only at its first place.  With the
tail, the outcomes are the entries and one more, "any other token", of teacher mass 1 - sum q (none
below 2^-20) and student mass p_t.  forward KL(q|p); reverse KL(p|q); jsd b KL(q|m) + (1-b) KL(p|m)
with m = b q + (1-b) p; forward without the tail renormalises q over the entries.  A row without
entries gives 0.  Cross entropy with smoothing e and z weight c: (lse - x_y) + e (x_y - mean x) +
c lse^2, rows with target -100 give 0.
"""

import math

import torch

own = False

VOCAB = 151936  # the vocabulary of the repository's benchmark workloads
TAIL_EPS = 2.0 ** -20


def listed():
    return [
        # One decoding step of eight sequences that reports the likeliest tokens: latency.
        dict(name="topk-decode", op="topk", N=8, V=VOCAB, K=20, dtype="bf16", temperature=1.0),
        # A teacher's pass over 4096 tokens, the rows of the benchmark's logits workload.
        dict(name="topk-teacher", op="topk", N=4096, V=VOCAB, K=64, dtype="bf16", temperature=1.0),
        # An odd vocabulary in 32 bits with many entries a row, at a softening temperature.
        dict(name="topk-odd", op="topk", N=777, V=50257, K=200, dtype="f32", temperature=1.5),
        # On-policy distillation of one short answer: few rows, an odd vocabulary, 32-bit logits.
        dict(name="distill-logits-short", op="distill", N=24, V=32003, K=16, dtype="f32", kind="reverse",
             tail=True, beta=0.5, temperature=1.0),
        # A training micro-batch on logits in memory (the FSDP branch), forward KL with the tail.
        dict(name="distill-logits-train", op="distill", N=4096, V=VOCAB, K=64, dtype="bf16", kind="forward",
             tail=True, beta=0.5, temperature=1.0),
        # Supervised tokens of one short sequence over an odd vocabulary.
        dict(name="xent-logits-short", op="xent", N=61, V=50257, dtype="bf16", smoothing=0.0, z=1e-4),
        # A supervised micro-batch on logits in memory, a third of it prompt or padding.
        dict(name="xent-logits-train", op="xent", N=4096, V=VOCAB, dtype="bf16", smoothing=0.1, z=1e-4),
        # One answer's tokens through the 0.6B-sized head: the weight's bytes bound it.
        dict(name="distill-head-short", op="distill_head", N=96, H=1024, V=VOCAB, K=32, kind="jsd", tail=True,
             beta=0.5, temperature=2.0),
        # A distillation micro-batch through the 8B-sized head.
        dict(name="distill-head-train", op="distill_head", N=8192, H=4096, V=VOCAB, K=64, kind="forward",
             tail=True, beta=0.5, temperature=1.0),
        # A small supervised step through a narrow head with an odd vocabulary.
        dict(name="xent-head-short", op="xent_head", N=130, H=512, V=32003, smoothing=0.1, z=0.0),
        # A supervised micro-batch through the 0.6B-sized head, a third of it prompt or padding.
        dict(name="xent-head-train", op="xent_head", N=16384, H=1024, V=VOCAB, smoothing=0.1, z=1e-4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["topk", "distill", "distill", "xent", "distill_head", "distill_head", "xent_head"])
    V = _log_int(rng, 1000, VOCAB)
    if op in ("topk", "distill", "xent"):
        case = dict(op=op, N=_log_int(rng, 1, 4096), V=V, dtype=rng.choice(["bf16", "bf16", "f32"]))
        if case["dtype"] == "f32":
            case["N"] = max(1, case["N"] // 2)
    else:
        case = dict(op=op, N=_log_int(rng, 1, 8192), H=8 * _log_int(rng, 8, 512), V=V)
    if op == "topk":
        case.update(K=_log_int(rng, 1, 256), temperature=rng.choice([1.0, rng.uniform(0.5, 3.0)]))
    elif op in ("distill", "distill_head"):
        kind = rng.choice(["forward", "reverse", "jsd"])
        case.update(K=_log_int(rng, 1, 128), kind=kind, tail=kind != "forward" or rng.random() < 0.6,
                    beta=rng.uniform(0.1, 0.9), temperature=rng.choice([1.0, rng.uniform(0.5, 3.0)]))
    else:
        case.update(smoothing=rng.choice([0.0, rng.uniform(0.0, 0.2)]), z=rng.choice([0.0, rng.uniform(0.0, 1e-3)]))
    return case


# ---- inputs ---------------------------------------------------------------------------------------

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _likely(N, V, n, g):
    """n likely tokens a row and their logits above the rest, as a trained model's rows have."""
    ids = torch.randint(0, V, (N, n), generator=g, device="cuda")
    boost = 12.0 - 0.8 * torch.arange(n, device="cuda") + torch.randn(N, n, generator=g, device="cuda")
    return ids, boost


def _teacher(N, V, K, ids, boost, g):
    """Entries of a teacher near the student: its likely tokens and others, a tail of 1-20%, a few
    rows with fewer entries (padded with -1) and a few with none."""
    n = ids.shape[1]
    rest = torch.randint(0, V, (N, K - n), generator=g, device="cuda")
    other = 3.0 + torch.randn(N, K - n, generator=g, device="cuda")
    lg = torch.cat([boost + 0.7 * torch.randn(N, n, generator=g, device="cuda"), other], 1)
    tail = 0.01 + 0.19 * torch.rand(N, 1, generator=g, device="cuda")
    lp = torch.log_softmax(lg, 1) + torch.log1p(-tail)
    t_ids = torch.cat([ids, rest], 1)
    row = torch.arange(N, device="cuda")[:, None]
    short = (row % 16 == 5) & (torch.arange(K, device="cuda")[None] >= max(1, K // 2))
    t_ids = torch.where(short | (row % 64 == 63), -1, t_ids)
    return t_ids, lp.float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, V, op = case["N"], case["V"], case["op"]
    n = min(8, case.get("K", 8))
    ids, boost = _likely(N, V, n, g)
    st = {"case": case}
    if "H" in case:
        H = case["H"]
        w = (0.02 * torch.randn(V, H, generator=g, device="cuda")).to(torch.bfloat16)
        h = torch.randn(N, H, generator=g, device="cuda")
        h += ((boost / (H * 4e-4))[:, :, None] * w[ids].float()).sum(1)
        st["hidden"] = h.to(torch.bfloat16).requires_grad_(True)
        st["weight"] = w.requires_grad_(True)
    else:
        x = torch.randn(N, V, generator=g, device="cuda").mul_(2.0).scatter_(1, ids, boost).to(_DTYPES[case["dtype"]])
        st["logits"] = x.requires_grad_(op != "topk")
    if "kind" in case:
        st["teacher_ids"], st["teacher_log_probs"] = _teacher(N, V, case["K"], ids, boost, g)
    if op != "topk":
        # upstream gradient of a masked mean over the tokens: a third carries none
        mask = torch.rand(N, generator=g, device="cuda") >= 1.0 / 3
        mask[0] = True
        if "kind" not in case:
            st["targets"] = torch.where(mask, ids[:, 0], -100)
        st["upstream"] = mask.float() / mask.sum()
    return st


# ---- one pass -------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    if c["op"] == "topk":
        return _plain_topk(state["logits"], c["K"], c["temperature"])
    if "H" in c:
        return _plain_head(c, state)
    x = state["logits"].detach().float()
    loss, d = _plain_rows(c, state, x, slice(None))
    return loss, (d * state["upstream"][:, None]).to(state["logits"].dtype)


def _run_own(c, state):
    from invokerl_b200 import ops

    if c["op"] == "topk":
        return ops.logits_topk(state["logits"], c["K"], temperature=c["temperature"])
    if "H" in c:
        leaves = (state["hidden"], state["weight"])
    else:
        leaves = (state["logits"],)
    if "kind" in c:
        f = ops.lmhead_distill if "H" in c else ops.logits_distill
        loss = f(*leaves, state["teacher_ids"], state["teacher_log_probs"], kind=c["kind"], beta=c["beta"],
                 temperature=c["temperature"], tail=c["tail"])
    else:
        f = ops.lmhead_cross_entropy if "H" in c else ops.logits_cross_entropy
        loss = f(*leaves, state["targets"], label_smoothing=c["smoothing"], z_loss=c["z"])
    return (loss.detach(),) + torch.autograd.grad(loss, leaves, state["upstream"])


def _plain_topk(logits, k, temperature):
    z = logits.detach().float() / temperature
    m = z.amax(1, keepdim=True)
    lse = m + torch.exp(z - m).sum(1, keepdim=True, dtype=torch.float64).log().float()
    # Order by value, then by the lower index: one whole number holds both.
    bits = logits.detach().float().view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32)
    key -= torch.arange(logits.shape[1], device=logits.device)
    top = torch.topk(key, k, dim=1).values
    ids = -top & 0xFFFFFFFF
    return z.gather(1, ids) - lse, ids


def _entries(ids, lp, V):
    """Which entries count, and which rows name a token outside the vocabulary."""
    valid = (ids >= 0) & (lp > -math.inf)
    same = (ids[:, :, None] == ids[:, None, :]) & valid[:, None, :]
    repeated = torch.tril(same, -1).any(2)
    return valid & ~repeated, (valid & (ids >= V)).any(1)


def _xlogr(w, r):
    return torch.where(w > 0, w * r, 0.0)


def _plain_rows(c, state, x, rows):
    """Loss and its gradient in the logits, for an upstream gradient of 1, of rows of 32-bit logits."""
    if "kind" not in c:
        return _plain_xent(c, state["targets"][rows], x)
    V = x.shape[1]
    ids, lp = state["teacher_ids"][rows], state["teacher_log_probs"][rows]
    use, bad = _entries(ids, lp, V)
    at = torch.where(use, ids, V).clamp(max=V)  # column V: a spare one for what does not count
    z = x / c["temperature"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True, dtype=torch.float64).float()
    member = torch.zeros(x.shape[0], V + 1, dtype=torch.bool, device=x.device).scatter_(1, at, True)[:, :V]
    rest = torch.where(member, 0.0, e).sum(1, keepdim=True, dtype=torch.float64).float()
    log_pt = rest.log() - total.log()
    log_p = z.gather(1, at.clamp(max=V - 1)) - m - total.log()
    q64 = torch.where(use, lp.double().exp(), 0.0).sum(1, keepdim=True)
    if c["tail"]:
        left = 1.0 - q64
        qt = torch.where(left >= TAIL_EPS, left, 0.0).float()
        log_qt = left.clamp(min=TAIL_EPS).log().float()
    else:
        lp = (lp.double() - q64.log()).float()
    q = torch.where(use, lp.exp(), 0.0)
    p = torch.where(use, log_p.exp(), 0.0)
    pt = log_pt.exp()
    if not c["tail"]:
        loss = _xlogr(q, lp - log_p).sum(1)
        dk, scale = p - q, 1.0
    elif c["kind"] == "forward":
        loss = _xlogr(q, lp - log_p).sum(1) + _xlogr(qt, log_qt - log_pt)[:, 0]
        s = (q64 + qt).float()
        dk = s * p - q
        scale = torch.where(pt > 0, s - qt / pt, s)
    else:
        if c["kind"] == "reverse":
            ck, ct = log_p - lp, log_pt - log_qt
            loss = _xlogr(p, ck).sum(1) + _xlogr(pt, ct)[:, 0]
        else:
            b = c["beta"]
            log_m = torch.logaddexp(lp + math.log(b), log_p + math.log1p(-b))
            mt = b * qt + (1 - b) * pt
            ck, ct = (1 - b) * (log_p - log_m), (1 - b) * (log_pt - mt.log())
            loss = b * (_xlogr(q, lp - log_m).sum(1) + _xlogr(qt, log_qt - mt.log())[:, 0])
            loss = loss + _xlogr(p, ck).sum(1) + _xlogr(pt, ct)[:, 0]
        mean = (_xlogr(p, ck).sum(1, keepdim=True) + _xlogr(pt, ct))
        dk = _xlogr(p, ck - mean)
        scale = torch.where(pt > 0, ct - mean, 0.0)
    d = torch.cat([e * (scale / total), torch.zeros_like(m)], 1).scatter_(1, at, dk)[:, :V] / c["temperature"]
    empty = ~use.any(1)
    loss = torch.where(empty, 0.0, torch.where(bad, math.nan, loss))
    d = torch.where(empty[:, None], 0.0, torch.where(bad[:, None], math.nan, d))
    return loss, d


def _plain_xent(c, targets, x):
    V = x.shape[1]
    live = targets != -100
    y = torch.where(live, targets, 0)[:, None]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    rest = e.scatter(1, y, 0.0).sum(1, keepdim=True, dtype=torch.float64).float()
    lse = m + total.log().float()
    xy = x.gather(1, y)
    nll = torch.log1p(rest / torch.exp(xy - m))
    mean = (x.sum(1, keepdim=True, dtype=torch.float64) / V).float()
    loss = nll + c["smoothing"] * (xy - mean) + c["z"] * lse * lse
    a = 1.0 + 2.0 * c["z"] * lse
    p = e / total.float()
    d = a * p - c["smoothing"] / V
    py = p.gather(1, y)
    dy = (a - 1.0) * py - rest / total.float() + c["smoothing"] * (1.0 - 1.0 / V)
    d = d.scatter_(1, y, dy)
    return torch.where(live, loss[:, 0], 0.0), torch.where(live[:, None], d, 0.0)


def _plain_head(c, state, chunk=4096):
    h, w = state["hidden"].detach().float(), state["weight"].detach().float()
    dw = torch.zeros_like(w)
    loss, dh = [], []
    for s in range(0, h.shape[0], chunk):
        rows = slice(s, s + chunk)
        part, d = _plain_rows(c, state, h[rows] @ w.t(), rows)
        d *= state["upstream"][rows, None]
        loss.append(part)
        dh.append((d @ w).to(torch.bfloat16))
        dw += d.t() @ h[rows]
    return torch.cat(loss), torch.cat(dh), dw.to(torch.bfloat16)


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    N, V = case["N"], case["V"]
    if case["op"] == "topk":
        b = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": N * V * b + 12 * N * case["K"], "flops": 2 * N * V}
    side = 12 * N * case["K"] if "K" in case else 8 * N
    side += 8 * N  # loss and upstream
    live = N if "kind" in case else (2 * N + 2) // 3  # rows with a target
    if "H" in case:
        H = case["H"]
        act = (2 * N + 2) // 3  # rows with an upstream gradient
        return {"bytes": 4 * N * H + 4 * V * H + side, "flops": 2 * H * V * (live + 2 * act)}
    b = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": (live + N) * V * b + side, "flops": 6 * live * V}


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "topk":
        lps, ids = [], []
        for x in st["logits"].split(512):
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["K"]]
            ids.append(order)
            lps.append(torch.log_softmax(x.double() / case["temperature"], 1).gather(1, order))
        return torch.cat(lps), torch.cat(ids)
    head = "H" in case
    N = case["N"]
    if head:
        h, w = st["hidden"].detach().double(), st["weight"].detach().double()
        dw = torch.zeros_like(w)
    losses, grads = [], []
    for s in range(0, N, 1024):
        rows = slice(s, min(N, s + 1024))
        x = (h[rows] @ w.t() if head else st["logits"].detach()[rows].double()).requires_grad_(True)
        loss = _exact_rows(case, st, x, rows)
        d, = torch.autograd.grad(loss, x, st["upstream"][rows].double())
        losses.append(loss.detach())
        del loss, x
        if head:
            grads.append(d @ w)
            dw += d.t() @ h[rows]
        else:
            grads.append(d)
    out = (torch.cat(losses), torch.cat(grads))
    return out + (dw,) if head else out


def _exact_rows(case, st, x, rows):
    V = case["V"]
    if "kind" not in case:
        t = st["targets"][rows]
        live = t != -100
        lse = torch.logsumexp(x, 1)
        e = case["smoothing"]
        want = torch.gather(x, 1, t.clamp(min=0)[:, None])[:, 0]
        return torch.where(live, lse - (1 - e) * want - e * x.mean(1) + case["z"] * lse ** 2, 0.0)
    ids, lp = st["teacher_ids"][rows], st["teacher_log_probs"][rows].double()
    n, K = ids.shape
    use = (ids >= 0) & torch.isfinite(lp)
    for k in range(1, K):  # a repeated id counts at its first place
        use[:, k] &= ~((ids[:, :k] == ids[:, k:k + 1]) & use[:, :k]).any(1)
    live = use.any(1)
    logp = torch.log_softmax(x / case["temperature"], 1)
    taken = torch.zeros(n, V, dtype=torch.bool, device=x.device)
    r, k = use.nonzero(as_tuple=True)
    taken[r, ids[r, k]] = True
    lpk = torch.where(use, logp.gather(1, ids.clamp(min=0)), 0.0)
    q = torch.where(use, lp.exp(), 0.0)
    if not case["tail"]:
        q = q / torch.where(live, q.sum(1), 1.0)[:, None]
        lq = torch.where(use, q, 1.0).log()
        return (q * (lq - lpk)).sum(1)
    left = 1.0 - q.sum(1)
    log_pt = torch.logsumexp(logp.masked_fill(taken, -math.inf), 1)
    qt = torch.where(left >= TAIL_EPS, left, 0.0)
    lq = torch.cat([torch.where(use, lp, 0.0), left.clamp(min=TAIL_EPS).log()[:, None]], 1)
    q = torch.cat([q, qt[:, None]], 1)
    lpk = torch.cat([lpk, log_pt[:, None]], 1)
    there = torch.cat([use, torch.ones_like(use[:, :1])], 1)
    p = torch.where(there, lpk.exp(), 0.0)
    if case["kind"] == "forward":
        loss = (q * (lq - lpk)).sum(1)
    elif case["kind"] == "reverse":
        loss = (p * (lpk - lq)).sum(1)
    else:
        b = case["beta"]
        lm = torch.where(there, b * q + (1 - b) * p, 1.0).log()
        loss = (b * q * (lq - lm) + (1 - b) * p * (lpk - lm)).sum(1)
    return torch.where(live, loss, 0.0)
