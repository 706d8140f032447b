"""The row losses from their definitions in 64 bits (gradients by autograd), and the error bounds the
tests hold the kernels to."""

from __future__ import annotations

import math

import torch

TAIL_EPS = 2.0 ** -20
EPS32 = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def entry_mask(ids, lp):
    """Entries that count: id >= 0, log-prob above -inf, a repeated id at its first place."""
    use = (ids >= 0) & (lp != -math.inf)
    for k in range(1, ids.shape[1]):
        use[:, k] &= ~((ids[:, :k] == ids[:, k:k + 1]) & use[:, :k]).any(1)
    return use


def distill_rows(x, ids, lp, kind="forward", beta=0.5, temperature=1.0, tail=True):
    """Loss [n] (float64, differentiable in x) of logits x [n, V], row by row."""
    out = []
    x = x.double() if x.dtype != torch.float64 else x
    use = entry_mask(ids, lp)
    V = x.shape[1]
    for r in range(x.shape[0]):
        cols, l = ids[r][use[r]], lp[r][use[r]].double()
        if len(cols) == 0:
            out.append(x.new_zeros(()))
            continue
        if int(cols.max()) >= V:
            out.append(x[r].sum() * math.nan)
            continue
        logp = torch.log_softmax(x[r] / temperature, 0)
        q, lpk = l.exp(), logp[cols]
        if not tail:
            l = l - q.sum().log()
            q = l.exp()
        elif len(cols) < V:
            rest = torch.ones(V, dtype=torch.bool, device=x.device)
            rest[cols] = False
            left = 1.0 - q.sum()
            lpk = torch.cat([lpk, torch.logsumexp(logp[rest], 0)[None]])
            q = torch.cat([q, torch.where(left >= TAIL_EPS, left, 0.0)[None]])
            l = torch.cat([l, left.clamp(min=TAIL_EPS).log()[None]])
        # outcomes the student excludes (-inf) have no part in p log p, and no gradient
        on = lpk > -math.inf
        if kind == "forward":
            on |= q > 0
            out.append((q[on] * (l[on] - lpk[on])).sum())
        elif kind == "reverse":
            out.append((lpk[on].exp() * (lpk[on] - l[on])).sum())
        else:
            p = lpk[on].exp()
            lm = (beta * q[on] + (1 - beta) * p).log()
            first = torch.where(q[on] > 0, q[on] * (torch.where(q[on] > 0, l[on], 0.0) - lm), 0.0).sum()
            # an excluded outcome still has its teacher side: q log(q / (beta q))
            first = first + (q[~on] * -math.log(beta)).sum()
            out.append(beta * first + (1 - beta) * (p * (lpk[on] - lm)).sum())
    return torch.stack(out) if out else x.new_zeros(0)


def xent_rows(x, targets, label_smoothing=0.0, z_loss=0.0):
    x = x.double() if x.dtype != torch.float64 else x
    out = []
    for r in range(x.shape[0]):
        t = int(targets[r])
        if t == -100:
            out.append(x.new_zeros(()))
        elif not 0 <= t < x.shape[1]:
            out.append(x[r].sum() * math.nan)
        else:
            lse = torch.logsumexp(x[r], 0)
            v = lse - x[r, t] + z_loss * lse ** 2
            if label_smoothing:
                v = v + label_smoothing * (x[r, t] - x[r].mean())
            out.append(v)
    return torch.stack(out) if out else x.new_zeros(0)


def loss_and_grad(fn, x, upstream):
    """(loss, d sum(upstream loss) / dx) in float64.  A row without an upstream gradient has none, NaN or
    not (autograd would make it 0 * NaN)."""
    x = x.detach().double().requires_grad_(True)
    loss = fn(x)
    d, = torch.autograd.grad(loss, x, upstream.double())
    return loss.detach(), torch.where(upstream[:, None] == 0, 0.0, d)


def fp32_tol(V: int, K: int, span: float) -> float:
    """Relative error a row's fp32 arithmetic may gather: a thread's running sum has V / 512 terms
    plus a few merges, an exponential is off by 4 steps plus those of its argument (as large as
    `span`, the spread of the logits in use, each operation half a step), the K entries add K."""
    return EPS32 * (V / 512 + K + 48 + 4 * span)


def check_loss(got, want, tol):
    """tol: relative to 1 + the loss's own terms, which are at most of the order of its log-probs."""
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    ok = ~(inf | want.isnan())
    err = (got[ok] - want[ok]).abs()
    assert bool((err <= tol).all()), (float(err.max()), tol)


def check_grad(got, want, dtype, scale, tol, ref_err=0.0):
    """Each element within half a step of its type of the 64-bit gradient, plus `tol` times `scale`
    (what its fp32 terms are made of: |upstream| / T times the probabilities that enter it), plus what
    the 64-bit gradient itself may be off by."""
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    tiny = torch.finfo(torch.float32).smallest_normal
    err = (got - want).abs()
    lim = half_step(dtype) * (1 + 2 ** -7) * want.abs() + tol * scale.cpu() + ref_err + 2 * tiny
    bad = ok & ~(err <= lim)
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(),
                                 lim[bad][:4].tolist())


def grad_scale(x, ids, lp, upstream, temperature=1.0):
    """Per element, |upstream| / T times the probabilities whose fp32 errors reach it: p and q at an
    entry (times its log-ratio, at most the spread of the log-probs), the tail's share of column v
    (softmax over the tail) elsewhere."""
    x = x.detach().double()
    n, V = x.shape
    logp = torch.log_softmax(x / temperature, 1)
    use = entry_mask(ids, lp) & (ids < V)
    taken = torch.zeros(n, V, dtype=torch.bool, device=x.device)
    r, k = use.nonzero(as_tuple=True)
    taken[r, ids[r, k]] = True
    share = torch.softmax((x / temperature).masked_fill(taken, -math.inf), 1).nan_to_num(0.0)
    q = torch.zeros(n, V, dtype=torch.float64, device=x.device)
    q[r, ids[r, k]] = lp[r, k].double().exp()
    span = 1 + (-logp.masked_fill(~taken, 0.0)).clamp(max=200).amax(1, keepdim=True) + \
        (-lp.double().masked_fill(~use, 0.0)).clamp(max=200).amax(1, keepdim=True)
    return upstream.double().abs()[:, None] / temperature * span * torch.where(taken, logp.exp() + q, share)
