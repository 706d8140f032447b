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
    # Taken off before anything else: a row of -1e30 would swallow the logarithms of its sums.
    top = x.detach().amax(1)
    top = torch.where(top.isfinite(), top, 0.0)
    for r in range(x.shape[0]):
        cols, l = ids[r][use[r]], lp[r][use[r]].double()
        if len(cols) == 0:
            out.append(x.new_zeros(()))
            continue
        if int(cols.max()) >= V:
            out.append(x[r].sum() * math.nan)
            continue
        logp = torch.log_softmax((x[r] - top[r]) / temperature, 0)
        q, lpk = l.exp(), logp[cols]
        if not tail:
            l = l - q.sum().log()
            q = l.exp()
        elif len(cols) < V:
            rest = torch.ones(V, dtype=torch.bool, device=x.device)
            rest[cols] = False
            left = 1.0 - q.sum()
            # from the tail's own maximum: beside a mask of -1e30 even 64 bits lose the logarithm of the sum
            z = (x[r] - top[r]) / temperature
            mx = z[rest].detach().max()
            mx = mx if mx > -math.inf else torch.zeros_like(mx)
            log_pt = torch.logsumexp(z[rest] - mx, 0) + (mx - torch.logsumexp(z, 0))
            lpk = torch.cat([lpk, log_pt[None]])
            q = torch.cat([q, torch.where(left >= TAIL_EPS, left, 0.0)[None]])
            l = torch.cat([l, left.clamp(min=TAIL_EPS).log()[None]])
        # outcomes the student excludes (p is 0, in 64 bits) have no part in p log p, and no gradient
        on = lpk.exp() > 0
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
            top = x[r].detach().max()
            top = top if bool(top.isfinite()) else torch.zeros_like(top)
            rel = torch.logsumexp(x[r] - top, 0)
            v = rel - (x[r, t] - top) + z_loss * (rel + top) ** 2
            if label_smoothing:
                v = v + label_smoothing * (x[r, t] - x[r].mean())
            out.append(v)
    return torch.stack(out) if out else x.new_zeros(0)


def loss_size(x, ids, lp, kind="forward", beta=0.5, temperature=1.0, tail=True):
    """Per row, the sum of the magnitudes its loss is formed from: each outcome's weight times the logarithms
    beside it.  An entry at a masked column (log p = -1e9, say) makes a forward loss of that size, whose
    fp32 terms are off by half steps of that size; in the other losses such an outcome weighs nothing."""
    V = x.shape[1]
    logp = torch.log_softmax(x.detach().double() / temperature, 1)
    use = entry_mask(ids, lp) & (ids < V)
    out = torch.ones(x.shape[0], dtype=torch.float64)
    for r in range(x.shape[0]):
        cols, l = ids[r][use[r]], lp[r][use[r]].double()
        if len(cols) == 0 or not bool(logp[r].isfinite().any()):
            continue
        lpk, q = logp[r, cols], l.exp()
        rest = torch.ones(V, dtype=torch.bool)
        rest[cols] = False
        if tail and bool(rest.any()):
            left = max(float(1 - q.sum()), TAIL_EPS)
            lpk = torch.cat([lpk, torch.logsumexp(logp[r, rest], 0)[None]])
            l = torch.cat([l, torch.tensor([math.log(left)], dtype=torch.float64)])
            q = l.exp()
        p = lpk.exp()
        lpa = lpk.abs().nan_to_num(posinf=0.0)
        if kind == "forward":
            out[r] += float((q * (l.abs() + lpa)).sum())
        elif kind == "reverse":
            out[r] += float(torch.where(p > 0, p * (l.abs() + lpa), 0.0).sum())
        else:
            lm = (beta * q + (1 - beta) * p).log().abs()
            out[r] += float((q * (l.abs() + lm) + torch.where(p > 0, p * (lpa + lm), 0.0)).sum())
    return out


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
    """tol: an absolute bound, for all rows or for each."""
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    ok = ~(inf | want.isnan())
    err = (got[ok] - want[ok]).abs()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)[ok]
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


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
