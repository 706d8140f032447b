"""Row losses on the GPU where their inputs are not what a healthy step gives them."""

import math
from types import SimpleNamespace

import pytest
import torch

from invokerl_b200 import ops
from row_loss_math import (EPS32, check_grad, check_loss, distill_rows, fp32_tol, grad_scale, loss_and_grad,
                           loss_size, xent_rows)
from test_row_losses_gpu import (DEV, KINDS, _tiny_policy, check_distill, check_head, make_head, make_rows, run_distill,
                                 run_head, span_of)

pytestmark = pytest.mark.gpu


# ---- teachers -------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("n", [4, 310])  # one launch, and three
def test_nan_log_prob_of_an_entry_makes_its_row_nan(n, kind, tail):
    """Where the entry counts: not behind an id below 0, and not as a repeat of a column that is there already."""
    x, ids, lp, up = make_rows(n, 700, 6, torch.float32, 41)
    up = up.abs() + 0.1
    lp[1, 2] = math.nan
    ids[2, 3], lp[2, 3] = -1, math.nan
    ids[0, 4], lp[0, 4] = ids[0, 1], math.nan
    lp[3] = math.nan
    loss, d = check_distill(x, ids, lp, up, kind, tail)
    nan = torch.arange(n) % 2 == 1
    nan[4:] = False
    assert torch.equal(loss.isnan().cpu(), nan) and torch.equal(d.isnan().all(1).cpu(), nan)


@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("n", [30, 1100])
def test_nan_log_prob_through_the_head(n, kind, tail):
    h, w, ids, lp, up = make_head(n, 64, 1000, 6, 42)
    up = up.abs() + 0.1
    want = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind=kind, tail=tail)
    lp[3, 2] = math.nan
    loss, dh, dw = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind=kind, tail=tail)
    ok = torch.arange(n) != 3
    assert bool(loss[3].isnan()) and bool(dh[3].isnan().all()) and bool(dw.isnan().all())
    assert torch.equal(loss[ok], want[0][ok]) and torch.equal(dh[ok], want[1][ok])
    up[3] = 0.0
    _, dh, dw = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind=kind, tail=tail)
    assert bool(dh.isfinite().all()) and bool(dw.isfinite().all())


@pytest.mark.parametrize("kind,tail", KINDS)
def test_nan_in_the_teachers_logits_reaches_the_students_loss(kind, tail):
    x, _, _, _ = make_rows(5, 3000, 4, torch.bfloat16, 43)
    t = x.clone()
    t[2, 1717] = math.nan
    lp, ids = ops.logits_topk(t.to(DEV), 8)
    loss, d = run_distill(x, ids, lp, torch.ones(5), kind=kind, tail=tail)
    assert loss.isnan().tolist() == [False, False, True, False, False]
    assert d.isnan().all(1).tolist() == [False, False, True, False, False]


@pytest.mark.parametrize("n", [4, 310])
def test_renormalised_teacher_of_any_mass(n):
    """Without the tail only the entries' ratios count, also where their mass is 0 in 64 bits; entries masked
    with a very low value beside others weigh nothing."""
    x, ids, lp, up = make_rows(n, 700, 6, torch.float32, 44)
    lp[0, 3] = -1e30
    lp[1] -= 2000
    lp[2] = -1e30
    lp[3] = torch.finfo(torch.float32).min
    loss, d = run_distill(x, ids, lp, up, kind="forward", tail=False)
    ratios = torch.log_softmax(lp.double(), 1)
    want, dw = loss_and_grad(lambda y: distill_rows(y, ids, ratios, tail=False), x, up)
    tol = fp32_tol(700, 6, span_of(x, ids, ratios, 1.0))
    check_loss(loss, want, tol * loss_size(x, ids, ratios, tail=False))
    check_grad(d, dw, x.dtype, grad_scale(x, ids, ratios, up), tol)


# ---- masks ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V", [(4, 9001), (310, 9001), (3, 17), (330, 9)])
def test_label_smoothing_beside_the_lowest_value(n, V, dtype):
    """The mean of a row half masked with the type's lowest value is in range, its sum is not."""
    x, ids, _, up = make_rows(n, V, 1, dtype, 45)
    t = ids[:, 0]
    g = torch.Generator().manual_seed(n)
    keep = (torch.rand(n, V, generator=g) < 0.5).scatter_(1, ids, True)
    keep[:, V - 3:] = False
    keep.scatter_(1, ids, True)
    x = torch.where(keep, x, torch.finfo(dtype).min)
    xd = x.to(DEV).requires_grad_(True)
    loss = ops.logits_cross_entropy(xd, t.to(DEV), 0.1)
    d, = torch.autograd.grad(loss, xd, up.to(DEV))
    want, dw = loss_and_grad(lambda y: xent_rows(y, t, 0.1), x, up)
    # nearly all of it is 0.1 of the mean, a sum of values of one sign
    check_loss(loss.detach(), want, fp32_tol(V, 1, 1.0) * want.abs())
    logp = torch.log_softmax(x.double(), 1)
    span = float(logp[keep].abs().max())
    p = logp.exp()
    scale = p.scatter(1, ids, 1 - p.gather(1, ids) + 0.1) + 0.1 / V
    # the 64-bit p_y - 1 is rounded at the size of 1 and of the logits it comes from
    ref_err = up.double().abs()[:, None] * 2.0 ** -52 * (1 + float(x[keep].double().abs().max()))
    check_grad(d, dw, dtype, up.double().abs()[:, None] * scale, fp32_tol(V, 1, span), ref_err)


@pytest.mark.parametrize("loss", ["distill", "xent"])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("cache", ["auto", "off"])
@pytest.mark.parametrize("n", [40, 300, 1100])
def test_padding_rows_may_hold_nan(n, cache, captured, loss):
    """Rows without entries (or a target) or without an upstream gradient reach no gradient, whatever their hidden
    state holds: attention leaves NaN in padding."""
    h, w, ids, lp, up = make_head(n, 64, 1000, 6, 46)
    up = up.abs() + 0.1
    ids[3] = -1
    up[5] = 0.0
    t = torch.where(torch.arange(n) == 3, -100, ids[:, 0])
    clean = h.clone()
    clean[3] = clean[5] = 0.0
    h[3] = math.nan
    h[5] = math.inf

    def step(h, w, up, ids, lp, t):
        a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out = ops.lmhead_distill(a, b, ids, lp, "jsd") if loss == "distill" else ops.lmhead_cross_entropy(a, b, t, 0.1)
        return (out.detach(), *torch.autograd.grad(out, (a, b), up))

    prev = ops.set_logit_cache(cache)
    try:
        rest = [a.to(DEV) for a in (w, up, ids, lp, t)]
        want, got = step(clean.to(DEV), *rest), None
        bad = h.to(DEV)
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(bad, *rest)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step(bad, *rest)
            graph.replay()
        else:
            got = step(bad, *rest)
    finally:
        ops.set_logit_cache(prev["mode"])
    ok = torch.arange(n, device=DEV) != 5
    assert torch.equal(got[0][ok], want[0][ok])
    for g, ref in zip(got[1:], want[1:]):
        # a capture recomputes what an eager step may take from the cache: the roundings of dS
        assert bool(g.isfinite().all())
        assert float((g.float() - ref.float()).norm()) <= 2 ** -6 * float(ref.float().norm())
        assert float(got[1][3].float().abs().max()) == float(got[1][5].float().abs().max()) == 0.0


# ---- memory ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("n", [60, 300])
def test_a_small_cache_is_only_taken_where_memory_is_left(n, monkeypatch):
    """Neither a reserve that leaves nothing nor an allocation that fails stops a call: it recomputes the logits."""
    h, w, ids, lp, up = make_head(n, 64, 1000, 6, 47)
    prev = ops.set_logit_cache("off")
    try:
        want = run_head(ops.lmhead_distill, h, w, up, ids, lp)
        made = []

        class Failing(ops.LogitCache):
            def __init__(self, *a):
                made.append(a)
                raise torch.OutOfMemoryError("no memory left")

        monkeypatch.setattr(ops, "LogitCache", Failing)
        for reserve, tried in ((1 << 50, 0), (0, 1)):
            ops.set_logit_cache("auto", reserve)
            got = run_head(ops.lmhead_distill, h, w, up, ids, lp)
            assert len(made) == tried
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        ops.set_logit_cache(prev["mode"], prev["reserve_bytes"], prev["fraction"])


# ---- policies -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_policies_with_logits_in_memory_keep_their_bits(dtype):
    """Models that yield fp32 (or fp16) logits: their losses and top log-probs are those of the logits themselves."""
    from invokerl_b200.policy import PolicyModel

    policy = PolicyModel.from_model(_tiny_policy(2).to(dtype), fsdp_wrapped=True)
    g = torch.Generator().manual_seed(4)
    tok = torch.randint(0, 1000, (2, 20), generator=g).to(DEV)
    am = torch.ones_like(tok)
    lp, ids = policy.topk_log_probs(tok, am, 9, temperature=1.3)
    x = policy.model(input_ids=tok, attention_mask=am).logits.detach()[:, :-1].reshape(-1, 1000)
    assert x.dtype == dtype
    wl, wi = ops.logits_topk(x.float(), 9, 1.3)
    assert torch.equal(ids[:, 1:].reshape(-1, 9), wi) and torch.equal(lp[:, 1:].reshape(-1, 9), wl)
    other = torch.log_softmax(torch.randn(2, 20, 9, generator=g), -1).to(DEV) - 0.1
    kl = policy.distill_loss(tok, am, ids, other, kind="jsd")
    assert torch.equal(kl[:, 1:].reshape(-1), ops.logits_distill(x.float(), wi, other[:, 1:].reshape(-1, 9), "jsd"))
    ce = policy.cross_entropy_loss(tok, am, 0.1, 1e-4)
    assert torch.equal(ce[:, 1:].reshape(-1), ops.logits_cross_entropy(x.float(), tok[:, 1:].reshape(-1), 0.1, 1e-4))
    (kl.sum() + ce.sum()).backward()
    assert all(bool(p.grad.isfinite().all()) for p in policy.model.parameters())


@pytest.mark.parametrize("fsdp", [False, True])
@pytest.mark.parametrize("B,T", [(0, 7), (2, 1), (1, 2)])
def test_policies_on_the_smallest_batches(B, T, fsdp):
    """No sequences, and sequences without a second token: nothing to learn from, and no error."""
    from invokerl_b200.policy import PolicyModel

    w = torch.randn(50, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)

    class Body:
        lm_head = SimpleNamespace(weight=w)

        def model(self, input_ids, attention_mask):
            return SimpleNamespace(last_hidden_state=torch.ones(*input_ids.shape, 64, device=DEV, dtype=w.dtype))

        def __call__(self, input_ids, attention_mask):
            return SimpleNamespace(logits=self.model(input_ids, attention_mask).last_hidden_state @ w.t())

    policy = PolicyModel.from_model(Body(), fsdp_wrapped=fsdp)
    tok = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    am = torch.ones_like(tok)
    lp, ids = policy.topk_log_probs(tok, am, 3)
    assert lp.shape == ids.shape == (B, T, 3) and bool((ids[:, :1] == -1).all())
    ce = policy.cross_entropy_loss(tok, am)
    assert bool((ce[:, 1:] > 0).all())
    for loss in (policy.distill_loss(tok, am, ids, lp), ce):
        assert loss.shape == (B, T) and not bool(loss[:, :1].any()) and bool(loss.isfinite().all())
        dw, = torch.autograd.grad(loss.sum(), w)
        assert bool(dw.isfinite().all())


# ---- many column tiles ----------------------------------------------------------------------------


@pytest.mark.parametrize("loss", ["reverse", "xent"])
@pytest.mark.parametrize("n,H,V", [(1100, 64, 40000), (1100, 1024, 40001), (2300, 1024, 32000), (4500, 128, 9001)])
def test_gathered_rows_over_many_column_tiles(n, H, V, loss):
    """Some tens of column tiles, dealt out on the device for the rows that count: every column is in every row's
    sums once.  A logit errs by at most 2 H half-steps of fp32 (the accumulators cut) of its terms' magnitudes, E;
    a loss by the sum of its derivatives times E beside its own arithmetic; the gradients' whole as check_head."""
    h, w, ids, lp, up = make_head(n, H, V, 20 if loss == "reverse" else 1, n + H)
    off = torch.arange(n) % 3 == 1
    t = torch.where(off, -100, ids[:, 0])
    ids[off] = -1
    if loss == "reverse":
        got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="reverse")
        rows = lambda y: distill_rows(y, ids, lp, "reverse")  # noqa: E731
    else:
        got = run_head(ops.lmhead_cross_entropy, h, w, up, t, label_smoothing=0.1)
        rows = lambda y: xent_rows(y, t, 0.1)  # noqa: E731
    h, w, ids, lp, up, t = (a.to(DEV) for a in (h, w, ids, lp, up, t))
    x = h.double() @ w.double().t()
    err = 2 * H * EPS32 * (h.double().abs() @ w.double().abs().t())
    want, ds = loss_and_grad(rows, x, torch.ones(n, device=DEV))
    span = float((x.amax(1) - x.amin(1)).max())
    tol = fp32_tol(V, ids.shape[1], span) * (1 + span) + 1.01 * (ds.abs() * err).sum(1)
    check_loss(got[0], want, tol.cpu())
    ds *= up.double()[:, None]
    for g, ref in ((got[1], ds @ w.double()), (got[2], ds.t() @ h.double())):
        assert float((g.double() - ref).norm() / ref.norm()) <= 2 ** -7 + 8 * float(err.max())


@pytest.mark.parametrize("loss", ["jsd", "xent"])
@pytest.mark.parametrize("slots", [0, 1, 250, 599, 600])
def test_a_cache_of_some_rows_of_a_small_batch(slots, loss, monkeypatch):
    """Up to 1024 rows a cache is used when it holds all of them, and otherwise left alone: both directions of the C
    entries agree on which."""
    n, H, V = 600, 64, 1000
    h, w, ids, lp, up = make_head(n, H, V, 9, 48)
    ids[1::3] = -1
    made = []

    def some(*a):
        made.append(ops.LogitCache(n, V, slots, torch.device(DEV, 0)) if slots else None)
        if slots:
            made[-1].slot.fill_(7)
            made[-1].q.fill_(3.0)
        return made[-1]

    monkeypatch.setattr(ops, "_row_cache", some)
    if loss == "jsd":
        got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="jsd", temperature=1.3)
        rows, scale = lambda y: distill_rows(y, ids, lp, "jsd", 0.5, 1.3), lambda x: grad_scale(x, ids, lp, up, 1.3)
        span = span_of(h.double() @ w.double().t(), ids, lp, 1.3)
    else:
        t = torch.where(ids[:, 0] < 0, -100, ids[:, 0])
        got = run_head(ops.lmhead_cross_entropy, h, w, up, t, label_smoothing=0.1)
        rows = lambda y: xent_rows(y, t, 0.1)  # noqa: E731
        x = h.double() @ w.double().t()
        span = float((x.amax(1) - x.amin(1)).max())

        def scale(x):
            p = torch.softmax(x, 1)
            return up.double().abs()[:, None] * (p + 0.1 / V).scatter(1, t.clamp(min=0)[:, None], 1.0)

    check_head(h, w, up, got, rows, scale, 9, span, cached=True)
    if slots:
        assert bool((made[0].slot == 7).all()) and bool((made[0].q == 3.0).all()) == (slots < n)


# ---- the gradients' precision and range -------------------------------------------------------------


def own_rounding(ref):
    """Size of what rounding the 64-bit value to bf16 alone leaves."""
    return float((ref.bfloat16().double() - ref).norm())


@pytest.mark.parametrize("cache", ["auto", "off"])
@pytest.mark.parametrize("loss", ["reverse", "jsd", "xent"])
@pytest.mark.parametrize("n,H,V", [(1500, 72, 5000), (1100, 1024, 2056), (3000, 128, 1003)])
def test_gradients_of_gathered_rows_err_by_their_own_rounding(n, H, V, loss, cache, monkeypatch):
    """dS is rounded to fp16 (twice, with numerators from a cache), whose half step is an eighth of bf16's: beside
    the final rounding, sqrt(1 + 2 / 64) = 1.016 times its error; the logits' own errors are far below.  With equal
    upstream gradients, which round alike, a bf16 dS would leave 1.4 to 1.7 times."""
    monkeypatch.setattr(ops, "_ROW_CACHE_MIN_HIDDEN", 1)
    h, w, ids, lp, _ = make_head(n, H, V, 12, n + V)
    up = torch.where(torch.arange(n) % 3 == 1, 0.0, 1.0 / n)
    prev = ops.set_logit_cache(cache)
    try:
        if loss == "xent":
            got = run_head(ops.lmhead_cross_entropy, h, w, up, ids[:, 0].contiguous(), label_smoothing=0.05)
        else:
            got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind=loss)
    finally:
        ops.set_logit_cache(prev["mode"])
    h, w, ids, lp, up = (a.to(DEV) for a in (h, w, ids, lp, up))
    rows = (lambda y: xent_rows(y, ids[:, 0], 0.05)) if loss == "xent" else (lambda y: distill_rows(y, ids, lp, loss))
    _, ds = loss_and_grad(rows, h.double() @ w.double().t(), up)
    for g, ref in ((got[1], ds @ w.double()), (got[2], ds.t() @ h.double())):
        assert float((g.double() - ref).norm()) <= 1.05 * own_rounding(ref)


@pytest.mark.parametrize("cache", ["auto", "off"])
@pytest.mark.parametrize("ws,us", [(-40, 0), (30, 0), (0, -60), (0, 40), (-20, -50), (25, 30)])
def test_powers_of_two_pass_through_the_gradients(ws, us, cache, monkeypatch):
    """2^ws W and 2^-ws h have the same logits: dW and dH are 2^-ws and 2^ws times as large, bit for bit, and 2^us
    times with an upstream gradient that is."""
    monkeypatch.setattr(ops, "_ROW_CACHE_MIN_HIDDEN", 1)
    n = 1100
    h, w, ids, lp, up = make_head(n, 64, 1000, 9, 51)
    prev = ops.set_logit_cache(cache)
    try:
        want = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="jsd")
        got = run_head(ops.lmhead_distill, h * 2.0 ** -ws, w * 2.0 ** ws, up * 2.0 ** us, ids, lp, kind="jsd")
    finally:
        ops.set_logit_cache(prev["mode"])
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[1].double(), want[1].double() * 2.0 ** (us + ws))
    assert torch.equal(got[2].double(), want[2].double() * 2.0 ** (us - ws))


def test_rows_of_very_different_gradients():
    """Each row's dH keeps its bits beside rows with a gradient 2^40 times as large, and infinite ones; dW is the
    large rows'."""
    n = 1100
    h, w, ids, lp, up = make_head(n, 64, 1000, 9, 52)
    up = up.abs() + 0.5
    want = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="reverse")
    small = torch.arange(n) % 2 == 1
    few = torch.where(small, 2.0 ** -40, 1.0)
    got = run_head(ops.lmhead_distill, h, w, up * few, ids, lp, kind="reverse")
    assert torch.equal(got[1].double(), want[1].double() * few.to(DEV)[:, None].double())
    large = run_head(ops.lmhead_distill, h, w, torch.where(small, 0.0, up), ids, lp, kind="reverse")
    # both within half a bf16 step (2^-8) of fp32 sums of the same large terms in another order
    assert float((got[2].double() - large[2].double()).norm()) <= 2.0 ** -7 * 1.01 * float(large[2].double().norm())
    up[6] = math.inf
    _, dh, dw = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="reverse")
    ok = torch.arange(n) != 6
    assert torch.equal(dh[ok], want[1][ok]) and not bool(dh[6].isfinite().any()) and not bool(dw.isfinite().all())
    zero = run_head(ops.lmhead_distill, h, torch.zeros_like(w), up.clamp(max=1.0), ids, lp, kind="reverse")
    assert not bool(zero[1].any()) and bool(zero[2].isfinite().all())


def likely_head(n, H, V, seed):
    """Rows with eight likely tokens, as a trained model's: logits from 12 down over others of deviation 1.3.  Each
    lies in another eighth of the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    w = (0.02 * torch.randn(V, H, generator=g)).to(torch.bfloat16)
    ids = torch.randint(0, V // 8, (n, 8), generator=g) + V // 8 * torch.arange(8)
    boost = 12.0 - 0.8 * torch.arange(8) + torch.randn(n, 8, generator=g)
    h = torch.randn(n, H, generator=g) + ((boost / (H * 4e-4))[:, :, None] * w[ids].float()).sum(1)
    return h.to(torch.bfloat16), w, ids


@pytest.mark.parametrize("loss", ["xent", "reverse"])
@pytest.mark.parametrize("n,H,V", [(4, 4096, 6000), (14, 1992, 9001), (40, 1024, 20000), (1100, 4096, 20000)])
def test_losses_through_a_wide_head(n, H, V, loss):
    """The accumulators cut 1e-9 H of a logit; the likely tokens' logits are summed again in fp32.  Those err by 2^-24
    of a logit of 12, about 2e-7 of a loss of 4; the unlikely tokens, a fifth of the mass with logits of about 2, by
    4e-6 of that, 4e-7 of the loss.  With the likely ones from the accumulators it was 2e-6 to 5e-6."""
    h, w, ids = likely_head(n, H, V, n + H)
    if loss == "xent":
        got = ops.lmhead_cross_entropy(h.to(DEV), w.to(DEV), ids[:, 0].contiguous().to(DEV))
        rows = lambda y: xent_rows(y, ids[:, 0])  # noqa: E731
    else:
        few = ids[:, :2].contiguous()
        lp = torch.log_softmax(torch.randn(n, 2, generator=torch.Generator().manual_seed(n)), 1) - 0.5
        got = ops.lmhead_distill(h.to(DEV), w.to(DEV), few.to(DEV), lp.to(DEV), kind="reverse")
        rows = lambda y: distill_rows(y, few, lp, "reverse")  # noqa: E731
    want = rows(h.double() @ w.double().t())
    assert float((got.double().cpu() - want).norm()) <= 1e-6 * float(want.norm())
