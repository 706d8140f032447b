"""Row losses and top-k on the GPU against their 64-bit definitions: sizes, masks, layouts, streams,
captures, and a teacher and a student run together."""

import math

import pytest
import torch

from invokerl_b200 import _native as N
from invokerl_b200 import ops
from row_loss_math import (EPS32, check_grad, check_loss, distill_rows, fp32_tol, grad_scale, half_step,
                           loss_and_grad, loss_size, xent_rows)

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = [("forward", True), ("forward", False), ("reverse", True), ("jsd", True)]
DTYPES = [torch.bfloat16, torch.float32]


# ---- top-k ----------------------------------------------------------------------------------------


def check_topk(x, k, temperature=1.0):
    """x: logits on the GPU.  Ids exact, log-probs within the fp32 bound of the row's spread."""
    lp, ids = ops.logits_topk(x, k, temperature)
    assert lp.shape == ids.shape == (*x.shape[:-1], k)
    z = x.detach().double().cpu().reshape(-1, x.shape[-1])
    lp, ids = lp.cpu().reshape(-1, k), ids.cpu().reshape(-1, k)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids, order)
    want = torch.log_softmax(z / temperature, 1).gather(1, order)
    fin = want.isfinite()
    assert torch.equal(lp[~fin].double(), want[~fin])
    assert bool(((lp.double() - want)[fin].abs() <= fp32_tol(x.shape[-1], 1, want[fin].abs())).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (1, 5, 5), (3, 17, 1), (7, 1001, 256), (2, 256, 256), (5, 50257, 33),
                                   (2, 151936, 20), (320, 4097, 64), (1, 151936, 256), (700, 151, 16), (1000, 5, 3),
                                   (445, 9001, 128), (900, 40000, 30), (445, 200003, 64), (40, 200003, 128)])
def test_topk_sizes(n, V, k, dtype):
    g = torch.Generator().manual_seed(n + V + k)
    check_topk((2 * torch.randn(n, V, generator=g)).to(dtype).to(DEV), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["equal", "two", "rising", "falling", "masked", "lowest", "zeros"])
@pytest.mark.parametrize("n,V,k", [(3, 40001, 100), (400, 20000, 256), (450, 20000, 128), (446, 210000, 40)])
def test_topk_orders_and_ties(kind, n, V, k, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(n, V, generator=g)
    if kind == "equal":
        x = torch.full((n, V), 1.5)
    elif kind == "two":
        x = (x > 2.0).float()
    elif kind == "rising":  # every column beats those before it (in ties, for bf16)
        x = torch.arange(V).float().expand(n, V) / 512
    elif kind == "falling":
        x = -torch.arange(V).float().expand(n, V) / 512
    elif kind == "masked":  # fewer than k columns are left
        x[:, k // 2:] = -math.inf
        x = x[:, torch.randperm(V, generator=g)]
    elif kind == "lowest":
        x[:, k // 2:] = torch.finfo(dtype).min
    else:  # -0 and +0 are one value
        x = torch.where(x > 0, 0.0, -0.0)
    check_topk(x.to(dtype).to(DEV), k)


def test_topk_layouts_temperature_and_empty():
    g = torch.Generator().manual_seed(5)
    base = torch.randn(6, 3, 1100, generator=g).to(DEV)
    check_topk(base[:, :, 7:1008], 40, 0.5)  # rows neither dense nor aligned
    check_topk(base[0, 0], 3, 3.0)           # one row without a row dimension
    check_topk(base.to(torch.bfloat16)[:, 1, 1:], 17)
    check_topk(base.transpose(0, 2), 2)      # strided columns
    check_topk(base[:1, :1].expand(4, 2, 1100), 9)
    many = torch.randn(500, 1015, generator=g).to(DEV)
    for dtype in DTYPES:
        check_topk(many.to(dtype)[:, 5:1011], 100)
        check_topk(many.to(dtype)[1:451, 3:12], 9)
    check_topk(many[:1].expand(450, 1015), 9)
    lp, ids = ops.logits_topk(torch.empty(0, 50, device=DEV), 4)
    assert lp.shape == ids.shape == (0, 4)


@pytest.mark.parametrize("n", [4, 450])
def test_topk_nan_and_infinity(n):
    x = torch.randn(n, 30000, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :8]
    x[0, 12345] = math.nan
    x[1, 777] = math.inf
    x[1, 29999] = math.inf
    lp, ids = ops.logits_topk(x, 8)
    assert ids[0].tolist() == [12345] + want[0, :7].tolist() and bool(lp[0].isnan().all())
    assert ids[1].tolist() == [777, 29999] + want[1, :6].tolist() and bool(lp[1].isnan().any())
    assert torch.equal(ids[2:], want[2:]) and bool(lp[2:].isfinite().all())


def test_topk_refusals():
    x = torch.zeros(2, 30, device=DEV)
    for k in (0, 31, 257):
        with pytest.raises(ValueError, match="k ="):
            ops.logits_topk(x, k)
    with pytest.raises(TypeError, match="logits"):
        ops.logits_topk(x.half(), 3)


# ---- losses on logits -----------------------------------------------------------------------------


def make_rows(n, V, K, dtype, seed, spread=2.0, boost=8.0):
    """Logits with a few likely columns a row, and a teacher around them with distinct entries."""
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(n, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] if V >= K else torch.randint(0, V, (K,), generator=g)
                       for _ in range(n)])
    top = min(4, K)
    x.scatter_(1, ids[:, :top], boost + torch.randn(n, top, generator=g))
    lp = torch.log_softmax(2 * torch.randn(n, K, generator=g) + torch.arange(K, 0, -1) / K, 1)
    lp = lp + torch.log1p(-(0.02 + 0.3 * torch.rand(n, 1, generator=g)))
    up = torch.randn(n, generator=g)
    return x.to(dtype), ids, lp.float(), up


def span_of(x, ids, lp, temperature):
    z = torch.log_softmax(x.double() / temperature, 1)
    pick = z.gather(1, ids.clamp(0, x.shape[1] - 1))
    both = torch.cat([pick.flatten(), lp.double().flatten()])
    return float(both[both.isfinite()].abs().max().clamp(max=200)) if both.isfinite().any() else 0.0


def run_distill(x, ids, lp, up, **kw):
    xd = x.detach().to(DEV).requires_grad_(True)
    loss = ops.logits_distill(xd, ids.to(DEV), lp.to(DEV), **kw)
    d, = torch.autograd.grad(loss, xd, up.to(DEV))
    assert loss.dtype == torch.float32 and d.dtype == x.dtype and d.shape == x.shape
    return loss.detach(), d


def check_distill(x, ids, lp, up, kind="forward", tail=True, temperature=1.0, beta=0.5):
    kw = dict(kind=kind, tail=tail, temperature=temperature, beta=beta)
    loss, d = run_distill(x, ids, lp, up, **kw)
    want, dw = loss_and_grad(lambda y: distill_rows(y, ids, lp, kind, beta, temperature, tail), x, up)
    span = span_of(x, ids, lp, temperature)
    tol = fp32_tol(x.shape[1], ids.shape[1], span)
    check_loss(loss, want, tol * loss_size(x, ids, lp, kind, beta, temperature, tail))
    check_grad(d, dw, x.dtype, grad_scale(x, ids, lp, up, temperature), tol)
    return loss, d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (2, 7, 3), (3, 1001, 16), (5, 1000, 256), (2, 50257, 64),
                                   (300, 333, 5), (1, 151936, 100), (100, 20011, 40), (330, 20011, 40)])
def test_distill_sizes(n, V, K, kind, tail, dtype):
    x, ids, lp, up = make_rows(n, V, K, dtype, n + V + K)
    check_distill(x, ids, lp, up, kind, tail)


@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("temperature,beta", [(0.5, 0.1), (2.5, 0.9)])
def test_distill_temperature_and_beta(kind, tail, temperature, beta):
    x, ids, lp, up = make_rows(6, 5000, 33, torch.float32, 3)
    check_distill(x, ids, lp, up, kind, tail, temperature, beta)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,tail", KINDS)
def test_distill_entry_rules(kind, tail, dtype):
    """Repeated ids, padding, log-probs of -inf, rows without entries, entries that are the whole
    vocabulary, ids past it, in one batch."""
    x, ids, lp, up = make_rows(8, 12, 12, dtype, 4)
    ids[0, 5] = ids[0, 1]
    ids[0, 9] = ids[0, 1]
    ids[1, 4:] = -1
    ids[2] = -1
    lp[3] = -math.inf
    lp[4, 2:7] = -math.inf
    ids[5, 3] = 12
    ids[6, 3] = 2 ** 40
    up[6] = 0.0
    lp[7] = torch.log_softmax(lp[7], 0)  # row 7: all columns, all mass
    loss, d = check_distill(x, ids, lp, up, kind, tail)
    assert float(loss[2]) == 0.0 and float(loss[3]) == 0.0
    assert float(d[2].float().abs().max()) == 0.0 and float(d[6].float().abs().max()) == 0.0
    assert bool(loss[5].isnan()) and bool(loss[6].isnan()) and bool(d[5].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["reverse", "jsd", "forward"])
@pytest.mark.parametrize("hole", ["inf", "lowest", -1e4, -1e9, -1e30])
def test_distill_masked_columns(kind, hole, dtype):
    """Columns masked in the student (-inf, or the type's lowest value), whole vectors of them, a row
    that keeps its entries only."""
    x, ids, lp, up = make_rows(4, 3001, 8, dtype, 6)
    low = {"inf": -math.inf, "lowest": torch.finfo(dtype).min}.get(hole, hole)
    keep = torch.zeros(4, 3001, dtype=torch.bool).scatter_(1, ids, True)
    x[0, 64:2500] = torch.where(keep[0, 64:2500], x[0, 64:2500], low)
    x[1] = torch.where(keep[1], x[1], low)
    x[1, 3000 if not keep[1, 3000] else 2999] = 1.0
    x[2, ::2] = torch.where(keep[2, ::2], x[2, ::2], low)
    if kind == "reverse":  # p log p of a masked entry is 0
        x[3, ids[3, 5]] = low
    check_distill(x, ids, lp, up, kind)


@pytest.mark.parametrize("n", [3, 80, 310])  # one launch, and three
@pytest.mark.parametrize("low", [-1e9, -1e30, torch.finfo(torch.float32).min])
def test_losses_where_everything_is_masked(low, n):
    """Rows of one value, however low: a uniform softmax; and masks behind which whole vectors lie before
    the first other value comes."""
    x, ids, lp, up = make_rows(n, 9000, 8, torch.float32, 19)
    x[0] = low
    x[1, :8800] = low
    x[2] = low
    x[2, ids[2]] = 1.0
    for kind in ("forward", "reverse", "jsd"):
        check_distill(x, ids, lp, up, kind)
    check_xent(x, ids[:, 0], up, 0.0, 0.0)
    check_topk(x.to(DEV), 60)


@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("low", [-math.inf, -1e30, torch.finfo(torch.float32).min])
def test_distill_all_mass_on_the_entries(low, kind, tail):
    """Nothing left for the tail: every other column is masked, and the teacher's mass is 1."""
    x, ids, lp, up = make_rows(3, 200, 6, torch.float32, 7)
    keep = torch.zeros(3, 200, dtype=torch.bool).scatter_(1, ids, True)
    x = torch.where(keep, x, low)
    lp = torch.log_softmax(lp, 1)
    loss, d = run_distill(x, ids, lp, up, kind=kind, tail=tail)
    want, _ = loss_and_grad(lambda y: distill_rows(y, ids, lp, kind, 0.5, 1.0, tail), x, up)
    span = span_of(x, ids, lp, 1.0)
    check_loss(loss, want, fp32_tol(200, 6, span) * (1 + span))
    assert bool(d.isfinite().all()) and float(d[~keep.to(DEV)].abs().max()) == 0.0
    assert float(d.sum(1).abs().max()) <= fp32_tol(200, 6, span) * (1 + span) * float(up.abs().max())


@pytest.mark.parametrize("kind", ["forward", "reverse", "jsd"])
def test_distill_sure_student(kind):
    """A student whose tail mass is far below fp32's resolution of 1: the tail is still what its
    columns sum to."""
    x, ids, lp, up = make_rows(4, 4000, 4, torch.float32, 8, spread=0.5)
    x[torch.arange(4), ids[:, 0]] += torch.tensor([20.0, 30.0, 40.0, 60.0])
    check_distill(x, ids, lp, up, kind)


@pytest.mark.parametrize("kind,tail", KINDS)
def test_distill_gradient_matches_differences(kind, tail):
    """Along a direction u, (L(x + h u) - L(x - h u)) / 2h of the kernel's own fp32 loss.  L errs by
    tol (1 + span) at each end, the difference adds h^2 |L'''| / 6 <= h^2 for |u| = 1."""
    x, ids, lp, up = make_rows(5, 600, 10, torch.float32, 9, boost=3.0)
    g = torch.Generator().manual_seed(2)
    u = torch.nn.functional.normalize(torch.randn(5, 600, generator=g), dim=1)
    h = 0.05
    _, d = run_distill(x, ids, lp, torch.ones(5), kind=kind, tail=tail)
    ends = [ops.logits_distill((x + s * h * u).to(DEV), ids.to(DEV), lp.to(DEV), kind=kind, tail=tail).double()
            for s in (1, -1)]
    num = ((ends[0] - ends[1]) / (2 * h)).cpu()
    span = span_of(x, ids, lp, 1.0)
    tol = fp32_tol(600, 10, span) * (1 + span)
    assert bool(((d.double().cpu() * u).sum(1) - num).abs().max() <= tol / h + h * h + tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_losses_on_strided_and_unaligned_logits(dtype):
    g = torch.Generator().manual_seed(11)
    base = (2 * torch.randn(4, 5, 1300, generator=g)).to(dtype).to(DEV)
    for view in (base[:, 1:, 3:1004], base[:, :, ::2], base[1:2].expand(4, 5, 1300), base[0, 0, 1:]):
        x = view.detach().requires_grad_(True)
        shape = view.shape[:-1]
        V = view.shape[-1]
        ids = torch.randint(0, V, (*shape, 9), generator=g).to(DEV)
        lp = torch.log_softmax(torch.randn(*shape, 9, generator=g), -1).to(DEV) - 0.1
        up = torch.randn(shape, generator=g).to(DEV)
        loss = ops.logits_distill(x, ids, lp, "jsd")
        d, = torch.autograd.grad(loss, x, up)
        flat = (view.reshape(-1, V).cpu(), ids.reshape(-1, 9).cpu(), lp.reshape(-1, 9).cpu(), up.reshape(-1).cpu())
        loss2, d2 = run_distill(flat[0].contiguous(), *flat[1:], kind="jsd")
        # the same arithmetic on other groups of eight: equal up to the order of the sums
        assert float((loss.detach().reshape(-1) - loss2).abs().max()) <= fp32_tol(V, 9, 20) * 20
        want, dw = loss_and_grad(lambda y: distill_rows(y, flat[1], flat[2], "jsd"), flat[0], flat[3])
        check_grad(d.reshape(-1, V), dw, dtype, grad_scale(*flat), fp32_tol(V, 9, 20))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,ld,off", [(5, 1001, 1040, 0), (70, 1000, 1001, 1), (3, 2049, 2056, 7), (66, 9, 9, 5),
                                        (310, 1000, 1001, 1), (300, 9, 9, 5)])
def test_losses_on_a_matrix_with_a_row_stride(n, V, ld, off, dtype):
    """2-D views are taken as they are: rows of any alignment, gradients (dense) aligned otherwise."""
    x, ids, lp, up = make_rows(n, V, 7, dtype, n + ld)
    buf = torch.full((n * ld + 16,), 77.0, dtype=dtype, device=DEV)
    view = buf[off:off + n * ld].view(n, ld)[:, :V]
    view.copy_(x)
    xd = view.detach().requires_grad_(True)
    assert xd.stride(0) == ld
    t = ids[:, 0]
    for loss, rows in ((ops.logits_distill(xd, ids.to(DEV), lp.to(DEV), "reverse"),
                        lambda y: distill_rows(y, ids, lp, "reverse")),
                       (ops.logits_cross_entropy(xd, t.to(DEV)), lambda y: xent_rows(y, t))):
        d, = torch.autograd.grad(loss, xd, up.to(DEV))
        want, dw = loss_and_grad(rows, x, up)
        span = span_of(x, ids, lp, 1.0)
        tol = fp32_tol(V, 7, span)
        check_loss(loss.detach(), want, tol * (1 + span))
        check_grad(d, dw, dtype, grad_scale(x, ids, lp, up) + up.double().abs()[:, None] * torch.softmax(x.double(), 1),
                   tol * (1 + span))


@pytest.mark.parametrize("n", [3, 80, 310])  # one launch, and three
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_bad_logits_stay_in_their_row(n, bad):
    x, ids, lp, up = make_rows(n, 3000, 5, torch.float32, 17)
    ok = torch.arange(n) != 1
    clean = run_distill(x, ids, lp, up, kind="jsd")
    for col in (int(ids[1, 2]), [c for c in range(3000) if c not in ids[1].tolist()][1234]):
        y = x.clone()
        y[1, col] = bad
        loss, d = run_distill(y, ids, lp, up, kind="jsd")
        assert bool(loss[1].isnan()) and bool(d[1].isnan().any())
        assert torch.equal(loss[ok], clean[0][ok]) and torch.equal(d[ok], clean[1][ok])
        xd = y.to(DEV).requires_grad_(True)
        ce = ops.logits_cross_entropy(xd, ids[:, 0].to(DEV), 0.1)
        assert bool(ce[1].isnan()) and bool(ce[ok].isfinite().all())


def test_other_types_of_entries_and_no_grad():
    x, ids, lp, up = make_rows(4, 300, 6, torch.float32, 18)
    want, _ = run_distill(x, ids, lp, up)
    coarse = lp.to(torch.bfloat16)
    want_coarse, _ = run_distill(x, ids, coarse.float(), up)
    with torch.no_grad():
        xd = x.to(DEV)
        assert torch.equal(ops.logits_distill(xd, ids.to(DEV), lp.to(DEV)), want)
        assert torch.equal(ops.logits_distill(xd, ids.to(DEV, torch.int32), lp.to(DEV, torch.float64)), want)
        got = ops.logits_distill(xd, ids.to(DEV).t().contiguous().t(), coarse.to(DEV))
        assert torch.equal(got, want_coarse)
        ce = ops.logits_cross_entropy(xd, ids[:, 0].to(DEV, torch.int32))
        assert torch.equal(ce, ops.logits_cross_entropy(xd, ids[:, 0].to(DEV)))
    lpg = lp.to(DEV).requires_grad_(True)  # a teacher's log-probs are constants
    loss = ops.logits_distill(x.to(DEV).requires_grad_(True), ids.to(DEV), lpg)
    assert torch.autograd.grad(loss.sum(), lpg, allow_unused=True) == (None,)


def check_xent(x, t, up, smoothing, z):
    xd = x.to(DEV).requires_grad_(True)
    loss = ops.logits_cross_entropy(xd, t.to(DEV), smoothing, z)
    d, = torch.autograd.grad(loss, xd, up.to(DEV))
    want, dw = loss_and_grad(lambda y: xent_rows(y, t, smoothing, z), x, up)
    safe = t.clamp(0, x.shape[1] - 1)
    xx = x.double()
    logp = torch.log_softmax(xx, 1)
    fin = logp[logp.isfinite()]
    lse = torch.logsumexp(xx, 1)
    big = float(fin.abs().max().clamp(max=200)) + abs(z) * float(lse.abs().max()) ** 2 + float(lse.abs().max())
    tol = fp32_tol(x.shape[1], 1, float(fin.abs().max().clamp(max=200)))
    check_loss(loss.detach(), want, tol * (1 + big))
    p = logp.exp()
    rest = 1 - p.gather(1, safe[:, None])  # what the target's gradient is made of
    scale = (p * (1 + 2 * abs(z) * lse.abs()[:, None])).scatter(
        1, safe[:, None], rest + smoothing + 2 * abs(z) * lse.abs()[:, None]) + smoothing / x.shape[1]
    # The 64-bit gradient at a target is p_y - 1 with p_y rounded near 1 (2^-53) and the difference
    # formed from lse - x_y, rounded at the size of the logits: where p_y is 1 - 1e-18, as below, it is
    # 0 and off by the whole value, within 2^-52 of the logits' size.
    ref_err = up.double().abs()[:, None] * 2.0 ** -52 * (1 + float(lse.abs().max()))
    check_grad(d, dw, x.dtype, up.double().abs()[:, None] * scale, tol, ref_err)
    return loss.detach(), d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("smoothing,z", [(0.0, 0.0), (0.1, 1e-3)])
@pytest.mark.parametrize("n,V", [(1, 1), (2, 7), (9, 1001), (3, 50257), (400, 257), (2, 151936), (130, 20011),
                                 (330, 20011)])
def test_cross_entropy_sizes(n, V, smoothing, z, dtype):
    x, ids, _, up = make_rows(n, V, 1, dtype, n + V)
    t = ids[:, 0].clone()
    if n > 1:
        t[1] = -100
        up[-1] = 0.0
    loss, d = check_xent(x, t, up, smoothing, z)
    if n > 1:
        assert float(loss[1]) == 0.0 and float(d[1].float().abs().max()) == 0.0
        assert float(d[-1].float().abs().max()) == 0.0


def test_cross_entropy_sure_masked_and_out_of_range():
    x, ids, _, up = make_rows(5, 900, 1, torch.float32, 13, spread=0.5)
    t = ids[:, 0].clone()
    x[0, t[0]] += 40  # a loss near e^-50: log1p of the others, not 1 - p
    x[1, torch.arange(900) != t[1]] = -math.inf
    x[2, 100:] = torch.where(torch.arange(100, 900) == t[2], x[2, 100:], torch.finfo(torch.float32).min)
    loss, _ = check_xent(x, t, up, 0.0, 0.0)
    assert 0.0 < float(loss[0]) < 1e-15 and float(loss[1]) == 0.0
    t[3], t[4] = 900, -7
    xd = x.to(DEV).requires_grad_(True)
    loss = ops.logits_cross_entropy(xd, t.to(DEV))
    loss.sum().backward()
    assert bool(loss[3:].isnan().all()) and bool(loss[:3].isfinite().all())
    assert bool(xd.grad[3:].isnan().all()) and bool(xd.grad[:3].isfinite().all())


def test_empty_batches():
    x = torch.empty(0, 90, device=DEV, requires_grad=True)
    e = torch.empty(0, 4, device=DEV)
    for loss in (ops.logits_distill(x, e.long(), e), ops.logits_cross_entropy(x, e[:, 0].long())):
        assert loss.shape == (0,)
        loss.sum().backward()
    h = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(90, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    for loss in (ops.lmhead_distill(h, w, e.long(), e), ops.lmhead_cross_entropy(h, w, e[:, 0].long())):
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert dh.shape == h.shape and float(dw.float().abs().max()) == 0.0


def test_second_order_is_refused_and_backward_twice_repeats():
    x, ids, lp, up = make_rows(3, 100, 4, torch.float32, 1)
    xd = x.to(DEV).requires_grad_(True)
    loss = ops.logits_distill(xd, ids.to(DEV), lp.to(DEV)).sum()
    a, = torch.autograd.grad(loss, xd, retain_graph=True)
    b, = torch.autograd.grad(loss, xd, retain_graph=True)
    assert torch.equal(a, b)
    c, = torch.autograd.grad(loss, xd, create_graph=True)
    with pytest.raises(RuntimeError):
        c.sum().backward()


def test_rows_behind_the_matrix_and_other_streams():
    """Writes stay inside the outputs (a strided gradient through the C entry), and two streams do not
    share anything."""
    x, ids, lp, up = make_rows(6, 500, 8, torch.bfloat16, 15)
    xd, idd, lpd, upd = x.to(DEV), ids.to(DEV), lp.to(DEV), up.to(DEV)
    state = ops._row_state(6, 8, torch.device(DEV))
    loss = torch.full((8,), 7.0, device=DEV)
    prm = ops._distill_params("forward", 0.5, 1.0, True)
    s = N.stream_of(torch.device(DEV))
    N.call("ikrl_logits_distill_fwd", N.ptr(xd), N.i32(1), N.i64(500), N.i64(6), N.i32(500), N.ptr(idd), N.ptr(lpd),
           N.i32(8), prm, N.ptr(loss), N.ptr(state), N.sz(state.numel()), s)
    out = torch.full((8, 520), 3.0, device=DEV, dtype=torch.bfloat16)
    N.call("ikrl_logits_distill_bwd", N.ptr(xd), N.i32(1), N.i64(500), N.i64(6), N.i32(500), N.i32(8), prm,
           N.ptr(state), N.sz(state.numel()), N.ptr(upd), N.ptr(out), N.i64(520), s)
    want_loss, want_d = run_distill(x, ids, lp, up)
    assert torch.equal(loss[:6], want_loss) and torch.equal(out[:6, :500], want_d)
    assert bool((loss[6:] == 7).all()) and bool((out[:, 500:] == 3).all()) and bool((out[6:] == 3).all())
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    torch.cuda.synchronize()
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                xs = xd.detach().requires_grad_(True)
                ls = ops.logits_distill(xs, idd, lpd)
                res.append((ls.detach(), *torch.autograd.grad(ls, xs, upd)))
    torch.cuda.synchronize()
    for ls, ds in res:
        assert torch.equal(ls, want_loss) and torch.equal(ds, want_d)


# ---- through the LM head --------------------------------------------------------------------------


def make_head(n, H, V, K, seed, w_std=None):
    g = torch.Generator().manual_seed(seed)
    w_std = w_std or 1.5 / math.sqrt(H)
    w = (w_std * torch.randn(V, H, generator=g)).to(torch.bfloat16)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)]) if n else torch.empty(0, K).long()
    top = min(3, K)
    h = torch.randn(n, H, generator=g)
    h = h + ((5.0 / (w_std ** 2 * H)) * w[ids[:, :top]].float()).sum(1)
    lp = torch.log_softmax(2 * torch.randn(n, K, generator=g), 1) + math.log(0.85)
    up = torch.randn(n, generator=g) * (torch.rand(n, generator=g) < 0.7)
    return h.to(torch.bfloat16), w, ids, lp.float(), up


def check_head(h, w, up, got, rows_fn, scale_fn, K, span, cached=False):
    """(loss, dh, dw) against 64 bits.  A logit errs by at most H half-steps of fp32 of its terms'
    magnitudes (delta); dS is rounded to bf16 once (2^-8 of itself) from p, q that err by 4 delta; the
    second products add V (or n) half-steps; the outputs are rounded to bf16.

    cached, dS from the logit cache: dS = coef q + level with numerators q rounded to fp16, so the sum
    errs by 2^-11 of coef q (at most g p, which A holds), before the level is taken off, where q is at
    least 2^-14 of its chunk's maximum, and by 2^-25 of that maximum (its row's largest A) elsewhere."""
    loss, dh, dw = (t.detach().double().cpu() for t in got)
    hd, wd = h.double(), w.double()
    n, H = h.shape
    V = w.shape[0]
    x = hd @ wd.t()
    want, ds = loss_and_grad(rows_fn, x, up)
    delta = EPS32 * H * float((hd.abs() @ wd.abs().t()).max())
    tol = fp32_tol(V, K, span) * (1 + span)
    check_loss(loss, want, tol + 2 * delta * (2 + span))
    A = scale_fn(x)
    unit = 2 ** -8 * ds.abs() + (4 * delta + tol) * A
    if cached:
        unit = unit + 2 ** -11 * A + 2 ** -25 * A.amax(1, keepdim=True)
    for g, ref, e in ((dh, ds @ wd, unit @ wd.abs() + V * EPS32 * (ds.abs() @ wd.abs())),
                      (dw, ds.t() @ hd, unit.t() @ hd.abs() + n * EPS32 * (ds.abs().t() @ hd.abs()))):
        err = (g - ref).abs()
        lim = e + 2 ** -8 * ref.abs() + 1e-30
        assert bool((err <= lim).all()), (float(err.max()), float((err / lim).max()))
    # and the whole: independent roundings of 2^-8 at most leave far less than 2^-8 of the norm
    for g, ref in ((dh, ds @ wd), (dw, ds.t() @ hd)):
        if float(ref.norm()) > 0:
            assert float((g - ref).norm() / ref.norm()) <= 2 ** -7 + 8 * delta


def run_head(f, h, w, up, *args, **kw):
    hd, wd = h.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    loss = f(hd, wd, *[a.to(DEV) if isinstance(a, torch.Tensor) else a for a in args], **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (hd, wd), up.to(DEV)))


HEADS = [(1, 8, 5, 2), (130, 64, 1001, 16), (257, 512, 3000, 33), (64, 1024, 5003, 8), (300, 2048, 1536, 256),
         (1100, 256, 1003, 20)]


@pytest.mark.parametrize("kind,tail", KINDS)
@pytest.mark.parametrize("n,H,V,K", HEADS)
def test_head_distill(n, H, V, K, kind, tail):
    h, w, ids, lp, up = make_head(n, H, V, K, n + V)
    if n > 5:
        ids[2] = -1
        ids[3, K // 2:] = -1
        ids[4, 1] = ids[4, 0]
    t = 1.5
    got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind=kind, tail=tail, temperature=t, beta=0.3)
    span = span_of(h.double() @ w.double().t(), ids, lp, t)
    check_head(h, w, up, got, lambda y: distill_rows(y, ids, lp, kind, 0.3, t, tail),
               lambda x: grad_scale(x, ids, lp, up, t), K, span)
    if n > 5:
        assert float(got[0][2]) == 0.0 and float(got[1][2].float().abs().max()) == 0.0


@pytest.mark.parametrize("smoothing,z", [(0.0, 0.0), (0.1, 1e-3)])
@pytest.mark.parametrize("n,H,V,K", HEADS)
def test_head_cross_entropy(n, H, V, K, smoothing, z):
    h, w, ids, _, up = make_head(n, H, V, 1, n + V + 1)
    t = ids[:, 0].clone()
    if n > 5:
        t[1::3] = -100
    got = run_head(ops.lmhead_cross_entropy, h, w, up, t, label_smoothing=smoothing, z_loss=z)
    x = h.double() @ w.double().t()
    lse = torch.logsumexp(x, 1)
    span = float((x.amax(1) - x.amin(1)).max()) + abs(z) * float(lse.abs().max()) ** 2

    def scale(x):
        p = torch.softmax(x, 1)
        s = (p + smoothing / V).scatter(1, t.clamp(min=0)[:, None], 1.0) * (1 + 2 * z * lse.abs()[:, None])
        return up.double().abs()[:, None] * s

    check_head(h, w, up, got, lambda y: xent_rows(y, t, smoothing, z), scale, 1, span)
    if n > 5:
        assert float(got[0][1].abs()) == 0.0 and float(got[1][1].float().abs().max()) == 0.0


@pytest.mark.parametrize("n", [200, 1100])
@pytest.mark.parametrize("knobs", [dict(cta_pairs=0), dict(wide=0), dict(wide=1), dict(skip_zero_rows=0),
                                   dict(balance_splits=0)])
def test_head_under_each_kernel_choice(knobs, n):
    h, w, ids, lp, up = make_head(n, 1024, 2050, 12, 21)
    ids[5] = -1
    with N.tuning(**knobs):
        got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="jsd")
    span = span_of(h.double() @ w.double().t(), ids, lp, 1.0)
    check_head(h, w, up, got, lambda y: distill_rows(y, ids, lp, "jsd"), lambda x: grad_scale(x, ids, lp, up), 12,
               span)


@pytest.mark.parametrize("loss", ["jsd", "xent"])
@pytest.mark.parametrize("n,H,V,slots", [(200, 1024, 2056, 200), (3, 64, 40, 3), (600, 1024, 1000, 600),
                                         (600, 1024, 1000, 250), (600, 256, 1000, 1),
                                         (1100, 1024, 1000, 1100), (1100, 1024, 1000, 450), (1100, 256, 1000, 1)])
def test_head_with_the_logit_cache(n, H, V, slots, loss, monkeypatch):
    """dS from stored numerators: all rows in the cache, some, one; rows without entries hold no slot; a
    second backward, without the cache, agrees within the roundings; the kernel choices share it."""
    h, w, ids, lp, up = make_head(n, H, V, 9, n + V + slots)
    t = ids[:, 0].clone()
    if n > 5:
        ids[1::3] = -1
        t[1::3] = -100
    asked = []
    monkeypatch.setattr(ops, "logit_cache_rows", lambda *a: asked.append(a) or slots)
    monkeypatch.setattr(ops, "_ROW_CACHE_MIN_HIDDEN", 1)
    if loss == "jsd":
        f, args, kw = ops.lmhead_distill, (ids, lp), dict(kind="jsd", temperature=1.3)
        rows = lambda y: distill_rows(y, ids, lp, "jsd", 0.5, 1.3)  # noqa: E731
        scale = lambda x: grad_scale(x, ids, lp, up, 1.3)  # noqa: E731
        span = span_of(h.double() @ w.double().t(), ids, lp, 1.3)
    else:
        f, args, kw = ops.lmhead_cross_entropy, (t,), dict(label_smoothing=0.1)
        rows = lambda y: xent_rows(y, t, 0.1)  # noqa: E731
        x = h.double() @ w.double().t()
        span = float((x.amax(1) - x.amin(1)).max())

        def scale(x):
            p = torch.softmax(x, 1)
            return up.double().abs()[:, None] * (p + 0.1 / V).scatter(1, t.clamp(min=0)[:, None], 1.0)

    for knobs in ({}, dict(wide=0), dict(wide=1), dict(cta_pairs=0), dict(skip_zero_rows=0)):
        with N.tuning(**knobs):
            check_head(h, w, up, run_head(f, h, w, up, *args, **kw), rows, scale, 9, span, cached=True)
    assert bool(asked) == (n > 1024)
    hd, wd = h.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    out = f(hd, wd, *[a.to(DEV) for a in args], **kw)
    first = torch.autograd.grad(out, (hd, wd), up.to(DEV), retain_graph=True)
    again = torch.autograd.grad(out, (hd, wd), up.to(DEV))
    for g1, g2 in zip(first, again):
        assert float((g1.float() - g2.float()).norm()) <= 4 * 2 ** -8 * float(g2.float().norm())


@pytest.mark.parametrize("n", [400, 1100])
def test_head_in_chunks_one_sided_and_bad_rows(n):
    h, w, ids, lp, up = make_head(n, 256, 1000, 6, 22)
    up = up + 0.01
    whole = run_head(ops.lmhead_distill, h, w, up, ids, lp)
    parts = run_head(ops.lmhead_distill, h, w, up, ids, lp, chunk_rows=128)
    assert torch.equal(whole[0], parts[0]) and torch.equal(whole[1], parts[1])
    # dW: fp32 sums over the chunks instead of one, both rounded to bf16
    diff = (whole[2].float() - parts[2].float()).abs()
    assert bool((diff <= 2 ** -7 * whole[2].float().abs() + 1e-5).all())
    hd = h.to(DEV).requires_grad_(True)
    dh, = torch.autograd.grad(ops.lmhead_distill(hd, w.to(DEV), ids.to(DEV), lp.to(DEV)), hd, up.to(DEV))
    assert torch.equal(dh, whole[1])
    wd = w.to(DEV).requires_grad_(True)
    dw, = torch.autograd.grad(ops.lmhead_distill(h.to(DEV), wd, ids.to(DEV), lp.to(DEV)), wd, up.to(DEV))
    assert torch.equal(dw, whole[2])
    # an id past the vocabulary: NaN in its row, nowhere else as long as its upstream is 0
    ids[7, 2] = 1000
    up[7] = 0.0
    got = run_head(ops.lmhead_distill, h, w, up, ids, lp)
    assert bool(got[0][7].isnan()) and int(got[0].isnan().sum()) == 1
    assert bool(got[1].isfinite().all()) and bool(got[2].isfinite().all())


@pytest.mark.parametrize("n", [600, 1100])
def test_head_cache_in_chunks(n, monkeypatch):
    h, w, ids, lp, up = make_head(n, 256, 1000, 6, 24)
    monkeypatch.setattr(ops, "_ROW_CACHE_MIN_HIDDEN", 1)
    for slots in (n, n // 2):
        monkeypatch.setattr(ops, "logit_cache_rows", lambda *a: slots)
        span = span_of(h.double() @ w.double().t(), ids, lp, 1.0)
        got = run_head(ops.lmhead_distill, h, w, up, ids, lp, kind="reverse", chunk_rows=256)
        check_head(h, w, up, got, lambda y: distill_rows(y, ids, lp, "reverse"),
                   lambda x: grad_scale(x, ids, lp, up), 6, span, cached=True)


@pytest.mark.parametrize("n", [60, 400, 1100])
def test_head_c_entry_accumulates_an_fp32_dweight(n):
    """dW added to what is there, in fp32; dH left out; nothing written behind the outputs."""
    H, V = 128, 600
    h, w, ids, _, up = make_head(n, H, V, 1, 25)
    hd, wd, t, upd = h.to(DEV), w.to(DEV), ids[:, 0].contiguous().to(DEV), up.to(DEV)
    dev = torch.device(DEV)
    lib, s = N.lib(), N.stream_of(dev)
    state = ops._row_state(n, 1, dev)
    loss = torch.full((n + 3,), 7.0, device=DEV)
    ws = torch.empty(lib.ikrl_lmhead_row_loss_fwd_workspace_bytes(n, H, V), dtype=torch.uint8, device=DEV)
    none = (N.i64(0), None, None, None)
    N.call("ikrl_lmhead_cross_entropy_fwd", N.ptr(hd), N.ptr(wd), N.ptr(t), N.i64(n), N.i32(H), N.i32(V), N.f32(0.1),
           N.f32(0), N.ptr(loss), N.ptr(state), N.sz(state.numel()), *none, N.ptr(ws), N.sz(ws.numel()), s)
    base = torch.randn(V + 2, H, generator=torch.Generator().manual_seed(1)).to(DEV)
    acc = base.clone()
    wb = torch.empty(lib.ikrl_lmhead_row_loss_bwd_workspace_bytes(n, H, V, 0, N.IKRL_DTYPE_F32, 1), dtype=torch.uint8,
                     device=DEV)
    for _ in range(2):
        N.call("ikrl_lmhead_cross_entropy_bwd", N.ptr(hd), N.ptr(wd), N.i64(n), N.i32(H), N.i32(V), N.f32(0.1),
               N.f32(0), N.ptr(state), N.sz(state.numel()), N.ptr(upd), N.i64(0), None, N.ptr(acc),
               N.i32(N.IKRL_DTYPE_F32), N.i32(1), *none, N.ptr(wb), N.sz(wb.numel()), s)
    assert bool((loss[n:] == 7).all()) and torch.equal(acc[V:], base[V:])
    x = h.double() @ w.double().t()
    _, ds = loss_and_grad(lambda y: xent_rows(y, ids[:, 0], 0.1), x, up)
    want = 2 * (ds.t() @ h.double())
    got = (acc[:V] - base[:V]).double().cpu()
    # dS rounded to bf16, fp32 sums of n terms and two additions to values of about 1
    lim = 2 * (2 ** -8 + 8 * n * EPS32) * (ds.abs().t() @ h.double().abs()) + 1e-3 * (ds.abs().t() @ h.double().abs()) \
        + 4 * EPS32 * (base[:V].double().cpu().abs() + want.abs())
    assert bool(((got - want).abs() <= lim).all())


def test_head_fp32_weight_and_3d_hidden():
    h, w, ids, lp, up = make_head(24, 128, 700, 5, 23)
    got = run_head(ops.lmhead_distill, h.float().reshape(4, 6, 128), w.float(), up.reshape(4, 6),
                   ids.reshape(4, 6, 5), lp.reshape(4, 6, 5))
    want = run_head(ops.lmhead_distill, h, w, up, ids, lp)
    assert got[0].shape == (4, 6) and got[1].dtype == got[2].dtype == torch.float32
    assert torch.equal(got[0].reshape(-1), want[0])
    assert torch.equal(got[1].reshape(24, 128), want[1].float()) and torch.equal(got[2], want[2].float())


# ---- captures, and the operators together ---------------------------------------------------------


@pytest.mark.parametrize("head", [False, True])
def test_captured_step_replays_on_new_inputs(head):
    """Teacher top-k, distillation, its backward and a cross entropy in one graph; two graphs replayed
    in turn give what eager calls give on each of their inputs."""
    def inputs(seed):
        h, w, ids, _, up = make_head(70, 1024, 1500, 1, seed)
        t = ids[:, 0].clone()
        t[::4] = -100
        teacher = (h.float() @ w.float().t() * 0.8).to(torch.bfloat16)
        return [a.to(DEV) for a in (h, w, teacher, t, up + 0.01)]

    def step(h, w, teacher, t, up):
        lp, ids = ops.logits_topk(teacher, 12, 1.3)
        if head:
            leaves = (h.detach().requires_grad_(True), w.detach().requires_grad_(True))
            a = ops.lmhead_distill(*leaves, ids, lp, "reverse", temperature=1.3)
            b = ops.lmhead_cross_entropy(*leaves, t, 0.1, 1e-3)
        else:
            leaves = (teacher.detach().requires_grad_(True),)
            a = ops.logits_distill(*leaves, ids, lp, "reverse", temperature=1.3)
            b = ops.logits_cross_entropy(*leaves, t, 0.1, 1e-3)
        return (lp, ids, a.detach(), b.detach(), *torch.autograd.grad((a, b), leaves, (up, up)))

    graphs = []
    side = torch.cuda.Stream()
    for seed in (31, 32):
        buf = inputs(seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*buf)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*buf)
        graphs.append((g, buf, out))
    for seed in (33, 34):
        for i, (g, buf, out) in enumerate(graphs):
            new = inputs(seed + 10 * i)
            for dst, src in zip(buf, new):
                dst.copy_(src)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i, (g, buf, out) in enumerate(graphs):
            with N.tuning(skip_zero_rows=0):  # a capture runs every row
                want = step(*buf)
            for o, w_ in zip(out, want):
                assert torch.equal(o, w_)


def _tiny_policy(seed):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(vocab_size=1000, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=32, max_position_embeddings=256,
                      tie_word_embeddings=True, use_cache=False, initializer_range=0.08)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(seed)
    return Qwen3ForCausalLM(cfg).to(device=DEV, dtype=torch.bfloat16)


def test_teacher_and_student_policies():
    """A teacher's top log-probs into a student's distillation and supervised losses, through the fused
    head and through materialised logits, against the 64-bit definitions on the model's own rows."""
    from invokerl_b200.policy import PolicyModel

    teacher, student = (PolicyModel.from_model(_tiny_policy(s)) for s in (0, 1))
    g = torch.Generator().manual_seed(3)
    B, T, k = 3, 40, 12
    tok = torch.randint(0, 1000, (B, T), generator=g).to(DEV)
    am = (torch.arange(T)[None] < torch.tensor([40, 25, 7])[:, None]).to(DEV)
    lp, ids = teacher.topk_log_probs(tok, am, k, temperature=1.2)
    assert lp.shape == ids.shape == (B, T, k) and not lp.requires_grad
    off = ~am.clone()
    off[:, 0] = True
    assert bool((ids[off] == -1).all()) and bool((lp[off] == -math.inf).all())
    assert bool((ids[~off] >= 0).all()) and bool((lp[~off].exp().sum(-1) < 1).all())
    with torch.no_grad():
        hs = teacher.model.model(input_ids=tok, attention_mask=am).last_hidden_state
        tl = torch.nn.functional.linear(hs[:, :T - 1], teacher.model.lm_head.weight)
    wl, wi = ops.logits_topk(tl, k, 1.2)
    assert torch.equal(ids[:, 1:][~off[:, 1:]], wi[~off[:, 1:]])
    assert torch.equal(lp[:, 1:][~off[:, 1:]], wl[~off[:, 1:]])

    mask = am.clone()
    mask[:, :5] = False
    n = mask.sum()
    losses = {}
    for fsdp in (False, True):
        student._fsdp_wrapped = fsdp
        student.model.zero_grad(set_to_none=True)
        per = student.distill_loss(tok, am, ids, lp, kind="reverse", temperature=1.2)
        ce = student.cross_entropy_loss(tok, am, label_smoothing=0.1, z_loss=1e-4, loss_mask=mask)
        assert per.shape == ce.shape == (B, T) and per.dtype == torch.float32
        assert float(per[off].abs().max()) == 0.0 and float(ce[~mask].abs().max()) == 0.0
        ((per * mask).sum() / n + 0.5 * ce.sum() / n).backward()
        for name, prm in student.model.named_parameters():
            assert prm.grad is not None and bool(prm.grad.isfinite().all()), name
        losses[fsdp] = (per.detach(), ce.detach())
    with torch.no_grad():
        hs = student.model.model(input_ids=tok, attention_mask=am).last_hidden_state[:, :-1].reshape(-1, 128)
        w = student.model.lm_head.weight
    x = (hs.double() @ w.double().t()).cpu()
    i2, l2 = ids[:, 1:].reshape(-1, k).cpu(), lp[:, 1:].reshape(-1, k).cpu()
    want = distill_rows(x, i2, l2, "reverse", 0.5, 1.2).reshape(B, T - 1)
    tg = torch.where(mask[:, 1:], tok[:, 1:], -100).reshape(-1).cpu()
    want_ce = xent_rows(x, tg, 0.1, 1e-4).reshape(B, T - 1)
    span = float((x.amax(1) - x.amin(1)).max())
    delta = EPS32 * 128 * float((hs.double().abs() @ w.double().abs().t()).max())
    tol = (fp32_tol(1000, k, span) + 4 * delta) * (1 + span)
    # logits in memory are rounded to bf16: half a step of the largest, at both places of a log-prob
    coarse = tol + 2 * half_step(torch.bfloat16) * float(x.abs().max()) * (1 + span)
    for fsdp, t in ((False, tol), (True, coarse)):
        assert float((losses[fsdp][0][:, 1:].cpu() - want).abs().max()) <= t
        assert float((losses[fsdp][1][:, 1:].cpu() - want_ce).abs().max()) <= t


@pytest.mark.parametrize("n,V,k", [(2, 40000, 50), (40, 1500, 12), (400, 20000, 200), (700, 20000, 100)])
def test_topk_repeats_bit_for_bit(n, V, k):
    """Ids and log-probs do not depend on the order in which columns reach the buffer."""
    x = torch.randn(n, V, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(DEV)
    lp, ids = ops.logits_topk(x, k, 1.3)
    for _ in range(5):
        lp2, ids2 = ops.logits_topk(x, k, 1.3)
        assert torch.equal(lp, lp2) and torch.equal(ids, ids2)


# ---- offsets past 32 bits -------------------------------------------------------------------------


@pytest.mark.parametrize("n", [5, 310, 460])
def test_rows_far_apart(n):
    """Rows whose offsets pass 2^31 elements give what the same rows side by side give."""
    V, stride = 1003, (2 ** 31 + 2 ** 20) // (n - 1) // 8 * 8
    store = torch.empty((n - 1) * stride + V, dtype=torch.bfloat16, device=DEV)
    far = store.as_strided((n, V), (stride, 1))
    x, ids, lp, up = make_rows(n, V, 9, torch.bfloat16, n)
    near = torch.empty(n, 1008, dtype=torch.bfloat16, device=DEV)[:, :V]  # rows aligned alike
    far.copy_(x)
    near.copy_(x)
    res = []
    for logits in (far, near):
        a = logits.detach().requires_grad_(True)
        out = list(ops.logits_topk(a, 20))
        for loss in (ops.logits_distill(a, ids.to(DEV), lp.to(DEV), "jsd"),
                     ops.logits_cross_entropy(a, ids[:, 0].contiguous().to(DEV), 0.1)):
            g, = torch.autograd.grad(loss, a, up.to(DEV))
            out += [loss.detach(), g]
        res.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_gradients_past_2_31_elements():
    """Equal rows of a matrix of more than 2^31 elements: the first and the last get the same."""
    n, V, H = 14200, 151936, 1024
    assert n * V > 2 ** 31
    g = torch.Generator().manual_seed(2)
    row = (2 * torch.randn(V, generator=g)).to(torch.bfloat16).to(DEV)
    ids = torch.randperm(V, generator=g)[:7].expand(n, 7).contiguous().to(DEV)
    lp = (torch.log_softmax(torch.randn(7, generator=g), 0) - 0.1).expand(n, 7).contiguous().to(DEV)
    up = torch.ones(n, device=DEV)

    def first_and_last(loss, grad):
        assert bool((loss == loss[0]).all()) and bool(loss[0].isfinite())
        assert torch.equal(grad[0], grad[-1]) and float(grad[-1].abs().max()) > 0

    x = row.expand(n, V).contiguous().requires_grad_(True)
    top, _ = ops.logits_topk(x, 5)
    assert torch.equal(top[0], top[-1])
    for loss in (ops.logits_distill(x, ids, lp, "reverse"), ops.logits_cross_entropy(x, ids[:, 0].contiguous())):
        d, = torch.autograd.grad(loss, x, up)
        first_and_last(loss.detach(), d)
        del d
    del x, loss
    w = (0.03 * torch.randn(V, H, generator=g)).to(torch.bfloat16).to(DEV).requires_grad_(True)
    h = torch.randn(H, generator=g).to(torch.bfloat16).to(DEV).expand(n, H).contiguous().requires_grad_(True)
    for loss in (ops.lmhead_distill(h, w, ids, lp, "reverse"), ops.lmhead_cross_entropy(h, w, ids[:, 0].contiguous())):
        dh, dw = torch.autograd.grad(loss, (h, w), up)
        first_and_last(loss.detach(), dh)
        assert bool(dw[-1].isfinite().all())
