"""Row losses without a GPU: the 64-bit definitions the GPU tests compare with, refusals of the Python
entry points and of the C entries."""

import math

import pytest
import torch

from invokerl_b200 import _native as N
from invokerl_b200 import ops
from row_loss_math import TAIL_EPS, distill_rows, entry_mask, loss_and_grad, xent_rows

KINDS = [("forward", True), ("forward", False), ("reverse", True), ("jsd", True)]


def _case(n=4, V=23, K=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(n, V, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    lp = torch.log_softmax(torch.randn(n, K, generator=g), 1) + math.log(0.8)
    return x, ids, lp


@pytest.mark.parametrize("kind,tail", KINDS)
def test_gradient_formula_and_differences(kind, tail):
    """p_v (a - sum p a) with the outcomes' derivatives a, autograd, and central differences agree."""
    x, ids, lp = _case()
    T, b = 1.7, 0.3

    def f(y):
        return distill_rows(y, ids, lp, kind, b, T, tail)

    up = torch.tensor([1.0, -0.5, 2.0, 0.25], dtype=torch.float64)
    _, d = loss_and_grad(f, x, up)
    # differences: error ~ h^2 / 6 |f'''| + eps |f| / h with h = 1e-5
    h = 1e-5
    for v in range(x.shape[1]):
        e = torch.zeros_like(x)
        e[:, v] = h
        num = (f(x + e) - f(x - e)) / (2 * h) * up
        assert float((num - d[:, v]).abs().max()) <= 1e-9
    p = torch.softmax(x / T, 1)
    for r in range(x.shape[0]):
        q = lp[r].double().exp()
        pk = p[r, ids[r]]
        rest = torch.ones(x.shape[1], dtype=torch.bool)
        rest[ids[r]] = False
        pt, qt = p[r, rest].sum(), 1 - q.sum()
        if not tail:
            q = q / q.sum()
            want = p[r].clone()
            want[ids[r]] -= q
        else:
            P, Q = torch.cat([pk, pt[None]]), torch.cat([q, qt[None]])
            a = {"forward": -Q / P, "reverse": (P / Q).log() + 1,
                 "jsd": (1 - b) * (P / (b * Q + (1 - b) * P)).log()}[kind]
            per = torch.full_like(p[r], float(a[-1]))
            per[ids[r]] = a[:-1]
            want = p[r] * (per - (P * a).sum())
        assert float((want * up[r] / T - d[r]).abs().max()) <= 1e-12


def test_cross_entropy_definition_matches_torch():
    x, _, _ = _case()
    t = torch.tensor([3, -100, 0, 22])
    want = torch.nn.functional.cross_entropy(x, t, reduction="none", label_smoothing=0.1)
    got = xent_rows(x, t, 0.1)
    assert float((got - want).abs().max()) <= 1e-12
    z = xent_rows(x, t, 0.0, 0.5) - xent_rows(x, t)
    lse = torch.logsumexp(x, 1)
    assert float((z - torch.where(t == -100, 0.0, 0.5 * lse ** 2)).abs().max()) <= 1e-12


def test_entry_rules():
    ids = torch.tensor([[3, 3, -1, 5, 3], [-1, -1, -1, -1, -1]])
    lp = torch.tensor([[-math.inf, -1.0, -0.5, -2.0, -3.0], [0.0] * 5])
    assert entry_mask(ids, lp).tolist() == [[False, True, False, True, False], [False] * 5]
    x = torch.randn(2, 7, dtype=torch.float64)
    one = distill_rows(x[:1], torch.tensor([[3, 5]]), torch.tensor([[-1.0, -2.0]]))
    assert torch.equal(distill_rows(x, ids, lp), torch.cat([one, torch.zeros(1, dtype=torch.float64)]))
    assert TAIL_EPS == 2.0 ** -20


def _cpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_python_refusals_need_no_gpu():
    x, ids, lp = _cpu(2, 9), _cpu(2, 3, dtype=torch.int64), _cpu(2, 3)
    with pytest.raises(ValueError, match="kind"):
        ops.logits_distill(x, ids, lp, kind="backward")
    for f, a in ((ops.logits_distill, (x, ids, lp)), (ops.lmhead_distill, (x, x, ids, lp))):
        with pytest.raises(ValueError, match="tail"):
            f(*a, kind="reverse", tail=False)
        with pytest.raises(ValueError, match="beta"):
            f(*a, kind="jsd", beta=1.0)
        for t in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="temperature"):
                f(*a, temperature=t)
        with pytest.raises(RuntimeError, match="CUDA"):
            f(*a)
    for f, a in ((ops.logits_cross_entropy, (x, ids[:, 0])), (ops.lmhead_cross_entropy, (x, x, ids[:, 0]))):
        with pytest.raises(ValueError, match="label_smoothing"):
            f(*a, label_smoothing=1.5)
        with pytest.raises(ValueError, match="z_loss"):
            f(*a, z_loss=float("nan"))
        with pytest.raises(RuntimeError, match="CUDA"):
            f(*a)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.logits_topk(x, 2)


def test_row_argument_checks():
    ids, lp = _cpu(2, 3, dtype=torch.int64), _cpu(2, 3)
    with pytest.raises(TypeError, match="logits"):
        ops._logits_rows(_cpu(2, 9, dtype=torch.float16))
    with pytest.raises(ValueError, match="teacher"):
        ops._teacher_rows(ids, lp, (3,))
    with pytest.raises(ValueError, match="teacher"):
        ops._teacher_rows(ids, lp[:, :2], (2,))
    with pytest.raises(TypeError, match="whole"):
        ops._teacher_rows(lp, lp, (2,))
    with pytest.raises(TypeError, match="floating"):
        ops._teacher_rows(ids, ids, (2,))
    with pytest.raises(ValueError, match="K ="):
        ops._teacher_rows(_cpu(2, 257, dtype=torch.int64), _cpu(2, 257), (2,))
    with pytest.raises(ValueError, match="K ="):
        ops._teacher_rows(ids[:, :0], lp[:, :0], (2,))
    with pytest.raises(ValueError, match="targets"):
        ops._targets_rows(ids, (2,))
    with pytest.raises(TypeError, match="whole"):
        ops._targets_rows(lp[:, 0], (2,))
    with pytest.raises(ValueError, match="hidden"):
        ops._head_rows(_cpu(2, 8), _cpu(9, 16))
    # rows that overlap (an expanded row) or columns with a stride become a matrix of their own
    assert ops._logits_rows(_cpu(1, 9).expand(4, 9)).stride() == (9, 1)
    assert ops._logits_rows(_cpu(9, 4).t()).stride() == (9, 1)
    assert ops._ld(_cpu(4, 12)[:, :9]) == 12 and ops._ld(_cpu(4, 12)[:1, :9]) == 9


@pytest.fixture(scope="module")
def lib():
    from invokerl_b200.csrc.build import build

    build()
    return N.lib()


def test_c_entries_refuse_before_any_cuda_call(lib):
    p = N.c_void_p(256)

    def params(kind=0, tail=1, beta=0.5, t=1.0):
        return N.DistillParams(kind, tail, beta, t)

    def distill(dtype=1, ld=100, n=4, V=100, K=3, prm=None, nbytes=1 << 20, state=p, x=p):
        N.call("ikrl_logits_distill_fwd", x, N.i32(dtype), N.i64(ld), N.i64(n), N.i32(V), p, p, N.i32(K),
               params() if prm is None else prm, p, state, N.sz(nbytes), None)

    for kw, msg in [(dict(prm=params(kind=3)), "kind"), (dict(prm=params(t=0.0)), "temperature"),
                    (dict(prm=params(t=float("nan"))), "temperature"), (dict(prm=params(kind=1, tail=0)), "tail"),
                    (dict(prm=params(kind=2, beta=0.0)), "beta"), (dict(K=0), "K=0"), (dict(K=257), "K=257"),
                    (dict(ld=99), "bad sizes"), (dict(n=-1), "bad sizes"), (dict(dtype=7), "dtype"),
                    (dict(V=(1 << 21) + 1, ld=1 << 22), "exceeds"), (dict(nbytes=64), "state"),
                    (dict(state=None), "state"), (dict(state=N.c_void_p(264)), "aligned"),
                    (dict(x=N.c_void_p(257)), "aligned"), (dict(x=None), "null pointer")]:
        with pytest.raises(N.IkrlError, match=msg):
            distill(**kw)
    distill(n=0, x=None, state=None)  # no rows: nothing to do
    with pytest.raises(N.IkrlError, match="smoothing"):
        N.call("ikrl_logits_cross_entropy_fwd", p, N.i32(1), N.i64(9), N.i64(2), N.i32(9), p, N.f32(-0.1), N.f32(0), p,
               p, N.sz(1 << 20), None)
    with pytest.raises(N.IkrlError, match="ld_out"):
        N.call("ikrl_logits_cross_entropy_bwd", p, N.i32(1), N.i64(9), N.i64(2), N.i32(9), N.f32(0), N.f32(0), p,
               N.sz(1 << 20), p, p, N.i64(8), None)
    for k, msg in [(0, "K=0"), (257, "K=257"), (10, "of V=9")]:
        with pytest.raises(N.IkrlError, match=msg):
            N.call("ikrl_logits_topk", p, N.i32(1), N.i64(9), N.i64(2), N.i32(9), N.i32(k), N.f32(1), p, p, None)

    def head(n=4, H=64, K=3, nbytes=1 << 24, state_bytes=1 << 20, ws=p, V=100, cache=0, q=p):
        N.call("ikrl_lmhead_distill_fwd", p, p, p, p, N.i64(n), N.i32(H), N.i32(V), N.i32(K), params(), p, p,
               N.sz(state_bytes), N.i64(cache), p, p, q, ws, N.sz(nbytes), None)

    for kw, msg in [(dict(H=12), "multiple of 8"), (dict(n=-1), "bad sizes"), (dict(nbytes=256), "workspace"),
                    (dict(state_bytes=64), "state"), (dict(ws=N.c_void_p(264)), "aligned"), (dict(K=300), "K=300"),
                    (dict(V=1 << 24), "24 bits"),
                    (dict(cache=-1), "cache_rows"), (dict(cache=4, V=101), "multiple of 8"),
                    (dict(cache=4, V=104, q=None), "null cache"), (dict(cache=4, V=104, q=N.c_void_p(258)), "aligned")]:
        with pytest.raises(N.IkrlError, match=msg):
            head(**kw)
    def head_bwd(n, hidden=p, nbytes=1 << 26, state_bytes=1 << 20, ws=p, g=p, dh=p, dw=p):
        N.call("ikrl_lmhead_distill_bwd", hidden, p, N.i64(n), N.i32(64), N.i32(100), N.i32(3), params(), p,
               N.sz(state_bytes), g, N.i64(0), dh, dw, N.i32(N.IKRL_DTYPE_BF16), N.i32(0), N.i64(0), None, None, None,
               ws, N.sz(nbytes), None)

    odd = N.c_void_p(264)
    for n in (4, 400):
        for kw, msg in [(dict(hidden=odd), "aligned"), (dict(nbytes=512), "workspace"), (dict(state_bytes=64), "state"),
                        (dict(ws=odd), "aligned"), (dict(dh=odd), "aligned"), (dict(dw=odd), "aligned"),
                        (dict(g=None), "null pointer"), (dict(dh=None, dw=None), "null pointer")]:
            with pytest.raises(N.IkrlError, match=msg):
                head_bwd(n, **kw)
    with pytest.raises(N.IkrlError, match="bf16 dweight"):
        N.call("ikrl_lmhead_cross_entropy_bwd", p, p, N.i64(4), N.i32(64), N.i32(100), N.f32(0), N.f32(0), p,
               N.sz(1 << 20), p, N.i64(0), p, p, N.i32(N.IKRL_DTYPE_BF16), N.i32(1), N.i64(0), None, None, None, p,
               N.sz(1 << 24), None)


def test_workspace_sizes_grow_with_their_parts(lib):
    s = lib.ikrl_row_loss_state_bytes
    assert s(0, 5) == 256 and s(100, 64) >= 100 * (8 + 4 + 4 + 64 * 12 + 12)
    f = lib.ikrl_lmhead_row_loss_fwd_workspace_bytes
    # three sets of partial sums, the rows that count gathered (above 1024 rows, or 256 of a large product)
    assert f(2000, 1024, 5000) >= lib.ikrl_lmhead_fwd_workspace_bytes(2000, 1024, 5000) + 2000 * 1024 * 2
    assert f(1024, 1024, 5000) < f(1025, 1024, 5000) - 1024 * 1024 * 2
    assert f(256, 4096, 50000) < f(257, 4096, 50000) - 256 * 4096 * 2
    b = lib.ikrl_lmhead_row_loss_bwd_workspace_bytes
    assert b(2000, 1024, 5000, 0, 1, 0) >= lib.ikrl_lmhead_bwd_workspace_bytes(2000, 1024, 5000, 0, 1, 0) + 8000
