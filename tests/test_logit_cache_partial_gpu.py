"""A logit cache with fewer slots than active rows, all of which fit one backward chunk: with a bf16 dweight
the cached and the recomputed rows share the chunk, since the workspace holds no fp32 accumulator."""

import pytest
import torch

import oracle
from invokerl_b200 import ops
from invokerl_b200.synthetic import lmhead_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n,H,V,slots", [(600, 1024, 1000, 250), (300, 256, 2056, 1), (400, 2048, 1536, 399)])
def test_one_chunk_of_cached_and_recomputed_rows(n, H, V, slots):
    li = lmhead_inputs(n, H, V, seed=slots, w_std=0.05)
    g = torch.Generator().manual_seed(n)
    up = torch.randn(n, generator=g) * (torch.rand(n, generator=g) < 0.8)
    h, w, t = li.hidden.to(DEV), li.weight.to(DEV), li.targets.to(DEV)
    cache = ops.LogitCache(n, V, slots, h.device)
    logp, lse = ops.lmhead_forward_raw(h, w, t, cache)
    dh, dw = ops.lmhead_backward_raw(h, w, t, lse, up.to(DEV), cache=cache)
    lp_o, dh_o, dw_o = oracle.lmhead_logprob_grads(li.hidden, li.weight, li.targets, up)
    assert float((logp.cpu() - lp_o).abs().max()) <= 2e-3
    for a, b in ((dh, dh_o), (dw, dw_o)):
        assert float((a.cpu().float() - b).norm() / b.norm()) <= 1e-2
    # dW alone, and dH alone (which needs no accumulator and keeps its two chunks)
    _, dw1 = ops.lmhead_backward_raw(h, w, t, lse, up.to(DEV), want_dh=False, cache=cache)
    dh1, _ = ops.lmhead_backward_raw(h, w, t, lse, up.to(DEV), want_dw=False, cache=cache)
    assert torch.equal(dw1, dw)
    assert float((dh1.float() - dh.float()).norm() / dh.float().norm()) <= 1e-2
