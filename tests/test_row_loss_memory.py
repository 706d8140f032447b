"""The memory policy of small logit caches, without a GPU."""

import pytest
import torch

from invokerl_b200 import _native as N
from invokerl_b200 import ops

DEVICE = torch.device("cuda", 0)
N_ROWS, H, V = 100, 64, 1000
CACHE = N_ROWS * (2 * 1024 + 4 * 32)


@pytest.fixture
def policy(monkeypatch):
    """(clock, memory): a policy that sets nothing aside; `memory` holds the free bytes and the times they were asked."""
    from invokerl_b200.csrc.build import build

    build()
    clock, memory = [0.0], {"free": 0, "asked": 0}

    def free_bytes(device):
        memory["asked"] += 1
        return memory["free"]

    monkeypatch.setattr(ops, "_free_bytes", free_bytes)
    monkeypatch.setattr(ops.time, "monotonic", lambda: clock[0])
    prev = ops.set_logit_cache("auto", 0, 1.0)
    yield clock, memory
    ops.set_logit_cache(prev["mode"], prev["reserve_bytes"], prev["fraction"])


def rest():
    ws = N.lib().ikrl_lmhead_row_loss_bwd_workspace_bytes(N_ROWS, H, V, 0, N.IKRL_DTYPE_BF16, 0)
    return ws + 2 * (N_ROWS + V) * H


def fits():
    return ops._small_cache_fits(N_ROWS, H, V, DEVICE, None)


def test_size_of_a_cache_row():
    assert CACHE == N_ROWS * ops.LogitCache.bytes_per_row(V)


def test_the_backward_and_the_reserve_come_first(policy):
    _, memory = policy
    need = CACHE + rest()
    for reserve, fraction in ((0, 1.0), (1 << 30, 1.0), (1 << 20, 0.5)):
        ops.set_logit_cache("auto", reserve, fraction)
        # as for larger calls: (free - backward - outputs - reserve) * fraction
        least = int(rest() + reserve + CACHE / fraction)
        memory["free"] = least - 2
        assert not fits()
        memory["free"] = least + 2
        assert fits()
    assert need < 1 << 30


def test_memory_is_asked_for_once_a_second_and_when_it_runs_out(policy):
    clock, memory = policy
    memory["free"] = rest() + 3 * CACHE
    assert [fits() for _ in range(3)] == [True] * 3 and memory["asked"] == 1
    assert fits() and memory["asked"] == 2  # the three have been freed
    memory["free"] = rest()
    assert [fits() for _ in range(3)] == [True, True, False] and memory["asked"] == 3
    assert not fits() and memory["asked"] == 4
    memory["free"] = 1 << 40
    assert fits() and memory["asked"] == 5
    clock[0] += 0.9
    assert fits() and memory["asked"] == 5
    clock[0] += 0.2
    assert fits() and memory["asked"] == 6
    ops.set_logit_cache("auto", 1 << 41)
    assert not fits() and memory["asked"] == 7
