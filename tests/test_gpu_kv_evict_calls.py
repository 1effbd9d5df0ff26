"""Calls of eviction (qxg_kv_select, qxg_kv_compact) that its documentation allows, against numpy."""
import numpy as np
import pytest

from test_gpu_kv_evict import chosen, ctx, hip  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("positions", [900, 4000, 30000])
@pytest.mark.parametrize("budget", [64, 700])
def test_lengths_replaced_in_place(ctx, hip, positions, budget):  # noqa: F811
    """kept is lens: the lengths become the kept ones, the lists as with two arrays."""
    rng = np.random.default_rng(positions + budget)
    lens = np.array([positions, 0, budget - 1, budget, budget + 1, positions // 2, -1, 800], np.int32).clip(-1, positions)
    account = np.exp(rng.standard_normal((len(lens), positions))).astype(np.float32)
    keep, now = hip.put(np.full((len(lens), budget), -7, np.int32)), hip.put(lens)
    ctx.kv_select(hip.put(account), now, keep, now, sinks=3, recent=9)
    got, n = keep.get(), now.get()
    for g, length in enumerate(lens):
        want = chosen(account[g], positions if length < 0 else length, budget, 3, 9)
        assert n[g] == len(want) and np.array_equal(got[g, :n[g]], want) and (got[g, n[g]:] == -7).all(), length
