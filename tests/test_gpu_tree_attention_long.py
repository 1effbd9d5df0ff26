"""Tree attention whose workgroups go through many chunks of positions, of four tiles (the launches of much work) and of one,
with the lengths and launches that a program has: every kernel's loop over chunks, whole or in splits, against the
formula in 64 bits.  test_ops_host.py holds each case to the kernel and the chunks that it is meant for.

Tolerances as in test_gpu_tree_attention_numerics.py (22 bits and n 2^-31 of the size for n positions; up to 16048 here: 2^-17
of the size in all)."""
import numpy as np
import pytest

from devmem import HALF_STEP, decode
from test_gpu_tree_attention import Case, ctx, hip, run  # noqa: F401  (fixtures among them)
from test_gpu_tree_attention_numerics import formula

pytestmark = pytest.mark.gpu

# name: (the case, four tiles a workgroup, splits: 1 or more, chunks of a split at least)
PLANS = {
    "two_long": (dict(batch=2, nodes=48, heads=16, kv_heads=2, lens=(16000, 9000)), True, 2, 8),
    "two_long_counts": (dict(batch=2, nodes=48, heads=16, kv_heads=2, lens=(16000, 9000), counts=(48, 5)), True, 2, 6),
    "two_long_small_heads": (dict(batch=2, nodes=48, heads=16, kv_heads=2, dim=64, lens=(16000, 9001)), True, 2, 8),
    "one_long": (dict(nodes=64, heads=32, kv_heads=4, lens=(12000,)), True, 2, 8),
    "whole": (dict(batch=40, nodes=70, heads=16, kv_heads=4, lens=tuple(range(270, 350, 2)), counts=(70, 33, 1, 0) * 10), True, 1, 8),
    "whole_small_heads": (dict(batch=40, nodes=70, heads=16, kv_heads=4, dim=64, lens=tuple(range(270, 350, 2))), True, 1, 8),
    "whole_beyond_64": (dict(batch=66, nodes=20, heads=16, kv_heads=4, lens=tuple(range(490, 622, 2)), counts=(20, 7, 0) * 22), True, 1, 15),
    "splits_beyond_64": (dict(batch=70, nodes=24, heads=4, kv_heads=1, lens=tuple(range(1250, 1950, 10))), True, 2, 6),
    "chunk_of_a_prompt": (dict(nodes=1024, heads=16, kv_heads=8, lens=(200,), sees="chain"), True, 2, 8),
    "chunk_of_a_prompt_little_work": (dict(nodes=1024, heads=4, kv_heads=2, dim=64, lens=(200,), sees="chain"), False, 2, 4),
    "tree_of_1024": (dict(nodes=1024, heads=16, kv_heads=8, lens=(200,)), True, 2, 8),
    "one_token": (dict(nodes=1, heads=32, kv_heads=4, lens=(12000,)), False, 2, 4),
    "tokens_beyond_64": (dict(batch=70, nodes=1, heads=8, kv_heads=8, lens=tuple(range(1250, 1950, 10))), False, 1, 30),
}


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", sorted(PLANS))
def test_formula(ctx, hip, name, kind):  # noqa: F811
    case = Case(kind=kind, **PLANS[name][0])
    _, out, lse, acc = run(ctx, hip, case, max_len=int(case.lens.max()))
    w_out, w_lse, weight, size, sums, scores = formula(case)
    off = sums + scores
    err, tol = np.abs(decode(out.get(), kind) - w_out), size * (2 * off + 2.0 ** -17) + np.abs(w_out) * HALF_STEP[kind]
    g_lse, g_acc = lse.get(), acc.get().astype(np.float64)
    for b in range(case.batch):
        c, end = int(case.counts[b]), int(case.lens[b] + case.counts[b])
        assert (err[b, :c] <= tol[b, :c]).all(), (b, np.argwhere(~(err[b, :c] <= tol[b, :c]))[:4])
        assert (decode(out.get()[b, c:], kind) == 7).all() and (g_lse[b, c:] == 7).all()      # rows behind the last node
        assert (np.abs(g_lse[b, :c] - w_lse[b, :c]) <= off[b, :c, :, 0] + 2.0 ** -18 + np.abs(w_lse[b, :c]) * 2.0 ** -22).all()
        want = case.account[b, :end] * case.decay + weight[b, :end]
        t_acc = want * 2.0 ** -22 + weight[b, :end] * (2 * off[b].max() + 2.0 ** -17)
        assert (np.abs(g_acc[b, :end] - want) <= t_acc).all() and np.array_equal(g_acc[b, end:], case.account[b, end:].astype(np.float64))
