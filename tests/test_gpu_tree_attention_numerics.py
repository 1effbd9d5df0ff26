"""Tree attention's numerics where products or scales are far apart, against its formula in 64 bits.

Tolerances.  A score is off by at most d = 2^-19 of the sum of its products' magnitudes plus 2^-22 of its own size
(f32 sums of products with at least 22 bits; scaling and exponent).  The result is an average with weights p of
code * vscale: errors of the scores move it by at most 2 d of its size = 127 sum p vscale.  The weights enter the second
product with 22 bits, or within 2^-31 of the largest p vscale where they are far smaller (of n positions: n 2^-31 of the
size); with the f32 sums, joins and the division less than 2^-18 of the size for up to 4096 positions.  Then the
result's own rounding, half a step of its type.
"""
import numpy as np
import pytest

from devmem import HALF_STEP, decode, encode
from test_gpu_tree_attention import LONG, Case, bits, ctx, hip, run  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def formula(case):
    """out, lse, the account's new weights in 64 bits; a result's size; how far scores may be off by their sums and by themselves."""
    q = decode(case.q, case.kind)
    B, n, H, D = q.shape
    out, size, lse = np.zeros(q.shape), np.zeros((B, n, H, 1)), np.full((B, n, H), -np.inf)
    sums, scores = np.zeros((B, n, H, 1)), np.zeros((B, n, H, 1))
    weight = np.zeros((B, case.positions))
    for b in range(B):
        L, c = int(case.lens[b]), int(case.counts[b])
        T = L + c
        vis = np.concatenate([np.ones((c, L), bool), case.sees[b, :c, :c]], 1)
        some = vis.any(1)
        ks, vs = case.ks[b, :T, None].astype(np.float64), case.vs[b, :T, None].astype(np.float64)
        for h in range(H if T and c else 0):
            g = h // (H // case.kv_heads)
            k = case.k[b, :T, g] * ks
            s = np.where(vis, q[b, :c, h] @ k.T * case.scale, -np.inf)
            big = np.where(vis, np.abs(q[b, :c, h]) @ np.abs(k.T) * case.scale, 0)
            top = np.where(some, s.max(1, initial=-np.inf), 0)
            e = np.exp(s - top[:, None])
            den = e.sum(1, keepdims=True)
            p = e / np.where(den > 0, den, 1)
            out[b, :c, h], size[b, :c, h] = p @ (case.v[b, :T, g] * vs), 127 * (p @ vs)
            lse[b, :c, h] = np.where(some, top + np.log(np.where(den > 0, den, 1))[:, 0], -np.inf)
            sums[b, :c, h, 0], scores[b, :c, h, 0] = big.max(1) * 2.0 ** -19, np.abs(np.where(vis, s, 0)).max(1) * 2.0 ** -22
            weight[b, :T] += p.sum(0)
    return out, lse, weight, size, sums, scores


def check(case, out, lse, one_product=False, equal_scores=False):
    """one_product: a score has one product, whose sum does not round.  equal_scores: the scores that count are equal, so
    their errors cancel in the weights."""
    w_out, w_lse, _, size, sums, scores = formula(case)
    off = scores if one_product else sums + scores
    got = decode(out.get(), case.kind)
    err = np.abs(got - w_out)
    tol = size * ((0 if equal_scores else 2 * off) + 2.0 ** -18) + np.abs(w_out) * HALF_STEP[case.kind]
    l_tol = off[..., 0] + 2.0 ** -18 + np.abs(np.where(np.isneginf(w_lse), 0, w_lse)) * 2.0 ** -22
    for b in range(case.batch):
        c = int(case.counts[b])
        assert (err[b, :c] <= tol[b, :c]).all(), (b, (err[b, :c] / np.maximum(size[b, :c], 1e-300)).max(), np.argwhere(~(err[b, :c] <= tol[b, :c]))[:4])
        g, w = lse.get()[b, :c], w_lse[b, :c]
        some = ~np.isneginf(w)
        assert np.array_equal(np.isneginf(g), ~some) and (np.abs(g[some] - w[some]) <= l_tol[b, :c][some]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nodes,max_len", [(1, None), (6, None), (24, LONG)])
def test_weights_keep_their_bits(ctx, hip, kind, nodes, max_len):  # noqa: F811
    """Small scores over a few positions: a weight rounded to 11 bits would show in the small results."""
    case = Case(kind=kind, batch=2, nodes=nodes, heads=16, kv_heads=2, lens=(9, 3), qscale=2.0 ** -6)
    _, out, lse, _ = run(ctx, hip, case, max_len=max_len)
    check(case, out, lse)


def taken_over(kind, ratio, nodes, positions=640, early=256, code=0, batch=1, kv_heads=2, dim=128, seed=0):
    """The first `early` positions have V scales `ratio` times the last ones' and scores 0.  The others' scores are all 170,
    or higher by 10.2 bits for every 5 of `code` with each 128 positions, the scales shrinking with them.  q has one value
    that is not 0, so a score is one product, and equal scores come out equal."""
    case = Case(kind=kind, batch=batch, nodes=nodes, heads=16, kv_heads=kv_heads, dim=dim, lens=(positions - nodes,) * batch,
                sees=np.ones((batch, nodes, nodes), bool), spare=0, seed=seed)
    q = np.zeros(case.q.shape)
    q[..., 3] = 16
    case.q = encode(q, kind)[0]
    case.ks[:] = 1.0
    at = np.arange(positions)
    codes = np.where(at >= early, (at - early) // 128 + 1, 0) * code if code else np.where(at >= early, 120, 0)
    case.k[..., 3] = codes[None, :, None]
    fall = float(ratio) ** (1 - codes / codes.max())
    case.vs = (case.vs * fall).astype(np.float32)
    return case


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio", [1e-9, 1e4, 1e6, 1e9, 1e25])
@pytest.mark.parametrize("nodes,max_len", [(1, 0), (6, 0), (24, LONG)])
def test_small_values_that_take_over(ctx, hip, kind, ratio, nodes, max_len):  # noqa: F811
    """Positions whose V scales are far smaller (or larger) than those before them, and which outweigh them by 2^245."""
    case = taken_over(kind, ratio, nodes)
    _, out, lse, _ = run(ctx, hip, case, max_len=max_len, account=False)
    check(case, out, lse, one_product=True, equal_scores=True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("code,ratio", [(5, 1e6), (12, 1e12), (5, 1e20), (5, 1e30)])
def test_small_values_that_take_over_in_steps(ctx, hip, kind, code, ratio):  # noqa: F811
    """The maximum grows again and again while the values shrink; with 1e30, what comes first still counts most."""
    case = taken_over(kind, ratio, 3, positions=1024, early=128, code=code)
    _, out, lse, _ = run(ctx, hip, case, max_len=0, account=False)
    check(case, out, lse, one_product=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio", [1e-9, 1e6, 1e25])
@pytest.mark.parametrize("dim", [64, 128])
def test_small_values_that_take_over_in_many_columns(ctx, hip, kind, ratio, dim):  # noqa: F811
    """As many sequences and columns as take no splits: workgroups of four tiles, each over all chunks."""
    case = taken_over(kind, ratio, 20, batch=66, kv_heads=4, dim=dim)
    _, out, lse, _ = run(ctx, hip, case, account=False)
    check(case, out, lse, one_product=True, equal_scores=True)


@pytest.mark.parametrize("first,then", [(2.0 ** -130, 2.0 ** -20), (2.0 ** -112, 1.0)])
def test_smallest_values_first(ctx, hip, first, then):  # noqa: F811
    """V scales too small for the weights to be brought where they should do not keep those behind them from there."""
    case = Case(nodes=2, heads=16, kv_heads=2, lens=(638,), qscale=2.0 ** -6, spare=0)
    case.vs *= np.float32(then)
    case.vs[:, :256] = first
    _, out, lse, _ = run(ctx, hip, case, max_len=0, account=False)
    check(case, out, lse)


@pytest.mark.parametrize("heads,nodes,dim", [(2, 3, 128), (8, 3, 128), (2, 2, 64), (16, 3, 64)])
def test_not_finite_rows_in_the_account(ctx, hip, heads, nodes, dim):  # noqa: F811
    """A row whose q is not finite makes the weights of the positions that it sees NaN, and of no others, whether its
    scores are kept (few columns) or computed again."""
    case = Case(nodes=nodes, heads=heads, kv_heads=1, dim=dim, lens=(40,), sees=np.eye(nodes, dtype=bool)[None])
    case.q[0, 1, 1, 5] = np.nan
    _, _, _, acc = run(ctx, hip, case)
    got = acc.get()[0]
    nan = np.zeros(case.positions, bool)
    nan[:40] = nan[41] = True      # the cached positions and itself
    assert np.array_equal(np.isnan(got), nan)
    case.q[0, 1, 1, 5] = 0
    case.sees[0, 1] = False        # the others' weights, as if it saw nothing of the nodes
    _, _, weight, _, sums, scores = formula(case)
    for p in (40, 42)[:nodes - 1]:
        want = case.account[0, p] * case.decay + weight[0, p]
        off = (sums + scores).max()
        assert abs(got[p] - want) <= weight[0, p] * (2 * off + 2.0 ** -17) + want * 2.0 ** -22
    assert np.array_equal(got[40 + nodes:], case.account[0, 40 + nodes:])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("nodes,max_len", [(3, None), (24, LONG)])
@pytest.mark.parametrize("qscale,scale", [(2.0 ** -110, 1e-30), (2.0 ** -124, 1e-8), (2.0 ** -124, 1e-45), (1e37, 1e-38)])
def test_scales_at_the_ends(ctx, hip, kind, nodes, max_len, qscale, scale):  # noqa: F811
    """Tiny q and scales: all scores are as good as 0, and masked positions still count nothing."""
    case = Case(kind=kind, nodes=nodes, heads=8, kv_heads=2, lens=(37,), qscale=qscale)
    case.scale = float(np.float32(scale))
    q, k, v, ks, vs = hip.put(case.q, case.qtype), hip.put(case.k), hip.put(case.v), hip.put(case.ks), hip.put(case.vs)
    out, lse = hip.put(np.zeros_like(case.q), case.qtype), hip.put(np.zeros(case.q.shape[:3], np.float32))
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, max_len=max_len))
    ctx.tree_attention(q, k, v, ks, vs, hip.put(case.lens), out, mask=hip.put(bits(case.sees)), lse=lse, max_len=max_len, scale=scale, workspace=ws)
    check(case, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ks", [20.0, 35.0, 70.0, 140.0, -140.0, 300.0, -500.0, 1100.0, 30000.0])
@pytest.mark.parametrize("wide", [False, True])
def test_equal_scores_beyond_whole_numbers(ctx, hip, kind, ks, wide):  # noqa: F811
    """Scores whose size f32 holds in steps of 1 and more: equal ones weigh the same, wherever they stand and whatever
    the V scales around them.  A third of the positions have the largest score, the others one lower by an eighth."""
    case = taken_over(kind, 1.0, 20 if wide else 3, batch=66 if wide else 1, kv_heads=4 if wide else 2, dim=64)
    q = np.zeros(case.q.shape)
    q[..., 3] = 2.0 ** 15
    case.q, case.ks[:] = encode(q, kind)[0], ks
    rng = np.random.default_rng(7)
    top = rng.random(case.positions) < np.where(np.arange(case.positions) < 200, 0.1, 0.5)
    case.k[..., 3] = np.where(top, 112, 98)[None, :, None] * (1 if ks > 0 else -1)
    case.vs = (case.vs * np.exp2(rng.integers(-3, 4, case.positions))).astype(np.float32)
    _, out, lse, _ = run(ctx, hip, case, max_len=None if wide else 0, account=False)
    check(case, out, lse, one_product=True, equal_scores=True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("ks", [2.0 ** -9, 20.0, -140.0, 30000.0])
@pytest.mark.parametrize("nodes,batch,kv_heads", [(1, 1, 8), (3, 1, 2), (20, 66, 4), (20, 20, 2)])
def test_account_of_large_scores(ctx, hip, kind, ks, nodes, batch, kv_heads):  # noqa: F811
    """Scores from 900 on: the weights of equal ones are equal, and a row's weights are 1 in all, however far f32's steps
    at the score's size are apart.  (A weight below 2^-126, f32's smallest normal number, may come out 0: of 900 and 1 / 8
    less it is 2^-160, which f32 does not have.)"""
    case = taken_over(kind, 1.0, nodes, batch=batch, kv_heads=kv_heads, dim=64)
    q = np.zeros(case.q.shape)
    q[..., 3] = 2.0 ** 15
    case.q, case.ks[:] = encode(q, kind)[0], ks
    top = np.random.default_rng(7).random(case.positions) < 0.3
    case.k[..., 3] = np.where(top, 112, 98)[None, :, None] * (1 if ks > 0 else -1)
    case.account[:] = 0
    _, _, _, acc = run(ctx, hip, case)
    _, _, weight, _, _, _ = formula(case)
    assert (weight > 0.01).any() and (np.abs(acc.get() - weight) <= weight * 2.0 ** -17 + 2.0 ** -126 * nodes * 16).all()      # (of 16 heads)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("code", [5, 8, 11, 14, 17])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("wide", [False, True])
def test_many_small_weights(ctx, hip, kind, code, first, wide):  # noqa: F811
    """One position outweighs each of the others by 2^(2.04 code) and has the value 0: what the others sum up to."""
    case = taken_over(kind, 1.0, 20 if wide else 2, positions=640 if wide else 4096, batch=66 if wide else 1, kv_heads=4 if wide else 2)
    case.k[..., 3], case.v[:], case.vs[:] = 0, 101, 1 / 64
    at = 0 if first else case.positions - 1
    case.k[:, at, :, 3], case.v[:, at] = code, 0
    _, out, lse, _ = run(ctx, hip, case, max_len=None if wide else 0, account=False)
    check(case, out, lse, one_product=True)
