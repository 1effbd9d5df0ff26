"""cache_attention where scores are large or not finite, in its kernels of 16, 32 and 128 columns (test_cache_plans.py: that they are
reached)."""
import numpy as np
import pytest

from cacheref import U, Cache, check_attention, clamped, rounding
from devmem import decode
from test_gpu_cache_attention import Case, ctx, hip  # noqa: F401

pytestmark = pytest.mark.gpu

# name: (arguments, columns of a tile)
KERNELS = {
    "f32 of 8 bits": (dict(kind="f32", bits=8, batch=1, tokens=3, heads=4, kv_heads=2, dim=128, positions=110, lens=[107]), 16),
    "f32 of 4 bits": (dict(kind="f32", bits=4, batch=1, tokens=3, heads=4, kv_heads=2, dim=64, positions=110, lens=[107]), 16),
    "f16 of 8 bits": (dict(kind="f16", bits=8, batch=1, tokens=3, heads=4, kv_heads=2, dim=64, positions=110, lens=[107]), 16),
    "bf16 of 4 bits": (dict(kind="bf16", bits=4, batch=1, tokens=3, heads=4, kv_heads=2, dim=128, positions=110, lens=[107]), 16),
    "bf16, in splits": (dict(kind="bf16", bits=8, batch=1, tokens=1, heads=4, kv_heads=2, dim=64, positions=3000, lens=[2990]), 16),
    "32, f32": (dict(kind="f32", bits=8, batch=1, tokens=300, heads=8, kv_heads=2, dim=64, positions=4305, lens=[4000]), 32),
    "32, f16 of 4 bits": (dict(kind="f16", bits=4, batch=1, tokens=300, heads=8, kv_heads=2, dim=128, positions=4305, lens=[4000]), 32),
    "128": (dict(kind="bf16", bits=8, batch=1, tokens=256, heads=512, kv_heads=1, dim=64, positions=1900, lens=[1640]), 128),
    "128, in splits": (dict(kind="bf16", bits=8, batch=1, tokens=256, heads=32, kv_heads=4, dim=128, positions=26262, lens=[26001]), 128),
}


def far(c, sizes, heads):
    """A row of q a size, in turn: size times values of 1 to 2, of both signs."""
    rng = np.random.default_rng(1)
    q = rng.choice([-1, 1], (1, c["tokens"], c["heads"], c["dim"])) * rng.uniform(1, 2, (1, c["tokens"], c["heads"], c["dim"]))
    return q * np.resize(sizes, c["tokens"] * heads).reshape(1, c["tokens"], heads, 1)


def check(c, heads=None):
    """Scores that are equal or far apart: softmax in 64 bits weighs them as the formula does, whatever a dot product in f32 is off by.
    Tolerances are those of cacheref's attention without that, lse's with it."""
    out, lse = decode(c.out.get(), c.kind), c.lse.get()
    lens, counts = clamped(c.lens, c.counts, c.q.shape[1], c.cache.k.shape[1])
    n, count, dim, all_heads = lens[0] + counts[0], counts[0], c.q.shape[3], c.q.shape[2]
    p, j = lens[0] + np.arange(count)[:, None], np.arange(n)[None]
    for h in heads or range(all_heads):
        g = h * c.cache.k.shape[2] // all_heads
        k, v, q = c.cache.values(0, 0)[:n, g], c.cache.values(1, 0)[:n, g], decode(c.q[0, :count, h], c.kind)
        # exact before they are multiplied by the position's scale, or equal ones would differ here
        dot = q @ c.cache.k[0, :n, g].T.astype(np.float64) * c.cache.kscale[0, :n].astype(np.float64) if c.bits == 8 else q @ k.T
        s = np.where(j <= p, c.scale * dot, -np.inf)
        m = s.max(1, keepdims=True)
        w = np.exp(s - m)
        den = w.sum(1, keepdims=True)
        want, wlse, sums = w / den @ v, (m + np.log(den))[:, 0], (p + 65) * U
        tol = (2 * sums + 2.0 ** -21 + (U if c.kind == "f32" else 2.0 ** -18)) * (w / den @ np.abs(v)) + rounding(c.kind, want)
        assert (np.abs(out[0, :count, h] - want) <= tol).all(), (h, (np.abs(out[0, :count, h] - want) / tol).max(1))
        mag = (c.scale * (np.abs(q) @ np.abs(k).T)).max(1)
        ltol = (dim + 16) * U * mag + sums[:, 0] + 2.0 ** -20 + 2 * U * np.abs(wlse)
        assert (np.abs(lse[0, :count, h] - wlse) <= ltol).all(), (h, lse[0, :count, h], wlse)


def some(c):
    return sorted({0, 1, c["heads"] // 2, c["heads"] - 1})


SIZES = [2.0 ** e for e in (0, 10, 17, 18, 19, 20, 21, 22, 23, 24, 26, 28, 30, 31, 32, 34, 37, 40, 60, 100)]


@pytest.mark.parametrize("name", sorted(KERNELS))
@pytest.mark.parametrize("by", ["q", "scale"])
def test_equal_scores_of_any_size(ctx, hip, name, by):  # noqa: F811
    """All keys alike: the result is the mean of the values, of scores from 1 to 2^100 and -2^100."""
    c = KERNELS[name][0]
    cache = Cache(np.random.default_rng(0), c["bits"], 1, c["positions"], c["kv_heads"], c["dim"])
    cache.k[:], cache.kscale[:] = cache.k[0, 0], cache.kscale[0, 0]
    if by == "q":
        check(Case(hip, **c, q=far(c, SIZES if c["kind"] != "f16" else [1.0, 2.0 ** 13], c["heads"]), cache=cache).run(ctx), some(c))
        return
    for scale in (0.125, 2.0 ** 14, 2.0 ** 18 / 3, 2.0 ** 22 / 7, 2.0 ** 25 / 3, 2.0 ** 29 / 5, 2.0 ** 35, 2.0 ** 90 / 3):
        check(Case(hip, **c, q=far(c, [1.0], c["heads"]), cache=cache, scale=float(np.float32(scale))).run(ctx), some(c))


@pytest.mark.parametrize("name", sorted(KERNELS))
@pytest.mark.parametrize("rising", [True, False])
def test_scores_far_apart(ctx, hip, name, rising):  # noqa: F811
    """Keys of four sizes, in runs of positions: the largest scores have all of the weight, be they the first or the last that a row sees."""
    c = KERNELS[name][0]
    cache = Cache(np.random.default_rng(0), c["bits"], 1, c["positions"], c["kv_heads"], c["dim"])
    run = np.arange(c["positions"]) * 4 // c["positions"]
    run = run if rising else 3 - run
    cache.k[:], cache.kscale[:] = cache.k[0, 0], cache.kscale[0, 0]
    cache.kscale[:] = (2.0 ** run / 64 if c["bits"] == 8 else 124 + run).reshape(1, -1, *[1] * (cache.kscale.ndim - 2))
    sizes = [2.0 ** e for e in (20, 24, 28, 31, 32, 34, 40, 60, 100)] if c["kind"] != "f16" else [1.0, 2.0 ** 13]
    check(Case(hip, **c, q=far(c, sizes, c["heads"]), cache=cache, scale=1.0 if c["kind"] != "f16" else 2.0 ** 20).run(ctx), some(c))


@pytest.mark.parametrize("name", sorted(KERNELS))
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_rows_whose_scores_are_all_minus_infinity(ctx, hip, name, bad):  # noqa: F811
    """An infinite value of q over codes of one sign: all scores of the row are infinite, of one sign or the other, and it is NaN either way; the
    rows beside it are as they were."""
    c = KERNELS[name][0]
    cache = Cache(np.random.default_rng(0), c["bits"], 1, c["positions"], c["kv_heads"], c["dim"])
    cache.k[..., 3] = -5 if c["bits"] == 8 else cache.k[..., 3] | 0x88      # (of 4 bits the dims 6 and 7)
    if c["bits"] == 4:
        cache.k[..., 3] |= 0x11
    q = np.random.default_rng(1).standard_normal((1, c["tokens"], c["heads"], c["dim"]))
    clean = Case(hip, **c, q=q, cache=cache).run(ctx)
    rows = [(0, 1), (c["tokens"] - 1, c["heads"] - 1), (c["tokens"] // 2, 0)]
    for token, head in rows:
        q[0, token, head, 3 if c["bits"] == 8 else 7] = bad
    got = Case(hip, **c, q=q, cache=cache).run(ctx)
    out, lse, want, wlse = decode(got.out.get(), c["kind"]), got.lse.get(), decode(clean.out.get(), c["kind"]), clean.lse.get()
    for token, head in rows:
        assert np.isnan(out[0, token, head]).all() and np.isnan(lse[0, token, head])
        out[0, token, head], lse[0, token, head] = want[0, token, head], wlse[0, token, head]
    assert (out == want).all() and (lse == wlse).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,window", [([0], None), ([40], 1)])
def test_one_position_whose_score_is_minus_infinity(ctx, hip, kind, bits, lens, window):  # noqa: F811
    """The first token of a prompt, and a token that sees itself alone."""
    cache = Cache(np.random.default_rng(0), bits, 1, 50, 2, 64)
    cache.k[:] = np.abs(cache.k) // 2 + 1 if bits == 8 else (cache.k & 0x77) | 0x11
    q = np.random.default_rng(1).standard_normal((1, 1, 4, 64))
    q[0, 0, 1, 9], q[0, 0, 2, 9] = -np.inf, np.inf
    c = Case(hip, kind, bits, 1, 1, 4, 2, 64, 50, lens, window=window, q=q, cache=cache).run(ctx)
    out, lse = decode(c.out.get(), kind)[0, 0], c.lse.get()[0, 0]
    assert np.isnan(out[1:3]).all() and np.isnan(lse[1:3]).all()
    assert np.isfinite(out[[0, 3]]).all() and np.isfinite(lse[[0, 3]]).all()


@pytest.mark.parametrize("name", sorted(n for n in KERNELS if KERNELS[n][0]["kind"] == "f32"))
@pytest.mark.parametrize("large", [2.0 ** 10, 2.0 ** 20, 2.0 ** 40])
def test_one_large_channel_of_q_costs_the_others_no_bits(ctx, hip, name, large):  # noqa: F811
    """Where K is 0 there: products are those of f32 numbers, each value of q with all of its bits."""
    c = KERNELS[name][0]
    cache = Cache(np.random.default_rng(0), c["bits"], 1, c["positions"], c["kv_heads"], c["dim"])
    cache.k[..., 0] = 0 if c["bits"] == 8 else cache.k[..., 0] & 0xf0
    q = np.random.default_rng(1).standard_normal((1, c["tokens"], c["heads"], c["dim"]))
    q[..., 0] = large
    got = Case(hip, **c, q=q, cache=cache).run(ctx)
    if c["tokens"] == 3:
        got.check()
    else:      # (some rows: the bounds are computed row by row)
        some_rows(got, [0, 77, 299])


def some_rows(c, tokens):
    """check_attention of these tokens of sequence 0, each as a sequence of its own."""
    for i in tokens:
        n = int(c.lens[0]) + i
        check_attention(c.out.get()[:, i:i + 1], c.lse.get()[:, i:i + 1], c.q[:, i:i + 1], c.cache, np.array([n], np.uint32), np.array([1], np.uint32), 0, 0,
                        c.scale, c.kind)


@pytest.mark.parametrize("name", sorted(n for n in KERNELS if KERNELS[n][0]["bits"] == 4))
@pytest.mark.parametrize("side", [2, 3])
@pytest.mark.parametrize("window", [None, 40])
def test_scale_bytes_that_are_nan(ctx, hip, name, side, window):  # noqa: F811
    """E8M0's 255 is NaN: the rows of its kv head that see the position are NaN, all others as they were."""
    c = {**KERNELS[name][0], "window": window}
    tokens, heads, kv_heads = c["tokens"], c["heads"], c["kv_heads"]
    cache = Cache(np.random.default_rng(0), 4, 1, c["positions"], kv_heads, c["dim"])
    q = np.random.default_rng(1).standard_normal((1, tokens, heads, c["dim"]))
    clean = Case(hip, **c, q=q, cache=cache).run(ctx)
    want, wlse = decode(clean.out.get(), c["kind"]), clean.lse.get()
    for at, g, block in ((c["lens"][0] + tokens // 2, 0, 0), (c["lens"][0] - 45, kv_heads - 1, c["dim"] // 32 - 1), (c["lens"][0] + tokens - 1, 0, 1)):
        saved, cache.arrays()[side][0, at, g, block] = cache.arrays()[side][0, at, g, block], 255
        got = Case(hip, **c, q=q, cache=cache).run(ctx)
        cache.arrays()[side][0, at, g, block] = saved
        p, group = c["lens"][0] + np.arange(tokens), heads // kv_heads
        sees = np.zeros((tokens, heads), bool)
        sees[:, g * group:(g + 1) * group] = ((at <= p) & ((p - at < window) if window else True))[:, None]
        out, lse = decode(got.out.get(), c["kind"])[0], got.lse.get()[0]
        assert np.isnan(out[sees]).all() and np.isnan(lse[sees]).all()
        assert (out[~sees] == want[0][~sees]).all() and (lse[~sees] == wlse[0][~sees]).all()
