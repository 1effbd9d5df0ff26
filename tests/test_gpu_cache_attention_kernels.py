"""What cache_attention's kernels of 32 and 128 columns, and its join of many splits, do apart from prompts of usual values (test_cache_plans.py: that
they are reached)."""
import ctypes
import threading

import numpy as np
import pytest

from cacheref import Cache, check_attention
from devmem import Hip, decode, encode
from test_gpu_cache_attention import Case, ctx, hip  # noqa: F401
from test_gpu_cache_attention_scores import KERNELS
from test_gpu_cache_far import Far

pytestmark = pytest.mark.gpu
WIDE = sorted(n for n in KERNELS if KERNELS[n][1] > 16)

# name: arguments of calls with more than 64 splits
SPLITS = {
    "f32 of 8 bits": dict(kind="f32", bits=8, batch=1, tokens=1, heads=4, kv_heads=1, dim=64, positions=70007, lens=[70000], max_len=70000),
    "bf16 of 4 bits": dict(kind="bf16", bits=4, batch=1, tokens=1, heads=4, kv_heads=2, dim=128, positions=90007, lens=[90000], max_len=90000),
    "f16 of 8 bits": dict(kind="f16", bits=8, batch=1, tokens=2, heads=2, kv_heads=1, dim=128, positions=200007, lens=[200000], max_len=200000),
}


@pytest.mark.parametrize("name", sorted(SPLITS))
def test_more_splits_than_lanes(ctx, hip, name):  # noqa: F811
    """Lengths that all of the splits have a part of, that end shortly behind the 64th, at it, before it, and behind all that is cached."""
    c = Case(hip, **SPLITS[name]).run(ctx)
    c.check()
    longest = SPLITS[name]["lens"][0]
    for length in (longest * 3 // 4, longest * 7 // 10, longest * 2 // 3, longest // 2, 40, 0):
        c.lens = np.array([length], np.int32)
        c.dlens.set(c.lens)
        c.run(ctx).check()


# name: (arguments, columns of a tile) whatever the cached length
HEADS = {
    "32, f32": (dict(kind="f32", bits=8, batch=1, tokens=300, heads=64, kv_heads=4, dim=64), 32),
    "32, f16": (dict(kind="f16", bits=8, batch=1, tokens=300, heads=64, kv_heads=4, dim=128), 32),
    "128, dim 64": (dict(kind="bf16", bits=8, batch=1, tokens=256, heads=1024, kv_heads=1, dim=64), 128),
    "128, dim 128": (dict(kind="bf16", bits=8, batch=1, tokens=256, heads=1024, kv_heads=1, dim=128), 128),
}


def behind(name, n):
    """The tokens behind n cached positions."""
    c = HEADS[name][0]
    return {**c, "positions": n + c["tokens"], "lens": [n]}


def check_rows(q, out, lse, cache, lens, tokens, scale, kind):
    """check_attention of these tokens, of the first head, the last and one between: each as a sequence and a head of its own."""
    heads, one = q.shape[2], np.array([1], np.uint32)
    for b in range(q.shape[0]):
        for h in (0, heads // 2 + 1, heads - 1):
            g = h * cache.k.shape[2] // heads
            part = Cache.__new__(Cache)
            part.bits, part.k, part.v = cache.bits, cache.k[b:b + 1, :, g:g + 1], cache.v[b:b + 1, :, g:g + 1]
            part.kscale, part.vscale = (a[b:b + 1] if cache.bits == 8 else a[b:b + 1, :, g:g + 1] for a in (cache.kscale, cache.vscale))
            for i in tokens[b] if isinstance(tokens[0], tuple) else tokens:
                at = (slice(b, b + 1), slice(i, i + 1), slice(h, h + 1))
                check_attention(out[at], lse[at], q[at], part, np.array([lens[b] + i], np.uint32), one, 0, 0, scale, kind)


def check(c, tokens):
    check_rows(c.q, c.out.get(), c.lse.get(), c.cache, c.lens, tokens, c.scale, c.kind)


@pytest.mark.parametrize("name", sorted(HEADS))
def test_many_small_weights_beside_a_large_one(ctx, hip, name):  # noqa: F811
    """4000 weights of 2^-26 of the largest, whose values are 2^10 times as large: they make 1/16 of the result each way."""
    c = behind(name, 4000)
    cache = Cache(np.random.default_rng(0), 8, 1, c["positions"], c["kv_heads"], c["dim"])
    cache.k[:], cache.v[:] = 0, np.random.default_rng(1).integers(60, 128, cache.v.shape)
    cache.k[0, 7, :, 0], cache.kscale[:], cache.vscale[:] = 64, 1 / 64, 1.0
    cache.vscale[0, 7] = 2.0 ** -10
    q = np.zeros((1, c["tokens"], c["heads"], c["dim"]))
    q[..., 0] = 18.0      # (e^18 = 2^26)
    check(Case(hip, **c, q=q, cache=cache, scale=1.0).run(ctx), [0, c["tokens"] - 1])


@pytest.mark.parametrize("name", sorted(HEADS))
def test_the_largest_score_comes_late(ctx, hip, name):  # noqa: F811
    """Scores that rise by 7 to 9 in base 2 from chunk to chunk or every second one, about as much as the reference waits for, and values whose
    scales fall as fast: every chunk counts.  (By 120 in all, from 2^50: the results are far inside f32.)"""
    c = behind(name, 640)
    cache = Cache(np.random.default_rng(0), 8, 1, c["positions"], c["kv_heads"], c["dim"])
    chunk = np.arange(c["positions"]) // 32
    rise = np.cumsum(np.random.default_rng(2).uniform(7, 9, chunk[-1] + 1) * (np.arange(chunk[-1] + 1) % 2))
    cache.k[:], cache.k[..., 0] = 0, 64
    cache.kscale[0] = (rise / 64 * np.log(2))[chunk]
    cache.vscale[0] = (2.0 ** (50 - np.round(rise)))[chunk]
    q = np.zeros((1, c["tokens"], c["heads"], c["dim"]))
    q[..., 0] = 1.0
    check(Case(hip, **c, q=q, cache=cache, scale=1.0).run(ctx), [0, 31, 32, c["tokens"] - 1])


@pytest.mark.parametrize("name", sorted(HEADS))
def test_value_scales_far_apart(ctx, hip, name):  # noqa: F811
    c = behind(name, 2000)
    cache = Cache(np.random.default_rng(0), 8, 1, c["positions"], c["kv_heads"], c["dim"])
    top = 6 if c["kind"] == "f16" else 60      # (results are the type's numbers)
    cache.vscale[:] = 2.0 ** np.random.default_rng(1).integers(-90, top, cache.vscale.shape)
    check(Case(hip, **c, cache=cache).run(ctx), [0, c["tokens"] - 1])


@pytest.mark.parametrize("name", WIDE)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite_stay_alone(ctx, hip, name, bad):  # noqa: F811
    c = KERNELS[name][0]
    q = np.random.default_rng(2).standard_normal((1, c["tokens"], c["heads"], c["dim"]))
    cache = Cache(np.random.default_rng(0), c["bits"], 1, c["positions"], c["kv_heads"], c["dim"])
    clean = Case(hip, **c, q=q, cache=cache).run(ctx)
    rows = [(0, 0), (1, 3), (c["tokens"] // 2, 1), (c["tokens"] - 1, c["heads"] - 1)]
    for token, head in rows:
        q[0, token, head, 7] = bad
    got = Case(hip, **c, q=q, cache=cache).run(ctx)
    out, lse, want, wlse = decode(got.out.get(), c["kind"]), got.lse.get(), decode(clean.out.get(), c["kind"]), clean.lse.get()
    for token, head in rows:
        assert np.isnan(out[0, token, head]).all() and np.isnan(lse[0, token, head])
        out[0, token, head], lse[0, token, head] = want[0, token, head], wlse[0, token, head]
    assert (out == want).all() and (lse == wlse).all()


@pytest.mark.parametrize("name", WIDE)
def test_captured_with_eager_calls_between_the_replays(ctx, hip, name):  # noqa: F811
    """Replays of one graph, its lengths in device memory, give the bits of eager calls with the same lengths."""
    full = KERNELS[name][0]
    c = Case(hip, **full, counts=[full["tokens"]], max_len=full["lens"][0])
    stream, ws = hip.stream(), hip.workspace(c.need(ctx))
    ready = hip.capture(stream, lambda: c.run(ctx, stream=stream, wait=False, workspace=ws))
    for length, count in ((full["lens"][0], full["tokens"]), (33, 100), (full["lens"][0] // 2, 1), (0, full["tokens"]), (full["lens"][0], 0)):
        c.dlens.set(np.array([length], np.int32))
        c.dcounts.set(np.array([count], np.int32))
        c.out.set(np.full(c.q.shape, c.before))
        hip.sync()
        hip.hipGraphLaunch(ready, ctypes.c_void_p(stream))
        hip.hipStreamSynchronize(ctypes.c_void_p(stream))
        got, lse = c.out.get(), c.lse.get()
        assert (got[0, count:] == c.before).all()
        c.out.set(np.full(c.q.shape, c.before))
        c.run(ctx)
        assert (c.out.get() == got).all() and (c.lse.get()[0, :count] == lse[0, :count]).all()
        assert count == 0 or not (got[0, :count] == c.before).all()


@pytest.mark.parametrize("name", WIDE)
def test_two_at_once(ctx, hip, name):  # noqa: F811
    """Two threads, a stream and a workspace each, calls queued one behind the other: the bits of each alone."""
    cases = [Case(hip, **KERNELS[name][0], seed=seed) for seed in (1, 2)]
    alone = [c.run(ctx).out.get() for c in cases]
    streams, spaces = [hip.stream() for _ in cases], [hip.workspace(c.need(ctx)) for c in cases]
    for c in cases:
        c.out.set(np.full(c.q.shape, c.before))
    hip.sync()

    def work(c, stream, ws):
        for _ in range(5):
            c.run(ctx, stream=stream, wait=False, workspace=ws)
    threads = [threading.Thread(target=work, args=a) for a in zip(cases, streams, spaces)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    hip.sync()
    assert all((c.out.get() == want).all() for c, want in zip(cases, alone))


# name: (arguments, columns, bytes from one row of the cache to the next: its last rows are past 2^32)
FAR = {
    "32, f16 of 8 bits": (dict(kind="f16", bits=8, batch=1, tokens=300, heads=16, kv_heads=1, dim=64, lens=[100]), 32, 12 << 20),
    "32, bf16 of 4 bits": (dict(kind="bf16", bits=4, batch=2, tokens=200, heads=16, kv_heads=1, dim=128, lens=[200, 90], counts=[200, 150]), 32, 12 << 20),
    "128": (dict(kind="bf16", bits=8, batch=1, tokens=450, heads=1024, kv_heads=1, dim=64, lens=[3]), 128, 12 << 20),
}


@pytest.mark.parametrize("name", sorted(FAR))
def test_cache_past_4_gib(ctx, name):  # noqa: F811
    c, _, pitch = FAR[name]
    hip = Hip()      # (released at once: other tests' arrays are as large)
    try:
        rng, kind, bits, batch, tokens, heads, dim = np.random.default_rng(1), *(c[k] for k in ("kind", "bits", "batch", "tokens", "heads", "dim"))
        positions, lens = max(c["lens"]) + tokens, np.array(c["lens"], np.int32)
        counts = np.array(c.get("counts", [tokens] * batch), np.int32)
        assert positions * pitch > 1 << 32
        host = Cache(rng, bits, batch, positions, c["kv_heads"], dim)
        cache = [Far(hip, a, pitch).view for a in (host.k, host.v)]
        scales = [Far(hip, a, pitch).view if bits == 4 else hip.put(a) for a in (host.kscale, host.vscale)]
        q, dtype = encode(rng.standard_normal((batch, tokens, heads, dim)), kind)
        out, lse = hip.put(np.zeros_like(q), dtype), hip.put(np.zeros(q.shape[:3], np.float32))
        ws = hip.workspace(ctx.cache_attention_workspace(q.shape, host.k.shape, bits=bits, max_len=max(c["lens"])))
        ctx.cache_attention(hip.put(q, dtype), *cache, *scales, hip.put(lens), out, counts=hip.put(counts), lse=lse, max_len=max(c["lens"]), workspace=ws)
        check_rows(q, out.get(), lse.get(), host, lens, [(0, 170 if n > 170 else 1, n - 1) for n in counts], dim ** -0.5, kind)
    finally:
        hip.sync()
        hip.release()
