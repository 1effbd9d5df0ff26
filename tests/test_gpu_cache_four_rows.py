"""A cache of 4 bits whose positions have fewer than 16 scale bytes, its scale rows held 16 bytes apart: appended to, cut by kv_compact as rows of
bytes and attended over."""
import numpy as np
import pytest

from cacheref import Cache, check_attention, quantize
from devmem import decode, encode
from test_gpu_cache_attention import ctx, hip  # noqa: F401
from test_gpu_cache_together import rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (2, 64), (2, 128)])
def test_scale_rows_sixteen_bytes_apart(ctx, hip, kv_heads, dim):  # noqa: F811
    positions, n, heads, blocks = 70, 50, 4, kv_heads * dim // 32
    rng = np.random.default_rng(kv_heads + dim)
    host = Cache(rng, 4, 1, positions, kv_heads, dim)
    codes = [hip.put(a) for a in (host.k, host.v)]
    padded = [rng.integers(0, 256, (1, positions, 16)).astype(np.uint8) for _ in range(2)]
    for a, scale in zip(padded, (host.kscale, host.vscale)):
        a[..., :blocks] = scale.reshape(1, positions, blocks)
    scales = [hip.put(a) for a in padded]
    views = [s.view(0, (1, positions, kv_heads, dim // 32), (positions * 16, 16, dim // 32, 1)) for s in scales]
    x, dtype = encode(rng.standard_normal((1, n, heads + 2 * kv_heads, dim)), "bf16")
    q, k, v = np.split(x, [heads, heads + kv_heads], 2)
    dq, lens = hip.put(q, dtype), hip.put(np.array([0], np.int32))
    ctx.kv_append(dq, hip.put(k, dtype), hip.put(v, dtype), dq, *codes, *views, lens)
    for side, rows in ((0, k), (1, v)):
        host.arrays()[side][0, :n], host.arrays()[2 + side][0, :n] = quantize(decode(rows[0], "bf16").astype(np.float32), 4)
    keep = np.array([0, 1, *range(9, 33, 3), *range(40, 50)], np.int32)
    dkeep, kept = hip.put(keep[None]), hip.put(np.array([len(keep)], np.int32))
    pairs = [tuple(rows_of(a, positions) for a in pair) for pair in (codes, scales)]
    unused = [hip.put(np.ones((1, positions), np.float32)) for _ in range(2)]
    ws = hip.workspace(max(ctx.kv_compact_workspace(a.shape, (1, len(keep))) for a, _ in pairs))
    for pair in pairs:
        ctx.kv_compact(*pair, *unused, dkeep, kept, workspace=ws)
    for a in host.arrays():
        a[0, :len(keep)] = a[0, keep]
    for got, want in zip(scales, (host.kscale, host.vscale)):
        assert (got.get()[0, :len(keep), :blocks] == want[0, :len(keep)].reshape(len(keep), blocks)).all()
    last, out = hip.put(q[:, :1], dtype), hip.put(np.zeros_like(q[:, :1]), dtype)
    at = np.array([len(keep) - 1], np.int32)
    ws = hip.workspace(ctx.cache_attention_workspace(last.shape, host.k.shape, bits=4))
    ctx.cache_attention(last, *codes, *views, hip.put(at), out, workspace=ws)
    check_attention(out.get(), None, q[:, :1], host, at, np.array([1]), 0, 0, dim ** -0.5, "bf16")
