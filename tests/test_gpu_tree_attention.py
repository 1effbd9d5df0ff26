"""Tree attention over an INT8 cache (qxg_tree_attention) against its formula in 64 bits.

Tolerances.  A score is a sum of dim products q * code that f32 accumulates; q enters with 22 bits (f32) or
whole (16 bits), and up to 24 accumulations round by 2^-24 of sums no larger than S = scale * kscale *
sum |q| |code|: at most S * (2^-22 + 24 * 2^-24) < S * 2^-19 off.  Scaling and the exponent add 4 roundings
of the score's own size, |s| * 2^-22.  Errors of the scores by d move a softmax average of values no
larger than vmax by at most 2 d vmax; the second product, the joins and the division add less than
2^-18 vmax (f32), and for BF16 values the weights' rounding to 11 bits half a step each, 2^-11 vmax in
all (allowed to F16 too); the result's own rounding is half a step of its type.
"""
import numpy as np
import pytest

import qxg
from devmem import HALF_STEP, Hip, decode, encode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = qxg.Context(0)
    yield c
    c.close()


@pytest.fixture()
def hip(ctx):
    h = Hip()
    yield h
    h.sync()
    h.release()


def bits(flags):
    n = flags.shape[-1]
    f = np.zeros((*flags.shape[:-1], -(-n // 32) * 32), np.uint64)
    f[..., :n] = flags
    return (f.reshape(*f.shape[:-1], -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def tree_mask(rng, batch, nodes):
    """Each node sees itself and its ancestors; parents are earlier nodes or none."""
    sees = np.zeros((batch, nodes, nodes), bool)
    for b in range(batch):
        for i in range(nodes):
            p = rng.integers(-1, i)
            sees[b, i, i] = True
            if p >= 0:
                sees[b, i] |= sees[b, p]
    return sees


class Case:
    def __init__(self, kind="f32", batch=1, nodes=1, heads=32, kv_heads=4, dim=128, lens=(5,), counts=None, sees="tree", spare=3, seed=0,
                 qscale=2.0):
        rng = np.random.default_rng([seed, batch, nodes, heads, dim, *lens])
        self.kind, self.batch, self.nodes, self.heads, self.kv_heads, self.dim = kind, batch, nodes, heads, kv_heads, dim
        self.lens = np.array(lens, np.int32)
        self.counts = np.full(batch, nodes, np.int32) if counts is None else np.array(counts, np.int32)
        self.given_counts = counts is not None
        self.positions = P = int(max(lens)) + nodes + spare
        self.q, self.qtype = encode(rng.standard_normal((batch, nodes, heads, dim)) * qscale, kind)
        self.k = np.clip(np.rint(rng.standard_normal((batch, P, kv_heads, dim)) * 36), -127, 127).astype(np.int8)
        self.v = np.clip(np.rint(rng.standard_normal((batch, P, kv_heads, dim)) * 36), -127, 127).astype(np.int8)
        self.ks = (rng.uniform(3, 4.5, (batch, P)) / 127).astype(np.float32)
        self.vs = (rng.uniform(3, 4.5, (batch, P)) / 127).astype(np.float32)
        # what stands behind the last node must not matter
        for b in range(batch):
            end = int(self.lens[b] + self.counts[b])
            self.ks[b, end:], self.vs[b, end:] = np.nan, np.inf
        self.chain = isinstance(sees, str) and sees == "chain"
        self.sees = np.tril(np.ones((batch, nodes, nodes), bool)) if self.chain else tree_mask(rng, batch, nodes) if isinstance(sees, str) else sees
        self.account = rng.uniform(0, 4, (batch, P)).astype(np.float32)
        self.decay = 0.75
        self.scale = 1 / np.sqrt(dim)

    def expect(self):
        """out, lse, account in 64 bits, and how far each may be off."""
        q = decode(self.q, self.kind)
        B, n, H, D = q.shape
        out, lse, acc = np.zeros(q.shape), np.full((B, n, H), -np.inf), self.account.astype(np.float64)
        t_out, t_lse, t_acc = np.zeros(q.shape), np.zeros((B, n, H)), np.zeros(acc.shape)
        for b in range(B):
            L, c = int(self.lens[b]), int(self.counts[b])
            T = L + c
            vis = np.concatenate([np.ones((c, L), bool), self.sees[b, :c, :c]], 1)
            acc[b, :T] *= self.decay
            t_acc[b, :T] = np.abs(acc[b, :T]) * 2.0 ** -22
            for h in range(H):
                g = h // (H // self.kv_heads)
                ks, vs = self.ks[b, :T].astype(np.float64), self.vs[b, :T].astype(np.float64)
                k, v = self.k[b, :T, g] * ks[:, None], self.v[b, :T, g] * vs[:, None]
                for i in range(c):
                    w = vis[i]
                    if not w.any():
                        continue
                    s = k[w] @ q[b, i, h] * self.scale
                    big = (np.abs(k[w]) @ np.abs(q[b, i, h]) * self.scale).max()
                    d = big * 2.0 ** -19 + np.abs(s).max() * 2.0 ** -22
                    e = np.exp(s - s.max())
                    out[b, i, h] = e @ v[w] / e.sum()
                    lse[b, i, h] = s.max() + np.log(e.sum())
                    vmax = np.abs(v[w]).max()
                    t_out[b, i, h] = vmax * (2 * d + (2.0 ** -18 if self.kind == "f32" else 2.0 ** -11)) + np.abs(out[b, i, h]) * HALF_STEP[self.kind]
                    t_lse[b, i, h] = d + 2.0 ** -18 + abs(lse[b, i, h]) * 2.0 ** -22
                    p = e / e.sum()
                    at = np.flatnonzero(w)
                    acc[b, at] += p
                    t_acc[b, at] += p * (2 * d + 2.0 ** -17)
        return out, lse, acc, t_out, t_lse, t_acc


def run(ctx, hip, case, account=True, max_len=None, wait=True, stream=0, strided=False):
    B, n, H, D = case.q.shape
    P, Hk = case.positions, case.kv_heads
    junk = encode(np.full(case.q.shape, 7.0), case.kind)[0]
    q, k, v = hip.put(case.q, case.qtype), hip.put(case.k), hip.put(case.v)
    ks, vs = hip.put(case.ks), hip.put(case.vs)
    out, lse, acc = hip.put(junk, case.qtype), hip.put(np.full((B, n, H), 7.0, np.float32)), hip.put(case.account)
    mask = None if case.chain else hip.put(bits(case.sees))
    counts = hip.put(case.counts) if case.given_counts else None
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, max_len=max_len, account=account))
    lens = hip.put(case.lens)

    def call(wait=wait):
        ctx.tree_attention(q, k, v, ks, vs, lens, out, mask=mask, counts=counts, lse=lse, account=acc if account else None,
                           decay=case.decay, max_len=max_len, workspace=ws, stream=stream, wait=wait)
    call()
    return call, out, lse, acc


def check(case, out, lse, acc, account=True):
    w_out, w_lse, w_acc, t_out, t_lse, t_acc = case.expect()
    got = decode(out.get(), case.kind)
    g_lse, g_acc = lse.get().astype(np.float64), acc.get().astype(np.float64)
    for b in range(case.batch):
        c, end = int(case.counts[b]), int(case.lens[b] + case.counts[b])
        assert (got[b, c:] == 7).all() and (g_lse[b, c:] == 7).all()      # rows behind the last node
        err = np.abs(got[b, :c] - w_out[b, :c])
        assert (err <= t_out[b, :c]).all(), (b, err.max(), np.argwhere(~(err <= t_out[b, :c]))[:4])
        empty = np.isneginf(w_lse[b, :c])
        assert np.array_equal(np.isneginf(g_lse[b, :c]), empty) and not got[b, :c][empty].any()
        assert (np.abs(g_lse[b, :c][~empty] - w_lse[b, :c][~empty]) <= t_lse[b, :c][~empty]).all()
        if account:
            err = np.abs(g_acc[b, :end] - w_acc[b, :end])
            assert (err <= t_acc[b, :end]).all(), (b, err.max())
            assert np.array_equal(g_acc[b, end:], case.account[b, end:].astype(np.float64))


CASES = {
    "one_token": dict(lens=(5,)),
    "one_token_one_position": dict(lens=(0,), sees="chain"),
    "one_token_chain_of_32": dict(lens=(31,), sees="chain"),
    "no_cache_tree": dict(nodes=9, lens=(0,)),
    "empty_rows": dict(nodes=5, lens=(0,), sees=np.zeros((1, 5, 5), bool)),
    "some_empty_rows": dict(batch=2, nodes=3, lens=(0, 40), sees=np.eye(3, dtype=bool)[None].repeat(2, 0) & (np.arange(3) != 1)),
    "edges_of_a_chunk": dict(batch=4, nodes=3, heads=8, kv_heads=2, lens=(29, 31, 32, 33)),
    "two_mask_words": dict(nodes=33, heads=8, kv_heads=4, lens=(50,)),
    "three_mask_words_no_offset": dict(nodes=70, heads=4, kv_heads=4, dim=64, lens=(64,)),
    "mask_across_chunks": dict(nodes=100, heads=2, kv_heads=1, dim=64, lens=(17,)),
    "sees_later_nodes": dict(nodes=40, heads=4, kv_heads=2, lens=(7,), sees=np.ones((1, 40, 40), bool)),
    "counts": dict(batch=4, nodes=6, heads=14, kv_heads=2, dim=64, lens=(100, 3, 0, 77), counts=(6, 1, 3, 0)),
    "counts_zero_no_cache": dict(batch=2, nodes=2, heads=4, kv_heads=4, lens=(0, 9), counts=(0, 2)),
    "count_whole_tiles_behind": dict(batch=2, nodes=64, heads=32, kv_heads=4, lens=(20, 33), counts=(64, 3)),
    "group_of_1": dict(nodes=40, heads=4, kv_heads=4, lens=(200,)),
    "group_of_3": dict(nodes=13, heads=6, kv_heads=2, lens=(90,)),
    "group_of_40": dict(nodes=3, heads=40, kv_heads=1, dim=64, lens=(70,)),
    "splits": dict(nodes=5, heads=16, kv_heads=2, lens=(3000,)),
    "splits_ragged": dict(batch=3, nodes=4, heads=8, kv_heads=4, dim=64, lens=(2500, 1, 600), counts=(4, 4, 2)),
    "many_columns": dict(nodes=64, heads=32, kv_heads=4, lens=(777,)),
    "many_columns_ragged": dict(batch=2, nodes=37, heads=16, kv_heads=2, dim=64, lens=(410, 95), counts=(37, 20)),
    "many_sequences": dict(batch=33, nodes=2, heads=8, kv_heads=2, dim=64, lens=tuple(range(0, 990, 30)), counts=(2, 1, 0) * 11),
    "sequences_beyond_64": dict(batch=70, nodes=1, heads=4, kv_heads=1, lens=tuple(range(0, 910, 13))),
    "many_columns_beyond_64": dict(batch=66, nodes=20, heads=8, kv_heads=1, dim=64, lens=tuple(range(200, 464, 4)), counts=(20, 3, 0) * 22),
    "scores_kept_of_8_columns": dict(batch=3, nodes=2, heads=8, kv_heads=2, lens=(700, 31, 0), counts=(1, 2, 2)),
    "long_account": dict(nodes=9, heads=2, kv_heads=1, dim=64, lens=(33000,)),
    "long_account_of_two_sequences": dict(batch=2, nodes=5, heads=4, kv_heads=1, lens=(16500, 17000), counts=(5, 2)),
    "empty_rows_of_many_columns": dict(batch=2, nodes=12, lens=(0, 3), sees=np.zeros((2, 12, 12), bool)),
    "sharp": dict(nodes=7, heads=8, kv_heads=2, lens=(300,), qscale=60.0),
    "flat": dict(nodes=7, heads=8, kv_heads=2, lens=(300,), qscale=1e-30),
}


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_formula(ctx, hip, name, kind):
    spec = dict(CASES[name])
    if kind == "f16" and name == "flat":
        spec["qscale"] = 1e-3   # (1e-30 is 0 in F16)
    case = Case(kind=kind, **spec)
    _, out, lse, acc = run(ctx, hip, case)
    check(case, out, lse, acc)


# Cases of more than two tiles of columns, as a launch for many positions takes them (four tiles a workgroup)
LONG = 1 << 20
MANY_COLUMNS = sorted(n for n, c in CASES.items() if c.get("nodes", 1) * c.get("heads", 32) // c.get("kv_heads", 4) > 64)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", MANY_COLUMNS)
def test_formula_many_columns(ctx, hip, name, kind):
    case = Case(kind=kind, **CASES[name])
    _, out, lse, acc = run(ctx, hip, case, max_len=LONG)
    check(case, out, lse, acc)


@pytest.mark.parametrize("max_len", [0, 1, 300, 1 << 20])
def test_max_len_shapes_the_launch_only(ctx, hip, max_len):
    case = Case(nodes=5, heads=8, kv_heads=2, lens=(1000,))
    _, out, lse, acc = run(ctx, hip, case, max_len=max_len)
    check(case, out, lse, acc)


def test_without_account_and_lse(ctx, hip):
    case = Case(nodes=4, heads=8, kv_heads=2, lens=(700,), kind="bf16")
    _, out, lse, acc = run(ctx, hip, case, account=False)
    check(case, out, lse, acc, account=False)
    assert np.array_equal(acc.get(), case.account)
    q, k, v, ks, vs = hip.put(case.q, case.qtype), hip.put(case.k), hip.put(case.v), hip.put(case.ks), hip.put(case.vs)
    again, acc2 = hip.put(np.zeros_like(case.q), case.qtype), hip.put(case.account)
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, account=True))
    ctx.tree_attention(q, k, v, ks, vs, hip.put(case.lens), again, mask=hip.put(bits(case.sees)), account=acc2, decay=case.decay, workspace=ws)
    assert np.array_equal(again.get(), out.get())     # the account needs no lse of the caller's
    w_acc, t_acc = case.expect()[2], case.expect()[5]
    assert (np.abs(acc2.get() - w_acc) <= t_acc)[0, :704].all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("max_len", [None, LONG])
def test_equal_calls_give_equal_bits(ctx, hip, kind, max_len):
    case = Case(kind=kind, batch=2, nodes=20, heads=16, kv_heads=2, lens=(1500, 333))
    got = []
    for _ in range(3):
        _, out, lse, acc = run(ctx, hip, case, max_len=max_len)
        got.append((out.get().tobytes(), lse.get().tobytes(), acc.get().tobytes()))
    assert got[0] == got[1] == got[2]


@pytest.mark.parametrize("nodes,max_len", [(4, None), (24, LONG)])
def test_not_finite_q_stays_in_its_row(ctx, hip, nodes, max_len):
    case = Case(nodes=nodes, heads=8, kv_heads=2, lens=(100,), sees="chain")
    case.q[0, 1, 3, 5] = np.nan
    case.q[0, 2, 6, 0] = np.inf
    _, out, lse, _ = run(ctx, hip, case, account=False, max_len=max_len)
    got, g_lse = out.get(), lse.get()
    bad = np.zeros((nodes, 8), bool)
    bad[1, 3] = bad[2, 6] = True
    assert np.isnan(got[0][bad]).all() and np.isnan(g_lse[0][bad]).all()
    case.q[0, 1, 3], case.q[0, 2, 6] = 1, 1
    w, l, _, t, tl, _ = case.expect()
    assert (np.abs(got - w) <= t)[0][~bad].all() and (np.abs(g_lse - l) <= tl)[0][~bad].all()


@pytest.mark.parametrize("nodes,max_len", [(6, None), (30, LONG)])
def test_masked_nodes_with_bad_scales(ctx, hip, nodes, max_len):
    """A node whose scales are not finite reaches only the nodes that see it."""
    case = Case(nodes=nodes, heads=8, kv_heads=2, lens=(45,), sees=np.eye(nodes, dtype=bool)[None])
    w, l, _, t, tl, _ = case.expect()
    case.ks[0, 45 + 2], case.vs[0, 45 + 4] = np.inf, np.nan
    _, out, lse, _ = run(ctx, hip, case, account=False, max_len=max_len)
    ok = [i for i in range(nodes) if i not in (2, 4)]
    assert (np.abs(out.get() - w) <= t)[0, ok].all() and (np.abs(lse.get() - l) <= tl)[0, ok].all()
    assert np.isnan(out.get()[0, 4]).all()


def test_lens_past_the_cache_are_clamped(ctx, hip):
    case = Case(nodes=3, heads=4, kv_heads=2, lens=(60,), spare=0)
    call, out, lse, acc = run(ctx, hip, case)
    check(case, out, lse, acc)
    want = out.get()
    case.lens[:] = -1          # 2^32 - 1: clamped to positions - count, the 60 of the call before
    _, out2, _, _ = run(ctx, hip, case)
    assert np.array_equal(out2.get(), want)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("nodes,max_len", [(3, None), (40, LONG)])
def test_strides(ctx, hip, kind, nodes, max_len):
    """q and out inside wider rows, one layer of a [layers][positions] cache, accounts with a stride."""
    case = Case(kind=kind, batch=2, nodes=nodes, heads=8, kv_heads=2, dim=64, lens=(70, 41))
    B, n, H, D = case.q.shape
    P, Hk = case.positions, case.kv_heads
    wide = np.zeros((B, n, 3, H * D), case.q.dtype)
    wide[:, :, 1] = case.q.reshape(B, n, H * D)
    q_all, o_all = hip.put(wide, case.qtype), hip.put(np.zeros_like(wide), case.qtype)
    st = (n * 3 * H * D, 3 * H * D, D, 1)
    q, out = (a.view(H * D, (B, n, H, D), st) for a in (q_all, o_all))
    row = Hk * D + 32
    kv = [np.full((B, 4, P, row), 99, np.int8) for _ in range(2)]
    for a, x in zip(kv, (case.k, case.v)):
        a[:, 2, :, :Hk * D] = x.reshape(B, P, Hk * D)
    k, v = (hip.put(a).view(2 * P * row, (B, P, Hk, D), (4 * P * row, row, D, 1)) for a in kv)
    sc = [np.full((B, 4, P), np.nan, np.float32) for _ in range(2)]
    for a, x in zip(sc, (case.ks, case.vs)):
        a[:, 2] = x
    ks, vs = (hip.put(a).view(2 * P, (B, P), (4 * P, 1)) for a in sc)
    acc_all = np.zeros((B, P + 11), np.float32)
    acc_all[:, :P] = case.account
    acc_dev = hip.put(acc_all)
    lse = hip.put(np.zeros((B, n, H), np.float32))
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, max_len=max_len, account=True))
    ctx.tree_attention(q, k, v, ks, vs, hip.put(case.lens), out, mask=hip.put(bits(case.sees)), lse=lse,
                       account=acc_dev.view(0, (B, P), (P + 11, 1)), decay=case.decay, max_len=max_len, workspace=ws)
    w_out, w_lse, w_acc, t_out, t_lse, t_acc = case.expect()
    got = o_all.get()
    assert not got[:, :, 0].any() and not got[:, :, 2].any()
    assert (np.abs(decode(got[:, :, 1], kind).reshape(B, n, H, D) - w_out) <= t_out).all()
    assert (np.abs(lse.get() - w_lse) <= t_lse).all()
    g = acc_dev.get()
    assert (np.abs(g[:, :P] - w_acc) <= t_acc).all() and not g[:, P:].any()


@pytest.mark.parametrize("nodes,max_len", [(2, None), (40, LONG)])
def test_cache_past_4_gib(ctx, hip, nodes, max_len):
    """Rows 64 KiB apart: the last ones lie more than 2^32 bytes behind the first."""
    import ctypes
    case = Case(kind="f16", nodes=nodes, heads=2, kv_heads=1, dim=64, lens=(66000,), spare=0)
    P, pitch = case.positions, 1 << 16
    views = []
    for a in (case.k, case.v):
        ptr = hip.malloc(P * pitch)
        rows = np.ascontiguousarray(a.reshape(P, 64))
        hip.hipMemcpy2D(ctypes.c_void_p(ptr), ctypes.c_size_t(pitch), rows.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(64),
                        ctypes.c_size_t(64), ctypes.c_size_t(P), 1)
        base = hip.put(np.zeros(16, np.int8))
        view = base.view(0, (1, P, 1, 64), (0, pitch, 64, 1))
        view.ptr = ptr
        views.append(view)
    acc = hip.put(case.account)
    out, lse = hip.put(np.zeros_like(case.q), case.qtype), hip.put(np.zeros((1, nodes, 2), np.float32))
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, max_len=max_len, account=True))
    ctx.tree_attention(hip.put(case.q, case.qtype), *views, hip.put(case.ks), hip.put(case.vs), hip.put(case.lens), out,
                       mask=hip.put(bits(case.sees)), lse=lse, account=acc, decay=case.decay, max_len=max_len, workspace=ws)
    check(case, out, lse, acc)


@pytest.mark.parametrize("nodes,max_len", [(8, None), (24, LONG)])
def test_captured_and_replayed(ctx, hip, nodes, max_len):
    """One graph, replayed with other lengths, masks and cache contents, other work between."""
    import ctypes
    case = Case(batch=2, nodes=nodes, heads=8, kv_heads=2, lens=(900, 200))
    s = hip.stream()
    B, n, H, D = case.q.shape
    q, k, v, ks, vs = hip.put(case.q, case.qtype), hip.put(case.k), hip.put(case.v), hip.put(case.ks), hip.put(case.vs)
    out, lse, acc = hip.put(np.zeros_like(case.q)), hip.put(np.zeros((B, n, H), np.float32)), hip.put(case.account)
    mask, lens = hip.put(bits(case.sees)), hip.put(case.lens)
    ws = hip.workspace(ctx.tree_attention_workspace(case.q.shape, case.k.shape, max_len=max_len, account=True))
    graph = hip.capture(s, lambda: ctx.tree_attention(q, k, v, ks, vs, lens, out, mask=mask, lse=lse, account=acc, decay=case.decay,
                                                      max_len=max_len, workspace=ws, stream=s, wait=False))
    for step, ln in enumerate([(900, 200), (17, 900), (0, 3), (640, 641)]):
        now = Case(batch=2, nodes=nodes, heads=8, kv_heads=2, lens=(900, 200), seed=step)
        now.ks, now.vs = np.nan_to_num(now.ks, nan=0.03), np.nan_to_num(now.vs, posinf=0.03)
        now.lens = np.array(ln, np.int32)
        for d, a in ((q, now.q), (k, now.k), (v, now.v), (ks, now.ks), (vs, now.vs), (acc, now.account), (mask, bits(now.sees)), (lens, now.lens)):
            d.set(a)
        hip.hipGraphLaunch(graph, ctypes.c_void_p(s))
        hip.hipStreamSynchronize(ctypes.c_void_p(s))
        check(now, out, lse, acc)
        _, o2, l2, a2 = run(ctx, hip, now, max_len=max_len)      # the eager call, between the replays
        assert np.array_equal(o2.get(), out.get()) and np.array_equal(a2.get(), acc.get())


def test_two_streams_at_once(ctx, hip):
    cases = [Case(nodes=6, heads=32, kv_heads=4, lens=(2000 + i,), seed=i) for i in range(2)]
    streams = [hip.stream() for _ in cases]
    runs = [run(ctx, hip, c, wait=False, stream=s) for c, s in zip(cases, streams)]
    hip.sync()
    for c, (_, out, lse, acc) in zip(cases, runs):
        check(c, out, lse, acc)
