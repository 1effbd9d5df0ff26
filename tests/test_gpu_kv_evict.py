"""Eviction from a KV cache (qxg_kv_select, qxg_kv_compact) against numpy: whole numbers and moved bytes,
so everything has to be equal."""
import ctypes

import numpy as np
import pytest

import qxg
from devmem import Hip

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


def chosen(account, length, budget, sinks, recent):
    if length <= budget:
        return np.arange(length)
    w = np.where(np.isnan(account), -np.inf, account)
    middle = sorted(range(sinks, length - recent), key=lambda p: (-w[p], p))[:budget - sinks - recent]
    return np.array(sorted([*range(sinks), *middle, *range(length - recent, length)]))


ACCOUNTS = {
    "heavy": lambda r, n: np.exp(2 * r.standard_normal(n)),
    "equal": lambda r, n: np.full(n, 0.25),
    "zeros": lambda r, n: np.where(r.random(n) < 0.5, 0.0, -0.0),
    "few_values": lambda r, n: r.integers(0, 3, n) * 1.0,
    "nan_and_inf": lambda r, n: r.choice([np.nan, np.inf, -np.inf, 1.0, -1.0], n),
    "negative": lambda r, n: r.standard_normal(n),
    "next_to_each_other": lambda r, n: (np.float32(1).view(np.uint32) + r.integers(0, 4, n)).astype(np.uint32).view(np.float32),
}


@pytest.mark.parametrize("name", sorted(ACCOUNTS))
@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ((1, 2, 0, 3), 2, 1, 1), ((7, 6, 5, 4), 5, 0, 0), ((1023, 1024, 1025, 1026), 700, 4, 64), ((1025, 40, 900, 33), 33, 16, 17),
    ((5000, 4097, 2047, 4096), 2048, 3, 1), ((2050, 4099, 2048, 64), 1, 0, 0), ((3000, 2999, 17, 2500), 2500, 0, 2500),
    ((3000, 2999, 17, 2500), 2500, 2500, 0)])
def test_select(ctx, hip, name, lens, budget, sinks, recent):
    rng = np.random.default_rng(budget)
    P = max(lens) + 3
    account = np.stack([ACCOUNTS[name](rng, P) for _ in lens]).astype(np.float32)
    keep, kept = hip.put(np.full((len(lens), budget), -7, np.int32)), hip.put(np.zeros(len(lens), np.int32))
    ctx.kv_select(hip.put(account), hip.put(np.array(lens, np.int32)), keep, kept, sinks=sinks, recent=recent)
    got, n = keep.get(), kept.get()
    for g, length in enumerate(lens):
        want = chosen(account[g], length, budget, sinks, recent)
        assert n[g] == len(want) and np.array_equal(got[g, :n[g]], want), g
        assert (got[g, n[g]:] == -7).all()


@pytest.mark.parametrize("length,budget,max_len", [(70000, 5000, None), (131072, 131071, None), (40000, 39000, 100), (9000, 512, 1 << 20)])
def test_select_long(ctx, hip, length, budget, max_len):
    rng = np.random.default_rng(length)
    account = np.exp(2 * rng.standard_normal((2, length))).astype(np.float32)
    account[1] = np.round(account[1])      # many equal ones
    keep, kept = hip.put(np.zeros((2, budget), np.int32)), hip.put(np.zeros(2, np.int32))
    ctx.kv_select(hip.put(account), hip.put(np.array([length, length - 1], np.int32)), keep, kept, sinks=16, recent=100, max_len=max_len)
    for g in range(2):
        w = account[g].copy()
        n = length - g
        w[:16] = w[n - 100:n] = np.inf
        want = np.sort(np.argsort(-w[:n], kind="stable")[:budget])
        assert np.array_equal(keep.get()[g], want)


@pytest.mark.parametrize("name", sorted(ACCOUNTS))
@pytest.mark.parametrize("budget", [17, 9000, 19000])
def test_select_long_values(ctx, hip, name, budget):
    """Equal ones beyond what one histogram can part, infinities, numbers next to each other."""
    account = ACCOUNTS[name](np.random.default_rng(budget), 20000).astype(np.float32)[None]
    keep, kept = hip.put(np.zeros((1, budget), np.int32)), hip.put(np.zeros(1, np.int32))
    ctx.kv_select(hip.put(account), hip.put(np.array([20000], np.int32)), keep, kept, sinks=3, recent=5)
    assert np.array_equal(keep.get()[0], chosen(account[0], 20000, budget, 3, 5))


@pytest.mark.parametrize("budget", [10, 600, 5000])
def test_select_short_lengths_of_a_long_array(ctx, hip, budget):
    rng = np.random.default_rng(budget)
    lens = np.array([0, 9, 11, 700, 4095, 4096, 4097, 17000, 20000], np.int32)
    account = np.exp(rng.standard_normal((len(lens), 20000))).astype(np.float32)
    keep, kept = hip.put(np.full((len(lens), budget), -7, np.int32)), hip.put(np.zeros(len(lens), np.int32))
    ctx.kv_select(hip.put(account), hip.put(lens), keep, kept, sinks=2, recent=7)
    got, n = keep.get(), kept.get()
    for g, length in enumerate(lens):
        want = chosen(account[g], length, budget, 2, 7)
        assert n[g] == len(want) and np.array_equal(got[g, :n[g]], want) and (got[g, n[g]:] == -7).all(), length


def test_select_lens_past_the_array_are_clamped(ctx, hip):
    account = np.arange(50, dtype=np.float32)[None]
    keep, kept = hip.put(np.zeros((1, 10), np.int32)), hip.put(np.zeros(1, np.int32))
    ctx.kv_select(hip.put(account), hip.put(np.array([-1], np.int32)), keep, kept)
    assert np.array_equal(keep.get()[0], np.arange(40, 50))


class Cache:
    def __init__(self, hip, groups, positions, row, pad=0, seed=1):
        rng = np.random.default_rng([seed, groups, positions, row])
        self.hip = hip
        self.k, self.v = (rng.integers(-128, 128, (groups, positions, row + pad), dtype=np.int8) for _ in range(2))
        self.ks, self.vs, self.account = (rng.random((groups, positions)).astype(np.float32) for _ in range(3))
        self.dev = {n: hip.put(getattr(self, n)) for n in ("k", "v", "ks", "vs", "account")}
        self.out = hip.put(np.full((groups, positions), 7.0, np.float32))
        self.row, self.shape = row, (groups, positions, row)
        st = self.dev["k"].stride()
        self.kv = [self.dev[n].view(0, self.shape, st) for n in ("k", "v")]

    def compact(self, ctx, keep, kept, first=0, account=True, **kw):
        ws = self.hip.workspace(ctx.kv_compact_workspace(self.shape, keep.shape))
        ctx.kv_compact(*self.kv, self.dev["ks"], self.dev["vs"], keep, kept, account=self.dev["account"] if account else None,
                       account_out=self.out if account else None, first=first, workspace=ws, **kw)

    def check(self, lists, first=0, account=True):
        out = np.full(self.account.shape, 7.0, np.float32)
        for name in ("k", "v", "ks", "vs"):
            want = getattr(self, name).copy()
            for g, rows in enumerate(lists):
                if name in ("k", "v"):
                    want[g, first:first + len(rows), :self.row] = getattr(self, name)[g, rows, :self.row]
                else:
                    want[g, first:first + len(rows)] = getattr(self, name)[g, rows]
                if account:
                    out[g, first:first + len(rows)] = self.account[g, rows]
            got = self.dev[name].get()
            assert np.array_equal(got, want), (name, np.argwhere(got != want)[:4])
        assert np.array_equal(self.out.get(), out)
        assert np.array_equal(self.dev["account"].get(), self.account)


@pytest.mark.parametrize("groups,positions,row,pad", [(1, 1, 16, 0), (3, 100, 48, 16), (2, 3000, 512, 0), (5, 700, 128, 32), (1, 600, 4096, 0),
                                                      (2, 257, 1040, 0), (1, 20000, 512, 0), (40, 300, 64, 0)])
@pytest.mark.parametrize("share", [0.05, 0.5, 0.97, 1.0])
def test_compact(ctx, hip, groups, positions, row, pad, share):
    rng = np.random.default_rng(positions)
    lists = [np.flatnonzero(rng.random(positions) < share) for _ in range(groups)]
    lists[0] = np.arange(positions) if share == 1.0 else lists[0]
    if groups > 1:
        lists[1] = lists[1][:0]
    slots = max(1, max(len(x) for x in lists))
    keep = np.full((groups, slots), 0x7fffffff, np.int32)
    for g, x in enumerate(lists):
        keep[g, :len(x)] = x
    c = Cache(hip, groups, positions, row, pad)
    c.compact(ctx, hip.put(keep), hip.put(np.array([len(x) for x in lists], np.int32)))
    c.check(lists)


@pytest.mark.parametrize("shift", [1, 2, 63, 64, 65, 900])
def test_compact_short_moves(ctx, hip, shift):
    """Every row moves down by the same number of places: each is read before its place is written."""
    c = Cache(hip, 2, 5000, 512)
    rows = np.arange(shift, 5000)
    c.compact(ctx, hip.put(np.stack([rows, rows]).astype(np.int32)), hip.put(np.full(2, len(rows), np.int32)))
    c.check([rows, rows])


def test_compact_accepted_path_of_a_tree(ctx, hip):
    """One list for all layers (stride 0), behind the cached positions; without accounts."""
    c = Cache(hip, 6, 90, 512)
    first, path = 70, np.array([70, 73, 74, 81], np.int32)
    keep, kept = hip.put(path), hip.put(np.array([4], np.int32))
    c.compact(ctx, keep.view(0, (6, 4), (0, 1)), kept.view(0, (6,), (0,)), first=first, account=False)
    c.check([path] * 6, first=first, account=False)


def test_compact_clamps_and_skips(ctx, hip):
    c = Cache(hip, 2, 40, 64)
    keep = np.array([[0, 3, 9, 40, 50], [5, 6, 7, 8, 9]], np.int32)   # 40 and 50 are no rows
    c.compact(ctx, hip.put(keep), hip.put(np.array([5, -1], np.int32)))   # (2^32 - 1 kept: the slots)
    c.check([[0, 3, 9], [5, 6, 7, 8, 9]])


def test_compact_unordered_list_moves_only_its_rows(ctx, hip):
    """What the moved rows become is undefined then, but nothing else changes."""
    c = Cache(hip, 1, 3000, 512)
    rows = np.random.default_rng(3).permutation(3000)[:1500].astype(np.int32)
    c.compact(ctx, hip.put(rows[None]), hip.put(np.array([1500], np.int32)), account=False)
    for name in ("k", "v", "ks", "vs"):
        assert np.array_equal(c.dev[name].get()[0, 1500:], getattr(c, name)[0, 1500:])


def test_select_and_compact_captured(ctx, hip):
    """One graph over both calls, replayed as the cache fills again."""
    s = hip.stream()
    groups, P, budget = 3, 1200, 400
    c = Cache(hip, groups, P, 512)
    lens, keep, kept = hip.put(np.zeros(groups, np.int32)), hip.put(np.zeros((groups, budget), np.int32)), hip.put(np.zeros(groups, np.int32))
    ws = hip.workspace(ctx.kv_compact_workspace(c.shape, keep.shape))

    def work():
        ctx.kv_select(c.dev["account"], lens, keep, kept, sinks=2, recent=30, stream=s, wait=False)
        ctx.kv_compact(*c.kv, c.dev["ks"], c.dev["vs"], keep, kept, account=c.dev["account"], account_out=c.out, workspace=ws, stream=s,
                       wait=False)
    graph = hip.capture(s, work)
    rng = np.random.default_rng(8)
    for step in range(4):
        for n in ("k", "v", "ks", "vs"):
            setattr(c, n, c.dev[n].get())
        c.account = rng.random((groups, P)).astype(np.float32)
        c.dev["account"].set(c.account)
        c.out.set(np.full((groups, P), 7.0, np.float32))
        now = rng.integers(300, P + 1, groups).astype(np.int32)
        lens.set(now)
        hip.hipGraphLaunch(graph, ctypes.c_void_p(s))
        hip.hipStreamSynchronize(ctypes.c_void_p(s))
        c.check([chosen(c.account[g], now[g], budget, 2, 30) for g in range(groups)])
