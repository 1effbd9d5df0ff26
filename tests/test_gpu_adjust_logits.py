"""Penalties, biases, temperature and grammar mask on logits with the best tokens (qxg_adjust_logits).

Each step is one f32 operation, done here by numpy in the same order: the adjusted logits (rounded once to
their type), the picks and their logits have to be equal.  lse sums exponentials in f32: with the
maximum m, at most vocab terms of at most 1, whose exponentials and sums (16 a thread, then a tree) are off
by less than 2^-19 in all, plus the rounding of the result, |lse| * 2^-23."""
import ctypes

import numpy as np
import pytest

import qxg
from devmem import Hip, decode, encode

pytestmark = pytest.mark.gpu
f32 = np.float32


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


class Case:
    def __init__(self, kind="f32", rows=2, vocab=1000, slots=0, biases=0, masks=0, top_n=8, penalties=True, temperature=True, lens=True, seed=0):
        rng = self.rng = np.random.default_rng([seed, rows, vocab, slots, biases, masks])
        self.kind, self.rows, self.vocab, self.top_n = kind, rows, vocab, top_n
        self.logits, self.dtype = encode(rng.standard_normal((rows, vocab)) * 2.5, kind)
        self.history = (vocab ** rng.random((rows, slots))).astype(np.int32).clip(0, vocab - 1) if slots else None
        self.history_lens = rng.integers(0, slots + 1, rows).astype(np.int32) if slots and lens else None
        self.prompt_lens = rng.integers(0, slots + 1, rows).astype(np.int32) if slots and lens else None
        self.penalties = np.stack([rng.uniform(1, 1.5, rows), rng.uniform(-0.5, 0.5, rows), rng.uniform(0, 1, rows)], 1).astype(f32) if penalties else None
        self.temperature = rng.uniform(0.3, 1.7, rows).astype(f32) if temperature else None
        self.bias_ids = rng.integers(0, vocab, (rows, biases)).astype(np.int32) if biases else None
        self.bias_values = rng.standard_normal((rows, biases)).astype(f32) * 3 if biases else None
        self.mask_bits = rng.random((masks, vocab)) < rng.choice([0.02, 0.5, 0.95], (masks, 1)) if masks else None
        self.mask_rows = rng.integers(-1, masks + 1, rows).astype(np.int32) if masks else None

    def expect(self):
        x = decode(self.logits, self.kind).astype(f32)
        with np.errstate(all="ignore"):
            for r in range(self.rows):
                pen = self.penalties[r] if self.penalties is not None else np.array([1, 0, 0], f32)
                if self.history is not None:
                    n = min(int(np.uint32(self.history_lens[r])), self.history.shape[1]) if self.history_lens is not None else self.history.shape[1]
                    p = int(np.uint32(self.prompt_lens[r])) if self.prompt_lens is not None else 0
                    h = self.history[r, :n].view(np.uint32).astype(np.int64)
                    seen, made = np.unique(h[h < self.vocab]), h[p:][h[p:] < self.vocab]
                    x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / pen[0], x[r, seen] * pen[0])
                    for v, c in zip(*np.unique(made, return_counts=True)):
                        x[r, v] = (x[r, v] - pen[1] * f32(c)) - pen[2]
                if self.bias_ids is not None:
                    total = {}
                    for v, b in zip(self.bias_ids[r].view(np.uint32).tolist(), self.bias_values[r]):
                        if v < self.vocab:
                            total[v] = total[v] + b if v in total else b
                    for v, b in total.items():
                        x[r, v] += b
                if self.temperature is not None:
                    x[r] /= self.temperature[r]
                if self.mask_bits is not None:
                    m = int(np.uint32(self.mask_rows[r])) if self.mask_rows is not None else r
                    if m < len(self.mask_bits):
                        x[r, ~self.mask_bits[m]] = -np.inf
        return x

    def words(self):
        if self.mask_bits is None:
            return None
        f = np.zeros((len(self.mask_bits), -(-self.vocab // 32) * 32), np.uint64)
        f[:, :self.vocab] = self.mask_bits
        f[:, self.vocab:] = 1      # bits behind the vocabulary mean nothing
        return (f.reshape(len(f), -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)

    def run(self, ctx, hip, in_place=False, stream=0, wait=True):
        put = lambda a: None if a is None else hip.put(a)  # noqa: E731
        R, n = self.rows, self.top_n
        logits = hip.put(self.logits, self.dtype)
        out = logits if in_place else hip.put(np.zeros_like(self.logits), self.dtype)
        ids, vals = (hip.put(np.zeros((R, n), np.int32)), hip.put(np.zeros((R, n), f32))) if n else (None, None)
        lse = hip.put(np.zeros(R, f32))
        ws = hip.workspace(ctx.adjust_logits_workspace(self.logits.shape, n))
        ctx.adjust_logits(logits, out, history=put(self.history), history_lens=put(self.history_lens), prompt_lens=put(self.prompt_lens),
                          penalties=put(self.penalties), temperature=put(self.temperature), bias_ids=put(self.bias_ids),
                          bias_values=put(self.bias_values), mask=put(self.words()), mask_rows=put(self.mask_rows), top_ids=ids,
                          top_logits=vals, lse=lse, workspace=ws, stream=stream, wait=wait)
        return out, ids, vals, lse

    def check(self, out, ids, vals, lse):
        x = self.expect()
        want = encode(x, self.kind)[0]
        got = out.get()
        nan = np.isnan(x)
        assert np.array_equal(got[~nan].view(np.uint8), want[~nan].view(np.uint8)), np.argwhere(~nan & (got != want))[:4]
        assert np.isnan(decode(got, self.kind)[nan]).all()
        if ids is not None:
            g_ids, g_vals = ids.get(), vals.get()
            for r in range(self.rows):
                key = np.where(nan[r], -np.inf, x[r])
                order = np.argsort(-key, kind="stable")[:self.top_n]
                order = order[key[order] > -np.inf]
                n = len(order)
                assert np.array_equal(g_ids[r, :n], order), (r, g_ids[r], order)
                assert np.array_equal(g_vals[r, :n].view(np.uint32), x[r, order].view(np.uint32))
                assert (g_ids[r, n:] == -1).all() and np.isneginf(g_vals[r, n:]).all()
        g = lse.get()
        for r in range(self.rows):
            if nan[r].any():
                assert np.isnan(g[r])
                continue
            m = x[r].max()
            if not np.isfinite(m):
                assert g[r] == m
                continue
            want = m.astype(np.float64) + np.log(np.exp(x[r].astype(np.float64) - m).sum())
            assert abs(g[r] - want) <= 2.0 ** -19 + abs(want) * 2.0 ** -23, (r, g[r], want)


SPECS = {
    "one_token_vocabulary": dict(vocab=1, slots=3, biases=2, masks=2, top_n=4),
    "31": dict(vocab=31, slots=9, biases=3, masks=1, top_n=32),
    "32": dict(vocab=32, slots=9, biases=3, masks=3, top_n=32),
    "33": dict(vocab=33, slots=40, biases=3, masks=3, top_n=1),
    "4095": dict(rows=3, vocab=4095, slots=600, biases=40, masks=2, top_n=32),
    "4096": dict(rows=3, vocab=4096, slots=600, biases=40, masks=2),
    "4097": dict(rows=3, vocab=4097, slots=600, biases=1000, masks=2, top_n=32),
    "model": dict(rows=1, vocab=151936, slots=700, biases=30, masks=1),
    "model_rows": dict(rows=9, vocab=151936, slots=3000, biases=300, masks=3, top_n=32),
    "nothing": dict(vocab=777, penalties=False, temperature=False),
    "only_history": dict(vocab=777, slots=50, temperature=False, lens=False, top_n=0),
    "only_biases": dict(vocab=777, biases=1024, penalties=False, temperature=False),
    "only_masks": dict(rows=5, vocab=777, masks=2, penalties=False, temperature=False),
    "history_longer_than_the_vocabulary": dict(vocab=50, slots=5000),
    "many_rows": dict(rows=300, vocab=500, slots=20, biases=5, masks=7, top_n=3),
}


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", sorted(SPECS))
def test_adjusted(ctx, hip, name, kind):
    c = Case(kind=kind, **SPECS[name])
    c.check(*c.run(ctx, hip))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_in_place(ctx, hip, kind):
    c = Case(kind=kind, rows=4, vocab=9001, slots=200, biases=9, masks=2, top_n=32)
    c.check(*c.run(ctx, hip, in_place=True))


def test_entries_that_are_no_token(ctx, hip):
    c = Case(rows=2, vocab=600, slots=64, biases=16, masks=2)
    c.history[:, ::3], c.bias_ids[:, ::2] = -1, 600
    c.history_lens[:], c.prompt_lens[:] = (-1, 64), (2 ** 31 - 1, 0)      # 2^32 - 1 entries: all slots
    c.check(*c.run(ctx, hip))


def test_tokens_named_often(ctx, hip):
    """A token named three times in the bias list: its biases are added in list order, then to the logit."""
    c = Case(rows=1, vocab=64, slots=40, biases=9)
    c.bias_ids[0] = [5, 9, 5, 63, 5, 9, 0, 0, 63]
    c.bias_values[0] = f32([1e8, 0.1, -1e8, 3, 0.7, 0.3, 1, 2 ** -24, -3])
    c.history[0, :30] = 9
    c.history_lens[0], c.prompt_lens[0] = 35, 4
    c.check(*c.run(ctx, hip))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_values_at_the_edge(ctx, hip, kind):
    """Infinite logits, NaN, zeros of both signs, equal logits, the lowest value; rows without a choice."""
    c = Case(kind=kind, rows=7, vocab=5000, masks=2, top_n=32, penalties=False, temperature=False)
    x = decode(c.logits, kind)
    x[0] = 1.5                                     # all equal
    x[1] = np.where(np.arange(5000) % 3 == 0, -0.0, 0.0)
    x[2, [7, 4099]], x[2, 50] = np.inf, -np.inf
    x[3, [0, 4500]] = np.nan
    x[4] = -np.inf
    x[4, [4321, 17]] = [-1, -2]                    # two choices
    x[5] = np.finfo(np.float32).min if kind == "f32" else -60000
    c.logits = encode(x, kind)[0]
    c.mask_bits[0], c.mask_bits[1] = True, False
    c.mask_rows[:] = [0, -1, 2, 0, 0, 0, 1]        # the last row: nothing is allowed
    c.check(*c.run(ctx, hip))
    c.rows, c.mask_rows = 1, np.array([-1], np.int32)   # a row of -inf alone
    c.logits = encode(np.full((1, 5000), -np.inf), kind)[0]
    c.check(*c.run(ctx, hip))


def test_infinite_logit_among_nan(ctx, hip):
    c = Case(rows=1, vocab=5000, penalties=False, temperature=False)
    c.logits[0, 3], c.logits[0, 4700] = np.inf, np.nan
    c.check(*c.run(ctx, hip))


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_strides(ctx, hip, kind):
    """Rows inside wider ones, at an odd offset."""
    c = Case(kind=kind, rows=3, vocab=4999, slots=30, biases=4, masks=3)
    wide = np.zeros((3, 6001), c.logits.dtype)
    wide[:, 1:5000] = c.logits
    a, b = hip.put(wide, c.dtype), hip.put(np.zeros((3, 5003), c.logits.dtype), c.dtype)
    hist = np.full((3, 77), -1, np.int32)
    hist[:, 5:35] = c.history
    h = hip.put(hist)
    ids, vals, lse = hip.put(np.zeros((3, 8), np.int32)), hip.put(np.zeros((3, 8), f32)), hip.put(np.zeros(3, f32))
    out = b.view(3, (3, 4999), (5003, 1))
    ctx.adjust_logits(a.view(1, (3, 4999), (6001, 1)), out, history=h.view(5, (3, 30), (77, 1)), history_lens=hip.put(c.history_lens),
                      prompt_lens=hip.put(c.prompt_lens), penalties=hip.put(c.penalties), temperature=hip.put(c.temperature),
                      bias_ids=hip.put(c.bias_ids), bias_values=hip.put(c.bias_values), mask=hip.put(c.words()), mask_rows=hip.put(c.mask_rows),
                      top_ids=ids, top_logits=vals, lse=lse, workspace=hip.workspace(ctx.adjust_logits_workspace((3, 4999), 8)))
    whole = b.get()
    out.get = lambda: whole[:, 3:5002].copy()
    c.check(out, ids, vals, lse)
    assert not whole[:, :3].any() and not whole[:, 5002:].any()


def test_one_mask_a_row(ctx, hip):
    c = Case(rows=4, vocab=3001, masks=4)
    c.mask_rows = None
    c.check(*c.run(ctx, hip))


def test_captured_and_replayed(ctx, hip):
    s = hip.stream()
    c = Case(rows=3, vocab=30000, slots=100, biases=5, masks=2)
    dev = {n: hip.put(getattr(c, n)) for n in ("logits", "history", "history_lens", "prompt_lens", "penalties", "temperature", "bias_ids",
                                               "bias_values", "mask_rows")}
    dev["mask"] = hip.put(c.words())
    out, ids, vals, lse = hip.put(np.zeros_like(c.logits)), hip.put(np.zeros((3, 8), np.int32)), hip.put(np.zeros((3, 8), f32)), hip.put(np.zeros(3, f32))
    ws = hip.workspace(ctx.adjust_logits_workspace(c.logits.shape, 8))
    graph = hip.capture(s, lambda: ctx.adjust_logits(out=out, top_ids=ids, top_logits=vals, lse=lse, workspace=ws, stream=s, wait=False, **dev))
    for step in range(4):
        now = Case(rows=3, vocab=30000, slots=100, biases=5, masks=2, seed=step)
        for n, d in dev.items():
            d.set(now.words() if n == "mask" else getattr(now, n))
        hip.hipGraphLaunch(graph, ctypes.c_void_p(s))
        hip.hipStreamSynchronize(ctypes.c_void_p(s))
        now.check(out, ids, vals, lse)
        now.check(*now.run(ctx, hip))       # the eager call, between the replays


def test_best_of_many_equal_slices(ctx, hip):
    """More keys than the join has room for reach its bound: 40 large logits in each 1024 tokens, alike everywhere."""
    rng = np.random.default_rng(5)
    V, n = 600_000, 32
    x = (rng.standard_normal((1, V)) - 20).astype(f32)
    for j in range(40):
        x[0, j::1024] = j + 1
    ids, vals, out = hip.put(np.zeros((1, n), np.int32)), hip.put(np.zeros((1, n), f32)), hip.put(np.zeros_like(x))
    ctx.adjust_logits(hip.put(x), out, top_ids=ids, top_logits=vals, workspace=hip.workspace(ctx.adjust_logits_workspace(x.shape, n)))
    assert np.array_equal(out.get(), x)
    assert np.array_equal(ids.get()[0], 39 + 1024 * np.arange(n)) and (vals.get() == 40).all()
