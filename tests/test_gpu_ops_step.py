"""A drafted step as INTEGRATION.md writes it, over and over: attention with the account, the accepted path's rows and
account behind the cached ones, back to the budget, lengths in device memory.  Every token's account is followed by the token, not
by its place, in 64 bits: a token starts at 0 whatever stood in its place before.

Tolerances as in test_gpu_ops_together.py: a weight p is off by at most p (2 d + 2^-17), d = 2^-19 of the sum of magnitudes
of a score plus 2^-22 of the score; each step rounds an account by 2^-22 of it."""
import numpy as np
import pytest

from test_gpu_kv_evict import chosen
from test_gpu_ops_together import ctx, hip, path_to, tree, words  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu
f32 = np.float32
H, G, D, P, BUDGET, SINKS, RECENT, DECAY = 8, 2, 64, 160, 48, 4, 6, 0.75


class Token:
    def __init__(self, rng):
        self.k, self.v = (rng.integers(-127, 128, (G, D)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = rng.uniform(0.02, 0.04, 2).astype(f32)
        self.account = self.off = 0.0


@pytest.mark.parametrize("nodes", [1, 7, 40])
def test_step(ctx, hip, nodes):  # noqa: F811
    rng = np.random.default_rng(nodes)
    text = [Token(rng) for _ in range(30)]
    host = {"k": np.zeros((1, P, G, D), np.int8), "v": np.zeros((1, P, G, D), np.int8), "ks": np.ones((1, P), f32), "vs": np.ones((1, P), f32)}

    def append(tokens, at):
        """The program writes the tokens' rows."""
        for n, d in dev.items():
            a = d.get()
            for i, t in enumerate(tokens):
                a[0, at + i] = getattr(t, n)
            d.set(a)

    dev = {n: hip.put(a) for n, a in host.items()}
    append(text, 0)
    rows = [dev[n].view(0, (1, P, G * D), (P * G * D, G * D, 1)) for n in ("k", "v")]
    account, spare = hip.put(np.zeros((1, P), f32)), hip.put(np.full((1, P), 99, f32))
    lens, keep = hip.put(np.array([len(text)], np.int32)), hip.put(np.zeros((1, BUDGET), np.int32))
    q, out = (hip.put(np.zeros((1, nodes, H, D), f32)) for _ in range(2))
    ws = hip.workspace(ctx.tree_attention_workspace(q.shape, dev["k"].shape, account=True))
    ws3 = hip.workspace(max(ctx.kv_compact_workspace(rows[0].shape, (1, n)) for n in (nodes, BUDGET)))
    for _ in range(8):
        length = len(text)
        parent, sees = tree(rng, nodes)
        drafted = [Token(rng) for _ in range(nodes)]
        append(drafted, length)
        now = (rng.standard_normal((nodes, H, D)) * 0.5).astype(f32)
        q.set(now[None])
        ctx.tree_attention(q, dev["k"], dev["v"], dev["ks"], dev["vs"], lens, out, mask=hip.put(words(sees)[None]), account=account, decay=DECAY,
                           workspace=ws)
        # the same in 64 bits
        both = text + drafted
        for t in both:
            t.account *= DECAY
            t.off = t.off * DECAY + t.account * 2.0 ** -22
        for h in range(H):
            k = np.array([t.k[h * G // H] * float(t.ks) for t in both])
            for i in range(nodes):
                see = np.concatenate([np.ones(length, bool), sees[i]])
                s = k[see] @ now[i, h].astype(float) / np.sqrt(D)
                off = (np.abs(k[see]) @ np.abs(now[i, h].astype(float))).max() / np.sqrt(D) * 2.0 ** -19 + np.abs(s).max() * 2.0 ** -22
                p = np.exp(s - s.max())
                p /= p.sum()
                for t, w in zip([t for t, x in zip(both, see) if x], p):
                    t.account += w
                    t.off += w * (2 * off + 2.0 ** -17)
        # the accepted path: rows, scales and account go behind the cached ones; what is behind them is cleared
        path = path_to(parent, int(rng.integers(nodes)))
        text += [drafted[i] for i in path]
        accepted = np.zeros((1, nodes), np.int32)
        accepted[0, :len(path)] = np.array(path) + length
        old = account.get()
        old[:, length:] = 0
        spare.set(old)
        ctx.kv_compact(*rows, dev["ks"], dev["vs"], hip.put(accepted), hip.put(np.array([len(path)], np.int32)), account=account, account_out=spare,
                       first=length, workspace=ws3)
        account, spare = spare, account
        lens.set(lens.get() + len(path))
        check(text, dev, account)
        # back to the budget
        spare.set(np.zeros((1, P), f32))
        held = account.get()[0]
        ctx.kv_select(account, lens, keep, lens, sinks=SINKS, recent=RECENT)
        ctx.kv_compact(*rows, dev["ks"], dev["vs"], keep, lens, account=account, account_out=spare, workspace=ws3)
        account, spare = spare, account
        kept = chosen(held, len(text), BUDGET, SINKS, RECENT)
        assert np.array_equal(keep.get()[0, :len(kept)], kept)
        text = [text[i] for i in kept]
        assert lens.get()[0] == len(text)
        check(text, dev, account)


def check(text, dev, account):
    for n, d in dev.items():
        assert np.array_equal(d.get()[0, :len(text)], np.array([getattr(t, n) for t in text])), n
    got = account.get()[0].astype(np.float64)
    assert all(abs(a - t.account) <= t.off for a, t in zip(got, text))
    assert not got[len(text):].any()
