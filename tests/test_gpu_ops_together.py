"""The operators on device memory together, as a program that drafts trees uses them: every step attends a
tree over the cache and keeps the account, adjusts the nodes' logits, accepts a path of nodes, moves its rows
behind the cached ones, and at last keeps the cache within a budget, against the same steps in 64 bits.

The program's own parts are small: embeddings of its vocabulary as K, V and q, and the attention's output
times them as logits.  Each step starts from the same cache (the moved bytes are equal), so the tolerances are
those of one attention: an output off by at most T = vmax (2 d + 2^-18) + |out| 2^-24 (d: 2^-19 of the sum
of magnitudes of a score plus 2^-22 of the score) gives logits off by at most the sum of T |embedding|, and
the adjustment adds four roundings; accounts add up over the steps, each of them off by its weights' 2 d + 2^-17
and a rounding of 2^-22.  Picks are compared by their logits: a picked token's logit is within twice
that of the best.
"""
import ctypes

import numpy as np
import pytest

import qxg
from devmem import Hip

pytestmark = pytest.mark.gpu
f32 = np.float32
H, G, D, V = 8, 2, 64, 500      # q heads, kv heads, dims, vocabulary


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


def tree(rng, nodes):
    parent = np.array([rng.integers(-1, i) if i else -1 for i in range(nodes)])
    sees = np.eye(nodes, dtype=bool)
    for i, p in enumerate(parent):
        if p >= 0:
            sees[i] |= sees[p]
    return parent, sees


def words(flags):
    n = flags.shape[-1]
    f = np.zeros((*flags.shape[:-1], -(-n // 32) * 32), np.uint64)
    f[..., :n] = flags
    return (f.reshape(*f.shape[:-1], -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def path_to(parent, node):
    path = []
    while node >= 0:
        path.append(node)
        node = parent[node]
    return path[::-1]


class Program:
    """Both sides of it: device arrays, and what they have to hold."""

    def __init__(self, ctx, hip, nodes, positions, budget, seed):
        self.ctx, self.hip, self.nodes, self.budget = ctx, hip, nodes, budget
        self.rng = rng = np.random.default_rng(seed)
        self.k = np.zeros((1, positions, G, D), np.int8)
        self.v, self.ks, self.vs = self.k.copy(), np.ones((1, positions), f32), np.ones((1, positions), f32)
        self.account = np.zeros(positions)
        self.off = np.zeros(positions)          # how far the account may be off
        self.len, self.text = 0, []
        put = hip.put
        self.d = {"k": put(self.k), "v": put(self.v), "ks": put(self.ks), "vs": put(self.vs), "lens": put(np.zeros(1, np.int32)),
                  "account": put(np.zeros((1, positions), f32)), "spare": put(np.zeros((1, positions), f32)),
                  "q": put(np.zeros((1, nodes, H, D), f32)), "out": put(np.zeros((1, nodes, H, D), f32)),
                  "mask": put(np.zeros((1, nodes, -(-nodes // 32)), np.int32)), "logits": put(np.zeros((nodes, V), f32)),
                  "history": put(np.full((nodes, 64), -1, np.int32)), "ids": put(np.zeros((nodes, 4), np.int32)),
                  "best": put(np.zeros((nodes, 4), f32)), "penalties": put(np.full((nodes, 3), [1.25, 0.125, 0.0625], f32)),
                  "temperature": put(np.full(nodes, 0.5, f32)), "accepted": put(np.zeros((1, nodes), np.int32)),
                  "n": put(np.zeros(1, np.int32)), "keep": put(np.zeros((1, budget), np.int32)), "kept": put(np.zeros(1, np.int32))}
        ws = hip.workspace
        self.ws_tree = ws(ctx.tree_attention_workspace((1, nodes, H, D), self.k.shape, account=True))
        self.ws_logits = ws(ctx.adjust_logits_workspace((nodes, V), 4))
        self.ws_move = ws(max(ctx.kv_compact_workspace((1, positions, G * D), (1, nodes)), ctx.kv_compact_workspace((1, positions, G * D), (1, budget))))
        self.rows = [hip_rows(self.d[x], (1, positions, G * D)) for x in ("k", "v")]
        # the vocabulary's rows of K and V, and its embeddings
        self.vk, self.vv = (rng.integers(-127, 128, (V, G, D)).astype(np.int8) for _ in range(2))
        self.vs_k, self.vs_v = (rng.uniform(0.02, 0.04, V).astype(f32) for _ in range(2))
        self.embed = (rng.standard_normal((V, H * D)) * 0.1).astype(f32)

    def append(self, tokens, at):
        self.k[0, at:at + len(tokens)], self.v[0, at:at + len(tokens)] = self.vk[tokens], self.vv[tokens]
        self.ks[0, at:at + len(tokens)], self.vs[0, at:at + len(tokens)] = self.vs_k[tokens], self.vs_v[tokens]
        for x, a in (("k", self.k), ("v", self.v), ("ks", self.ks), ("vs", self.vs)):
            self.d[x].set(a)

    def queue_step(self, stream):
        """Attention with the account; what a captured step replays."""
        d = self.d
        self.ctx.tree_attention(d["q"], d["k"], d["v"], d["ks"], d["vs"], d["lens"], d["out"], mask=d["mask"], account=d["account"], decay=0.5,
                                workspace=self.ws_tree, stream=stream, wait=False)

    def queue_logits(self, stream):
        d = self.d
        self.ctx.adjust_logits(d["logits"], d["logits"], history=d["history"], penalties=d["penalties"], temperature=d["temperature"],
                               top_ids=d["ids"], top_logits=d["best"], workspace=self.ws_logits, stream=stream, wait=False)

    def queue_accept(self, stream):
        d = self.d
        self.ctx.kv_compact(*self.rows, d["ks"], d["vs"], d["accepted"], d["n"], first=self.len, workspace=self.ws_move, stream=stream, wait=False)

    def queue_evict(self, stream):
        d = self.d
        self.ctx.kv_select(d["account"], d["lens"], d["keep"], d["kept"], sinks=2, recent=5, stream=stream, wait=False)
        self.ctx.kv_compact(*self.rows, d["ks"], d["vs"], d["keep"], d["kept"], account=d["account"], account_out=d["spare"], workspace=self.ws_move,
                            stream=stream, wait=False)

    def same_cache(self):
        for x, a in (("k", self.k), ("v", self.v), ("ks", self.ks), ("vs", self.vs)):
            assert np.array_equal(self.d[x].get()[0, :self.len], a[0, :self.len]), x


def hip_rows(a, shape):
    return a.view(0, shape, (shape[1] * shape[2], shape[2], 1))


@pytest.mark.parametrize("nodes,captured", [(1, False), (7, False), (7, True), (40, True)])
def test_drafted_steps_within_a_budget(ctx, hip, nodes, captured):
    budget, positions, steps = 48, 160, 10
    p = Program(ctx, hip, nodes, positions, budget, seed=nodes)
    d, rng, stream = p.d, p.rng, hip.stream()
    start = rng.integers(0, V, 30)
    p.append(start, 0)
    p.len, p.text = 30, start.tolist()
    graphs = [hip.capture(stream, lambda f=f: f(stream)) for f in (p.queue_step, p.queue_logits, p.queue_evict)] if captured else None

    def run(i, f):
        hip.hipGraphLaunch(graphs[i], ctypes.c_void_p(stream)) if captured else f(stream)
        hip.hipStreamSynchronize(ctypes.c_void_p(stream))

    for _ in range(steps):
        parent, sees = tree(rng, nodes)
        tokens = rng.integers(0, V, nodes)
        p.append(tokens, p.len)
        T = p.len + nodes
        q = (rng.standard_normal((nodes, H, D)) * 0.5).astype(f32)
        for x, a in (("q", q[None]), ("mask", words(sees)[None]), ("lens", np.array([p.len], np.int32))):
            d[x].set(a)
        run(0, p.queue_step)
        # the attention and its account in 64 bits
        vis = np.concatenate([np.ones((nodes, p.len), bool), sees], 1)
        out, t_out = np.zeros((nodes, H, D)), np.zeros((nodes, H, D))
        p.account[:T] *= 0.5
        p.off[:T] = p.off[:T] * 0.5 + p.account[:T] * 2.0 ** -22
        for h in range(H):
            k, v = p.k[0, :T, h // (H // G)] * p.ks[0, :T, None].astype(float), p.v[0, :T, h // (H // G)] * p.vs[0, :T, None].astype(float)
            for i in range(nodes):
                w = np.flatnonzero(vis[i])
                s = k[w] @ q[i, h].astype(float) / np.sqrt(D)
                off = (np.abs(k[w]) @ np.abs(q[i, h].astype(float))).max() / np.sqrt(D) * 2.0 ** -19 + np.abs(s).max() * 2.0 ** -22
                e = np.exp(s - s.max())
                e /= e.sum()
                out[i, h] = e @ v[w]
                t_out[i, h] = np.abs(v[w]).max() * (2 * off + 2.0 ** -18) + np.abs(out[i, h]) * 2.0 ** -24
                p.account[w] += e
                p.off[w] += e * (2 * off + 2.0 ** -17)
        got = d["out"].get()[0].astype(np.float64)
        assert (np.abs(got - out) <= t_out).all()
        assert (np.abs(d["account"].get()[0, :T] - p.account[:T]) <= p.off[:T]).all()
        # logits of every node under its path's history
        d["logits"].set((got.reshape(nodes, -1) @ p.embed.T.astype(float)).astype(f32))
        logits = out.reshape(nodes, -1) @ p.embed.T.astype(float)
        t_logits = t_out.reshape(nodes, -1) @ np.abs(p.embed.T.astype(float)) + np.abs(logits) * 2.0 ** -24
        history = np.full((nodes, 64), -1, np.int32)
        for i in range(nodes):
            said = p.text[-20:] + tokens[path_to(parent, i)].tolist()
            history[i, :len(said)] = said
            for t, c in zip(*np.unique(said, return_counts=True)):
                x = logits[i, t]
                logits[i, t] = (x / 1.25 if x > 0 else x * 1.25) - 0.125 * c - 0.0625
                t_logits[i, t] = 1.25 * t_logits[i, t] + (1.25 * abs(x) + 0.125 * c + 0.0625) * 3 * 2.0 ** -24
        logits /= 0.5
        t_logits = t_logits / 0.5 + np.abs(logits) * 2.0 ** -24
        d["history"].set(history)
        run(1, p.queue_logits)
        assert (np.abs(d["logits"].get() - logits) <= t_logits).all()
        ids, best, dev = d["ids"].get(), d["best"].get(), d["logits"].get()
        for i in range(nodes):
            want = np.lexsort((np.arange(V), -dev[i]))[:4]
            assert np.array_equal(ids[i], want) and np.array_equal(best[i], dev[i, want])
            assert (logits[i, ids[i]] >= np.sort(logits[i])[::-1][:4] - 2 * t_logits[i].max()).all()
        # the path to the node with the largest logit is accepted: its rows go behind the cached ones
        path = path_to(parent, int(np.argmax(best[:, 0])))
        rows = np.zeros((1, nodes), np.int32)
        rows[0, :len(path)] = np.array(path) + p.len
        d["accepted"].set(rows)
        d["n"].set(np.array([len(path)], np.int32))
        p.queue_accept(stream)
        hip.hipStreamSynchronize(ctypes.c_void_p(stream))
        at, to = np.array(path) + p.len, np.arange(len(path)) + p.len
        for a in (p.k[0], p.v[0], p.ks[0], p.vs[0], p.account, p.off):
            a[to] = a[at]
        account = d["account"].get()      # (the program moves the account of the few nodes itself)
        account[0, to] = account[0, at]
        d["account"].set(account)
        p.text += tokens[path].tolist()
        p.len += len(path)
        p.same_cache()
        if p.len <= budget:
            continue
        # and the cache goes back to its budget
        d["lens"].set(np.array([p.len], np.int32))
        run(2, p.queue_evict)
        held = d["account"].get()[0].astype(float)
        keep = d["keep"].get()[0]
        middle = np.arange(2, p.len - 5)
        chosen = np.sort(np.concatenate([[0, 1], middle[np.lexsort((middle, -held[middle]))[:budget - 7]], np.arange(p.len - 5, p.len)]))
        assert d["kept"].get()[0] == budget and np.array_equal(keep, chosen)
        left = np.setdiff1d(middle, keep)
        assert (p.account[left] - p.off[left]).max() <= (p.account + p.off)[np.setdiff1d(keep, [0, 1, *range(p.len - 5, p.len)])].min() + 2 * p.off.max()
        for a in (p.k[0], p.v[0], p.ks[0], p.vs[0], p.account, p.off):
            a[:budget] = a[keep]
        p.len = budget
        p.same_cache()
        moved = d["spare"].get()
        assert np.array_equal(moved[0, :budget], d["account"].get()[0, keep])
        d["account"].set(np.concatenate([moved[:, :budget], np.zeros((1, positions - budget), f32)], 1))
        p.account[budget:] = p.off[budget:] = 0
