"""Operators of a decode step over the INT8 KV cache, as cases that can be timed: attention for a tree of
drafted tokens (and the account of attention weights that it keeps), eviction of cache rows by that
account, and the logits on their way to the chosen tokens.

`run` computes them in plain torch operations where `own` is false and through qxg.Context where it is
true.  Index arrays are int32 tensors, as a program that fills the framework's 32-bit arrays holds them."""
import functools
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False

VOCAB, CONTEXT = 151936, 4096
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token over the beginning of a conversation: single-token decode, where latency counts
        _tree("token_short", "f32", 1, 1, 32, 4, 128, 37),
        # a drafted tree in the middle of a conversation, the model's heads
        _tree("tree_step", "f32", 1, 16, 32, 4, 128, 1500),
        # a wide tree at the end of the context
        _tree("tree_context_end", "f32", 1, 64, 32, 4, 128, CONTEXT - 64),
        # several conversations of unlike lengths, short drafts, 16-bit activations, small heads
        _tree("tree_batch", "bf16", 8, 13, 14, 2, 64, 2900),
        # long documents
        _tree("tree_long", "f16", 2, 48, 32, 4, 128, 65500),
        # a drafted tree that also keeps the account of attention weights
        _tree("account_step", "f32", 1, 16, 32, 4, 128, 1500, weights=True),
        # the same for single tokens of several long conversations
        _tree("account_long", "bf16", 4, 1, 32, 8, 128, 30000, weights=True),
        # a short cache kept within its budget (one layer)
        _evict("evict_one", 1, 700, 700, 512, 4, 64, 512),
        # every layer of the model, the full context down to its half
        _evict("evict_layers", 48, CONTEXT, CONTEXT, CONTEXT // 2, 4, 256, 512),
        # long documents down to a quarter
        _evict("evict_long", 3, 131072, 131000, 32768, 16, 2048, 512),
        # the head's logits of one token under a grammar
        _logits("logits_one", "f32", 1, VOCAB, 500, 20, 1, 8),
        # a batch of drafted nodes or of conversations, with long histories
        _logits("logits_batch", "f32", 64, VOCAB, 4000, 50, 3, 32),
    ]


def _tree(name, dtype, batch, nodes, heads, kv_heads, dim, length, weights=False):
    return {"name": name, "kind": "tree", "type": dtype, "batch": batch, "nodes": nodes, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "len": length, "weights": weights}


def _evict(name, groups, positions, length, budget, sinks, recent, row):
    return {"name": name, "kind": "evict", "groups": groups, "positions": positions, "len": length, "budget": budget,
            "sinks": sinks, "recent": recent, "row": row}


def _logits(name, dtype, rows, vocab, history, biases, masks, top_n):
    return {"name": name, "kind": "logits", "type": dtype, "rows": rows, "vocab": vocab, "history": history, "biases": biases,
            "masks": masks, "top_n": top_n}


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "account", "account", "evict", "evict", "logits", "logits"])
    if kind in ("tree", "account"):
        kv_heads, group = rng.choice([1, 2, 4, 4, 8]), rng.choice([1, 2, 4, 7, 8, 8])
        batch, nodes, dim = rng.choice([1, 1, 2, 3, 5, 8]), _log_int(rng, 1, 64), rng.choice([64, 128, 128])
        # the longest cache whose work is no more than the largest listed case's
        most = 2 * 48 * 32 * 128 * 65500 // (batch * max(nodes, 4) * max(kv_heads * group, 8) * dim)
        most = min(most, 65500, 2 ** 30 // (batch * kv_heads * dim * 8))
        case = _tree("", rng.choice(["f32", "f32", "f16", "bf16"]), batch, nodes, kv_heads * group, kv_heads, dim, _log_int(rng, 3, most),
                     kind == "account")
    elif kind == "evict":
        groups = rng.choice([1, 1, 2, 5, 16, 48])
        length = _log_int(rng, 40, min(131000, 131000 * 3 // groups))
        budget = rng.randrange(length // 5 + 2, length + 1)
        sinks = rng.randrange(0, min(17, budget // 4 + 1))
        case = _evict("", groups, length + rng.randrange(0, 100), length, budget, sinks, rng.randrange(0, budget // 2 + 1),
                      rng.choice([128, 512, 512, 1024]) if length * groups < 131000 else 512)
    else:
        rows, vocab = _log_int(rng, 1, 64), rng.choice([_log_int(rng, 300, VOCAB), VOCAB])
        case = _logits("", rng.choice(["f32", "f32", "f16", "bf16"]), rows, vocab, _log_int(rng, 1, 4000), rng.randrange(0, 51), rng.randrange(0, 4),
                       rng.choice([1, 4, 8, 32]))
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"tree": _prepare_tree, "evict": _prepare_evict, "logits": _prepare_logits}[case["kind"]](case, g)


def _codes(g, *shape):
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float16) * 36).round_().clamp_(-127, 127).to(torch.int8)


def _uniform(g, lo, hi, *shape):
    return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo


def _whole(g, lo, hi, *shape):
    """int32 values lo .. hi, both included."""
    return torch.randint(lo, hi + 1, shape, device="cuda", generator=g, dtype=torch.int32)


def _ragged(g, n, most):
    """n lengths up to `most`, the first of them `most`."""
    lens = _whole(g, max(1, most // 3), most, n)
    lens[0] = most
    return lens


def _prepare_tree(case, g):
    B, n, H, Hk, D = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim"))
    dtype, P = TYPES[case["type"]], case["len"] + case["nodes"] + 5
    s = {"case": case, "q": (torch.randn((B, n, H, D), device="cuda", generator=g) * 2).to(dtype)}
    s["k"], s["v"] = _codes(g, B, P, Hk, D), _codes(g, B, P, Hk, D)
    # a row's scale is its largest magnitude / 127
    s["kscale"], s["vscale"] = (_uniform(g, 3.0, 4.5, B, P) / 127 for _ in range(2))
    s["lens"], s["counts"] = _ragged(g, B, case["len"]), _ragged(g, B, n)
    # a node's parent is a node before it or the last cached token; it sees its ancestors and itself
    up = (torch.rand((B, n), device="cuda", generator=g) * (torch.arange(n, device="cuda") + 1)).long() - 1
    sees = torch.eye(n, device="cuda", dtype=torch.bool).repeat(B, 1, 1)
    for i in range(1, n):
        rows = torch.gather(sees, 1, up[:, i].clamp(min=0)[:, None, None].expand(B, 1, n))[:, 0]
        sees[:, i] |= rows & (up[:, i] >= 0)[:, None]
    s["mask"] = _bits(sees)
    s["out"], s["lse"] = torch.zeros((B, n, H, D), device="cuda", dtype=dtype), torch.zeros((B, n, H), device="cuda")
    if case["weights"]:
        s["account"], s["decay"] = _uniform(g, 0.0, 4.0, B, P), 0.96875
    return s


def _bits(flags):
    """The truth values of the last axis as bits of int32 words, value j bit j % 32 of word j / 32."""
    n = flags.shape[-1]
    flags = torch.nn.functional.pad(flags, (0, -n % 32)).unflatten(-1, (-1, 32)).long()
    words = (flags << torch.arange(32, device=flags.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _prepare_evict(case, g):
    G, P, row, budget = (case[k] for k in ("groups", "positions", "row", "budget"))
    s = {"case": case, "k": _codes(g, G, P, row), "v": _codes(g, G, P, row)}
    s["kscale"], s["vscale"] = (_uniform(g, 3.0, 4.5, G, P) / 127 for _ in range(2))
    # few positions gather most of the weight; some have gathered the same
    w = torch.randn((G, P), device="cuda", generator=g).mul_(2).exp_()
    s["account"] = torch.where(_uniform(g, 0, 1, G, P) < 0.05, torch.zeros_like(w), w)
    s["lens"] = _ragged(g, G, case["len"])
    s["keep"] = torch.zeros((G, budget), device="cuda", dtype=torch.int32)
    s["kept"] = torch.zeros((G,), device="cuda", dtype=torch.int32)
    s["account_out"] = torch.zeros((G, P), device="cuda")
    return s


def _prepare_logits(case, g):
    R, V, T, nb, masks, n = (case[k] for k in ("rows", "vocab", "history", "biases", "masks", "top_n"))
    dtype = TYPES[case["type"]]
    s = {"case": case, "logits": (torch.randn((R, V), device="cuda", generator=g) * 2.5).to(dtype)}
    s["out"] = torch.zeros_like(s["logits"])
    # common tokens come often
    s["history"] = (V ** _uniform(g, 0.0, 1.0, R, T)).to(torch.int32).clamp_(0, V - 1)
    s["history_lens"] = _ragged(g, R, T)
    s["prompt_lens"] = (s["history_lens"] * _uniform(g, 0.0, 1.0, R)).to(torch.int32)
    s["penalties"] = torch.stack([_uniform(g, 1.0, 1.4, R), _uniform(g, 0.0, 0.3, R), _uniform(g, 0.0, 0.5, R)], 1).contiguous()
    s["temperature"] = _uniform(g, 0.5, 1.2, R)
    s["bias_ids"] = _whole(g, 0, V - 1, R, nb) if nb else None
    # (sums of the biases of one token come out the same in any order)
    s["bias_values"] = _whole(g, -16, 16, R, nb).float() / 4 if nb else None
    s["mask"] = s["mask_rows"] = None
    if masks:
        open_share = torch.tensor([0.02, 0.9, 0.5], device="cuda")[:masks, None]
        s["mask"] = _bits(torch.rand((masks, V), device="cuda", generator=g) < open_share)
        s["mask_rows"] = _whole(g, -1 if R > 1 else 0, masks - 1, R)
    s["top_ids"] = torch.zeros((R, n), device="cuda", dtype=torch.int32)
    s["top_logits"], s["lse"] = torch.zeros((R, n), device="cuda"), torch.zeros((R,), device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tree": _own_tree, "evict": _own_evict, "logits": _own_logits}[kind](state)
    return {"tree": _plain_tree, "evict": _plain_evict, "logits": _plain_logits}[kind](state)


@functools.lru_cache(maxsize=None)
def _context():
    """The program's context."""
    if os.path.join(ROOT, "qx-mini-c_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "qx-mini-c_amd"))
    import qxg
    return qxg.Context(torch.cuda.current_device())


@functools.lru_cache(maxsize=None)
def _workspace(nbytes):
    """The program's workspace of that size, which its calls on the one stream share."""
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")


def _own_tree(s):
    c, case = _context(), s["case"]
    need = c.tree_attention_workspace(s["q"].shape, s["k"].shape, max_len=case["len"], account=case["weights"])
    c.tree_attention(s["q"], s["k"], s["v"], s["kscale"], s["vscale"], s["lens"], s["out"], mask=s["mask"], counts=s["counts"], lse=s["lse"],
                     account=s["account"] if case["weights"] else None, decay=s["decay"] if case["weights"] else 1.0, max_len=case["len"],
                     workspace=_workspace(need), stream=torch.cuda.current_stream().cuda_stream, wait=False)
    return {"out": s["out"], "lse": s["lse"], **({"account": s["account"]} if case["weights"] else {})}


def _own_evict(s):
    c, case = _context(), s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    c.kv_select(s["account"], s["lens"], s["keep"], s["kept"], sinks=case["sinks"], recent=case["recent"], max_len=case["len"], stream=stream,
                wait=False)
    need = c.kv_compact_workspace(s["k"].shape, s["keep"].shape)
    c.kv_compact(s["k"], s["v"], s["kscale"], s["vscale"], s["keep"], s["kept"], account=s["account"], account_out=s["account_out"],
                 workspace=_workspace(need), stream=stream, wait=False)
    return {k: s[k] for k in ("keep", "kept", "k", "v", "kscale", "vscale", "account_out")}


def _own_logits(s):
    c = _context()
    need = c.adjust_logits_workspace(s["logits"].shape, s["case"]["top_n"])
    c.adjust_logits(s["logits"], s["out"], history=s["history"], history_lens=s["history_lens"], prompt_lens=s["prompt_lens"],
                    penalties=s["penalties"], temperature=s["temperature"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                    mask=s["mask"], mask_rows=s["mask_rows"], top_ids=s["top_ids"], top_logits=s["top_logits"], lse=s["lse"],
                    workspace=_workspace(need), stream=torch.cuda.current_stream().cuda_stream, wait=False)
    return {k: s[k] for k in ("out", "top_ids", "top_logits", "lse")}


def _visible(s):
    """[batch, nodes, positions]: the cached positions, and the nodes that the mask names."""
    B, P, _, _ = s["k"].shape
    n = s["q"].shape[1]
    p = torch.arange(P, device="cuda")
    j = p[None] - s["lens"][:, None].long()
    named = (torch.gather(s["mask"], 2, (j >> 5).clamp(0, s["mask"].shape[2] - 1)[:, None].expand(B, n, P)) >> (j & 31)[:, None]) & 1
    return (j < 0)[:, None] | ((j >= 0) & (j < s["counts"][:, None]))[:, None] & (named != 0)


def _plain_tree(s):
    B, P, Hk, D = s["k"].shape
    n, H = s["q"].shape[1:3]
    G = H // Hk
    q = s["q"].float().reshape(B, n, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B * Hk, n * G, D)
    k = (s["k"].float() * s["kscale"][:, :, None, None]).permute(0, 2, 3, 1).reshape(B * Hk, D, P)
    v = (s["v"].float() * s["vscale"][:, :, None, None]).permute(0, 2, 1, 3).reshape(B * Hk, P, D)
    score = torch.bmm(q, k).mul_(1 / math.sqrt(D)).view(B, Hk, n, G, P)
    score.masked_fill_(~_visible(s)[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = score.sub_(top).exp_()
    den = e.sum(-1, keepdim=True)
    out = torch.bmm(e.view(B * Hk, n * G, P), v).view(B, Hk, n, G, D) / torch.where(den > 0, den, 1.0)
    lse = torch.where(den > 0, top + den.log(), -math.inf)
    used = (torch.arange(n, device="cuda")[None] < s["counts"][:, None])[:, :, None]
    got = {"out": torch.where(used[..., None], out.permute(0, 2, 1, 3, 4).reshape(B, n, H, D).to(s["out"].dtype), s["out"]),
           "lse": torch.where(used, lse.permute(0, 2, 1, 3, 4).reshape(B, n, H), s["lse"])}
    if s["case"]["weights"]:
        share = e.div_(torch.where(den > 0, den, 1.0)).mul_(used[:, None, :, :, None])
        held = torch.arange(P, device="cuda")[None] < (s["lens"] + s["counts"])[:, None]
        s["account"].copy_(torch.where(held, s["account"] * s["decay"] + share.sum((1, 2, 3)), s["account"]))
        got["account"] = s["account"]
    return got


def _plain_evict(s):
    case = s["case"]
    G, P, budget = case["groups"], case["positions"], case["budget"]
    p, lens = torch.arange(P, device="cuda")[None], s["lens"][:, None].long()
    # the first and the last positions before all others, positions behind the end after them
    weight = torch.where((p < case["sinks"]) | (p >= lens - case["recent"]), math.inf, s["account"])
    weight = torch.where(p < lens, weight, -math.inf)
    best = torch.sort(weight, dim=1, descending=True, stable=True).indices[:, :budget]
    kept = lens.clamp(max=budget)
    i = torch.arange(budget, device="cuda")[None]
    order = torch.sort(torch.where(i < kept, best, P), dim=1).values
    s["keep"].copy_(torch.where(i < kept, order, s["keep"]))
    s["kept"].copy_(kept[:, 0])
    at, group = order.clamp(max=P - 1), torch.arange(G, device="cuda")[:, None]
    moved = i < kept
    for name in ("k", "v", "kscale", "vscale"):
        new = s[name][group, at]
        s[name][:, :budget] = torch.where(moved[..., None] if new.dim() == 3 else moved, new, s[name][:, :budget])
    s["account_out"][:, :budget] = torch.where(moved, s["account"][group, at], s["account_out"][:, :budget])
    return {k: s[k] for k in ("keep", "kept", "k", "v", "kscale", "vscale", "account_out")}


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    T = s["history"].shape[1]
    t = torch.arange(T, device="cuda")[None]
    token = torch.where(t < s["history_lens"][:, None], s["history"], V).long()
    seen = torch.zeros((R, V + 1), device="cuda", dtype=torch.int32).scatter_add_(1, token, torch.ones_like(s["history"]))[:, :V] > 0
    made = torch.zeros((R, V + 1), device="cuda", dtype=torch.int32)
    made = made.scatter_add_(1, torch.where(t >= s["prompt_lens"][:, None], token, V), torch.ones_like(s["history"]))[:, :V]
    again, often, present = (s["penalties"][:, i:i + 1] for i in range(3))
    x = torch.where(seen, torch.where(x > 0, x / again, x * again), x)
    x = x - often * made.float()
    x = x - present * (made > 0).float()
    if s["bias_ids"] is not None:
        same = s["bias_ids"][:, :, None] == s["bias_ids"][:, None, :]
        total = torch.where(same, s["bias_values"][:, None, :], 0.0).sum(-1)
        x = x + torch.zeros_like(x).scatter_(1, s["bias_ids"].long(), total)
    x = x / s["temperature"][:, None]
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        allowed = ((s["mask"][:, v >> 5] >> (v & 31)) & 1) != 0
        rows = s["mask_rows"].long()
        x = torch.where((rows < 0)[:, None] | allowed[rows.clamp(min=0)], x, -math.inf)
    top = torch.sort(x, dim=1, descending=True, stable=True)
    n = s["case"]["top_n"]
    some = top.values[:, :n] > -math.inf
    most = x.amax(1, keepdim=True)
    lse = (x - most).exp().sum(1).log() + most[:, 0]
    return {"out": x.to(s["out"].dtype), "top_ids": torch.where(some, top.indices[:, :n], -1).to(torch.int32), "top_logits": top.values[:, :n],
            "lse": lse}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "tree":
        B, n, H, Hk, D, L = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim", "len"))
        # of several sequences the others have about 2/3 of the longest's positions and nodes
        rows, nodes = (L + n) * (1 + (B - 1) * 2 / 3), n * (1 + (B - 1) * 2 / 3)
        size = 4 if case["type"] == "f32" else 2
        moved = rows * (2 * Hk * D + 8) + nodes * (2 * H * D * size + 4 * H + (n + 31) // 32 * 4) + (rows * 8 if case["weights"] else 0)
        return {"bytes": moved, "flops": 4 * H * D * n * (L + n) * (1 + (B - 1) * 4 / 9)}
    if case["kind"] == "evict":
        lens = case["len"] * (1 + (case["groups"] - 1) * 2 / 3)
        kept = min(case["budget"], case["len"]) * case["groups"]
        return {"bytes": 4 * lens + kept * (2 * (2 * case["row"] + 8) + 4 + 4), "flops": lens}
    size = 4 if case["type"] == "f32" else 2
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * (2 * V * size + 4 * case["history"] + 8 * case["biases"] + 8 * case["top_n"]) + case["masks"] * V / 8, "flops": 8 * R * V}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    return {"tree": _exact_tree, "evict": _exact_evict, "logits": _exact_logits}[case["kind"]](prepare(case, seed))


def _exact_tree(s):
    B, n, H, D = s["q"].shape
    Hk = s["k"].shape[2]
    out, lse = s["out"].double(), s["lse"].double()
    account = s["account"].double() if "account" in s else None
    for b in range(B):
        length, count = int(s["lens"][b]), int(s["counts"][b])
        words = s["mask"][b, :count].cpu().tolist()
        sees = torch.tensor([[(words[i][j // 32] >> (j % 32)) & 1 for j in range(count)] for i in range(count)], device="cuda", dtype=torch.bool)
        sees = torch.cat([torch.ones((count, length), device="cuda", dtype=torch.bool), sees], 1)
        total = 0.0
        for h in range(H):
            rows = slice(0, length + count)
            k = s["k"][b, rows, h * Hk // H].double() * s["kscale"][b, rows, None].double()
            v = s["v"][b, rows, h * Hk // H].double() * s["vscale"][b, rows, None].double()
            score = s["q"][b, :count, h].double() @ k.T / math.sqrt(D)
            score = torch.where(sees, score, -math.inf)
            lse[b, :count, h] = torch.logsumexp(score, 1)
            p = torch.softmax(score, 1)
            out[b, :count, h] = p @ v
            total = total + p.sum(0)
        if account is not None:
            account[b, :length + count] = s["decay"] * account[b, :length + count] + total
    return {"out": out, "lse": lse, **({} if account is None else {"account": account})}


def _exact_evict(s):
    case = s["case"]
    got = {k: s[k].clone() for k in ("keep", "kept", "k", "v", "kscale", "vscale", "account_out")}
    for g in range(case["groups"]):
        length = int(s["lens"][g])
        kept = min(length, case["budget"])
        if length <= case["budget"]:
            chosen = list(range(length))
        else:
            first, last = range(case["sinks"]), range(length - case["recent"], length)
            account = s["account"][g].tolist()
            middle = sorted(range(case["sinks"], length - case["recent"]), key=lambda p: (-account[p], p))
            chosen = sorted([*first, *last, *middle[:kept - len(first) - len(last)]])
        chosen = torch.tensor(chosen, device="cuda")
        got["keep"][g, :kept], got["kept"][g] = chosen.to(torch.int32), kept
        for name in ("k", "v", "kscale", "vscale"):
            got[name][g, :kept] = s[name][g, chosen]
        got["account_out"][g, :kept] = s["account"][g, chosen]
    return {k: v.double() if v.is_floating_point() else v for k, v in got.items()}


def _exact_logits(s):
    case = s["case"]
    x = s["logits"].double()
    n = case["top_n"]
    ids, values, lse = [], [], []
    for r in range(case["rows"]):
        made = s["history"][r, :int(s["history_lens"][r])].long()
        again, often, present = s["penalties"][r].double().tolist()
        seen = torch.unique(made)
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / again, x[r, seen] * again)
        token, count = torch.unique(made[int(s["prompt_lens"][r]):], return_counts=True)
        x[r, token] -= often * count + present
        if s["bias_ids"] is not None:
            for token, bias in zip(s["bias_ids"][r].tolist(), s["bias_values"][r].tolist()):
                x[r, token] += bias
        x[r] /= s["temperature"][r].double()
        if s["mask"] is not None and int(s["mask_rows"][r]) >= 0:
            words = s["mask"][int(s["mask_rows"][r])]
            bit = torch.stack([(words >> i) & 1 for i in range(32)], 1).reshape(-1)[:case["vocab"]]
            x[r, bit == 0] = -math.inf
        v, i = torch.topk(x[r], n)
        ids.append(torch.where(v > -math.inf, i, -1))
        values.append(v)
        lse.append(torch.logsumexp(x[r], 0))
    return {"out": x, "top_ids": torch.stack(ids).to(torch.int32), "top_logits": torch.stack(values), "lse": torch.stack(lse)}
