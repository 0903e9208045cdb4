"""Timed cases of the drafted-token tree operators: what a speculative decode step calls.

A drafter proposes a tree of tokens after the cached prefix; node 0 is the last emitted
token (whose cache row is not written yet), node t > 0 a drafted token below parents[t] < t.
One step checks all of them: their Q/K/V rows are biased, rotated at prefix + depth and laid
out (tree_qkv_rope), attention runs over the prefix and each node's ancestors
(tree_attention), the nodes' logits decide which path stands (tree_verify), and its rows go
into the caches of all layers (tree_commit).

Sizes are those of this repository's configurations and tests (16 heads x 128, 24 layers,
vocabulary 151936, caches up to 32768 rows), and grouped heads (32 and 8) as models with
shared K/V heads have them.  Inputs are synthetic: activations N(0, 1), cache rows N(0, 1),
logits with a few strong candidates over a wide tail, drafts drawn near the target.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

D = 128
ROPE_BASE = 10000.0
DEV = "cuda"


def _qdiy():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "llm-inference-diy_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import qdiy
    return qdiy


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a chain of four drafts after a chat-sized context: the smallest pass, launches and host cost
        dict(name="attn_chain5_512", kind="attn", heads=16, kv_heads=16, nodes=5, chain=True, prefix=512,
             layout="engine"),
        # a usual draft tree, odd in both lengths, over the benchmark's headline context
        dict(name="attn_tree27_8191", kind="attn", heads=16, kv_heads=16, nodes=27, chain=False, prefix=8191,
             layout="engine"),
        # a wide draft tree at the end of the longest context: 268 MB of cache
        dict(name="attn_tree64_32700", kind="attn", heads=16, kv_heads=16, nodes=64, chain=False, prefix=32700,
             layout="engine"),
        # shared K/V heads (four queries each), a cache with one block per head, ragged lengths
        dict(name="attn_grouped_tree48_16001", kind="attn", heads=32, kv_heads=8, nodes=48, chain=False,
             prefix=16001, layout="head_major"),
        # a tree so wide that the products weigh as much as the cache
        dict(name="attn_tree250_4001", kind="attn", heads=16, kv_heads=16, nodes=250, chain=False, prefix=4001,
             layout="engine"),
        # the same step's Q/K/V rows: a short chain ...
        dict(name="rope_chain5_512", kind="rope", heads=16, kv_heads=16, nodes=5, chain=True, prefix=512),
        # ... and a wide tree far into a context, shared K/V heads
        dict(name="rope_tree250_30001", kind="rope", heads=32, kv_heads=8, nodes=250, chain=False, prefix=30001),
        # greedy check of a short chain over the model's vocabulary
        dict(name="verify_greedy5", kind="verify", mode="greedy", nodes=5, chain=True, vocab=151936),
        # sampled check of a tree of most likely candidates (drafts without probabilities)
        dict(name="verify_point64", kind="verify", mode="point", nodes=64, chain=False, vocab=151936),
        # sampled check of a tree drawn from the drafter's own probabilities, a small odd vocabulary
        dict(name="verify_drawn27", kind="verify", mode="drawn", nodes=27, chain=False, vocab=32003),
        # keeping a usual accepted path in the caches of 24 layers
        dict(name="commit_4_of_27", kind="commit", heads=16, layers=24, nodes=27, keep=4, prefix=700, rows=800),
        # and a long accepted chain
        dict(name="commit_60_of_64", kind="commit", heads=16, layers=24, nodes=64, keep=60, prefix=700, rows=800),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "rope", "verify", "verify", "commit"))
    nodes = _log_int(rng, 1, 250)
    if kind == "attn":
        heads, kv_heads = rng.choice(((16, 16), (16, 16), (8, 8), (4, 4), (32, 8), (16, 2), (28, 4), (20, 20)))
        # at most the largest listed case's cache bytes and products
        most = min(32700, 64 * 32764 * 16 // (nodes * heads), 32764 * 16 // kv_heads)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, nodes=nodes, chain=rng.random() < 0.3,
                    prefix=_log_int(rng, 1, max(1, most - nodes)) - (rng.random() < 0.1),
                    layout=rng.choice(("engine", "engine", "head_major", "padded")))
    if kind == "rope":
        heads, kv_heads = rng.choice(((16, 16), (8, 8), (32, 8), (16, 2), (28, 4)))
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, nodes=nodes, chain=rng.random() < 0.3,
                    prefix=_log_int(rng, 1, 32000))
    if kind == "verify":
        mode = rng.choice(("greedy", "point", "drawn"))
        nodes = _log_int(rng, 1, 64)
        vocab = _log_int(rng, 500, 151936)
        if mode == "drawn":
            vocab = min(vocab, 64 * 151936 // (2 * nodes))
        return dict(kind=kind, mode=mode, nodes=nodes, chain=rng.random() < 0.3, vocab=vocab)
    nodes = min(nodes, 64)
    return dict(kind=kind, heads=rng.choice((4, 8, 16)), layers=rng.choice((2, 12, 24)), nodes=nodes,
                keep=rng.randint(1, min(nodes, 60)), prefix=rng.randint(0, 700), rows=800)


# ------------------------------------------------------------------ inputs

def _tree(rs, nodes, chain):
    """Parents of a drafted tree: a chain, or a tree whose nodes hang below one of the eight
    nodes before them."""
    return [-1] + [t - 1 if chain else int(rs.integers(max(0, t - 8), t)) for t in range(1, nodes)]


def _depths(parents):
    d = [0] * len(parents)
    for t in range(1, len(parents)):
        d[t] = d[parents[t]] + 1
    return d


def _visible(parents):
    """[nodes][nodes] truth values: node t sees itself and its ancestors."""
    n = len(parents)
    vis = np.zeros((n, n), bool)
    for t in range(n):
        if t:
            vis[t] = vis[parents[t]]
        vis[t, t] = True
    return vis


def _mask_words(vis):
    n = vis.shape[0]
    words = (n + 63) // 64
    bits = np.zeros((n, words * 64), np.uint8)
    bits[:, :n] = vis
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64)


def _rng(case, seed):
    rs = np.random.default_rng([seed, case["nodes"], 977])
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 17)
    return rs, g


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).half()


def _kv_strides(case):
    kvh, P = case["kv_heads"], max(1, case["prefix"])
    if case["layout"] == "head_major":              # [head][row][128]
        return D, P * D
    if case["layout"] == "padded":                  # rows padded beyond the heads
        return kvh * D + 64, D
    return kvh * D, D                               # [row][head][128], the engine's


def _attn_inputs(case, seed):
    rs, g = _rng(case, seed)
    T, P, H, KH = case["nodes"], case["prefix"], case["heads"], case["kv_heads"]
    s = dict(parents=_tree(rs, T, case["chain"]))
    s["q"] = _normal(g, T, H * D, scale=1.5)
    row, head = _kv_strides(case)
    n = max(1, P) * KH * D if head > row else max(1, P) * row
    s["k"], s["v"] = _normal(g, n), _normal(g, n)
    s["kt"], s["vt"] = _normal(g, T, KH * D), _normal(g, T, KH * D)
    s["out"] = torch.empty(T, H * D, dtype=torch.float16, device=DEV)
    return s


def _rope_inputs(case, seed):
    rs, g = _rng(case, seed)
    T, H, KH = case["nodes"], case["heads"], case["kv_heads"]
    s = dict(parents=_tree(rs, T, case["chain"]))
    s["qkv"] = _normal(g, T, (H + 2 * KH) * D)
    s["bias"] = _normal(g, (H + 2 * KH) * D, scale=0.3)
    s["q"] = torch.empty(T, H * D, dtype=torch.float16, device=DEV)
    s["kt"] = torch.empty(T, KH * D, dtype=torch.float16, device=DEV)
    s["vt"] = torch.empty(T, KH * D, dtype=torch.float16, device=DEV)
    s["depth"] = torch.tensor(_depths(s["parents"]), dtype=torch.int32, device=DEV)
    return s


def _verify_inputs(case, seed):
    rs, g = _rng(case, seed)
    T, V = case["nodes"], case["vocab"]
    parents = _tree(rs, T, case["chain"])
    logits = torch.randn(T, V, generator=g, device=DEV) * 2.0
    # a handful of strong candidates in each row
    top = torch.randint(0, V, (T, 6), generator=g, device=DEV)
    logits.scatter_(1, top, 11.0 + 2.0 * torch.randn(T, 6, generator=g, device=DEV))
    logits = logits.half()
    s = dict(parents=parents, logits=logits, draft=None, temperature=0.0 if case["mode"] == "greedy" else 0.8)
    par = torch.tensor([max(0, p) for p in parents], device=DEV)
    if case["mode"] == "drawn":
        s["draft"] = (logits.float() + 0.7 * torch.randn(T, V, generator=g, device=DEV)).half()
        q = torch.softmax(s["draft"].double() / 0.8, 1)
        tok = torch.multinomial(q[par], 1, generator=g)[:, 0]
    else:
        # siblings are their parent's most likely tokens, in order
        seen, rank = {}, []
        for p in parents:
            rank.append(seen.get(p, 0))
            seen[p] = rank[-1] + 1
        order = logits.float().topk(min(V, 8 + max(rank)), dim=1).indices
        tok = order[par, torch.tensor(rank, device=DEV)]
    s["tokens"] = tok.int()
    s["parents_dev"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
    s["accept_u"] = torch.rand(T, generator=g, device=DEV)
    s["sample_u"] = torch.rand(1, generator=g, device=DEV)
    kids = np.bincount([p for p in parents if p >= 0], minlength=1)
    s["max_children"] = int(kids.max())
    s["path"] = torch.empty(T, dtype=torch.int32, device=DEV)
    s["emitted"] = torch.empty(T, dtype=torch.int32, device=DEV)
    s["count"] = torch.empty(1, dtype=torch.int32, device=DEV)
    return s


def _commit_inputs(case, seed):
    rs, g = _rng(case, seed)
    T, H, L, R = case["nodes"], case["heads"], case["layers"], case["rows"]
    s = dict(kc=_normal(g, L, R, H * D), vc=_normal(g, L, R, H * D),
             kt=_normal(g, L, T, H * D), vt=_normal(g, L, T, H * D))
    path = np.full(T, -1, np.int32)
    path[:case["keep"]] = np.concatenate([[0], 1 + np.sort(rs.choice(T - 1, case["keep"] - 1, replace=False))]) \
        if case["keep"] > 1 else [0]
    s["path"] = torch.from_numpy(path).to(DEV)
    s["count"] = torch.tensor([case["keep"]], dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    kind = case["kind"]
    s = {"attn": _attn_inputs, "rope": _rope_inputs, "verify": _verify_inputs, "commit": _commit_inputs}[kind](case, seed)
    s["case"] = case
    if kind == "attn":
        s["mask"] = torch.from_numpy(_mask_words(_visible(s["parents"]))).to(DEV)
        s["visible"] = torch.from_numpy(_visible(s["parents"])).to(DEV)
        s["strides"] = _kv_strides(case)
    if own:
        qdiy = _qdiy()
        s["qdiy"] = qdiy
        if kind == "verify":
            n = qdiy.tree_verify_workspace_bytes(case["nodes"], case["vocab"], s["max_children"])
            s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
        else:
            row, head = s["strides"] if kind == "attn" else (case.get("kv_heads", case["heads"]) * D, D)
            rows = case["rows"] if kind == "commit" else case["prefix"] + case["nodes"]
            s["ctx"] = qdiy.Context(num_heads=case.get("kv_heads", case["heads"]), max_seqlen=rows,
                                    kv_row_stride=row, kv_head_stride=head, rope_base=ROPE_BASE)
            if kind == "attn":
                n = s["ctx"].tree_attention_workspace_bytes(case["nodes"], case["heads"])
                s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attn": _own_attn, "rope": _own_rope, "verify": _own_verify, "commit": _own_commit}[kind](s)
    return {"attn": _plain_attn, "rope": _plain_rope, "verify": _plain_verify, "commit": _plain_commit}[kind](s)


def _own_attn(s):
    c = s["case"]
    return s["ctx"].tree_attention(s["q"], s["k"], s["v"], s["kt"], s["vt"], s["mask"], s["out"], c["prefix"],
                                   c["nodes"], s["ws"], num_heads=c["heads"])


def _own_rope(s):
    c = s["case"]
    s["ctx"].tree_qkv_rope(s["qkv"], s["bias"], s["depth"], s["q"], s["kt"], s["vt"], c["prefix"], c["nodes"],
                           num_heads=c["heads"])
    return s["q"], s["kt"], s["vt"]


def _own_verify(s):
    c = s["case"]
    s["qdiy"].tree_verify(s["logits"], s["tokens"], s["parents_dev"], c["nodes"], c["vocab"], s["ws"], s["path"],
                          s["emitted"], s["count"], temperature=s["temperature"], accept_u=s["accept_u"],
                          sample_u=s["sample_u"], draft_logits=s["draft"], max_children=s["max_children"])
    return s["path"], s["emitted"], s["count"]


def _own_commit(s):
    c = s["case"]
    s["ctx"].tree_commit(s["kt"], s["vt"], s["kc"], s["vc"], s["path"], s["count"], c["prefix"], c["nodes"],
                         layers=c["layers"])
    return s["kc"], s["vc"]


def _rows(flat, case, strides):
    """The cached rows as [kv_heads][prefix][128]."""
    P, KH = case["prefix"], case["kv_heads"]
    return torch.as_strided(flat, (KH, P, D), (strides[1], strides[0], 1))


def _tree_rows(t, case):
    return t.view(case["nodes"], case["kv_heads"], D).transpose(0, 1)


def _plain_attn(s):
    c = s["case"]
    T, P, H, KH = c["nodes"], c["prefix"], c["heads"], c["kv_heads"]
    G = H // KH
    K = torch.cat([_rows(s["k"], c, s["strides"]), _tree_rows(s["kt"], c)], 1).float()
    V = torch.cat([_rows(s["v"], c, s["strides"]), _tree_rows(s["vt"], c)], 1).float()
    q = s["q"].view(T, KH, G, D).permute(1, 2, 0, 3).reshape(KH, G * T, D).float()
    a = torch.matmul(q, K.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
    a = a.view(KH, G, T, P + T)
    a[..., P:] = a[..., P:].masked_fill(~s["visible"], float("-inf"))
    a = torch.exp(a - a.amax(-1, keepdim=True))
    a = (a / a.sum(-1, keepdim=True)).view(KH, G * T, P + T)
    o = torch.matmul(a, V).view(KH, G, T, D).permute(2, 0, 1, 3).reshape(T, H * D)
    s["out"].copy_(o)
    return s["out"]


def _inv_freq():
    # the angle of pair i at position p is fl32(p * fl32(base^(-2i/128))), as in a decode step
    return (ROPE_BASE ** (-2.0 * np.arange(D // 2) / D)).astype(np.float32)


def _plain_rope(s):
    c = s["case"]
    T, H, KH = c["nodes"], c["heads"], c["kv_heads"]
    x = (s["qkv"].float() + s["bias"].float()).half().float().view(T, H + 2 * KH, D)
    inv = torch.from_numpy(_inv_freq()).to(DEV)
    th = ((c["prefix"] + s["depth"]).float()[:, None] * inv[None, :]).double()
    cs, sn = torch.cos(th).float()[:, None, :], torch.sin(th).float()[:, None, :]
    r = x[:, :H + KH]
    r = torch.cat([r[..., :64] * cs - r[..., 64:] * sn, r[..., 64:] * cs + r[..., :64] * sn], -1)
    s["q"].copy_(r[:, :H].reshape(T, H * D))
    s["kt"].copy_(r[:, H:].reshape(T, KH * D))
    s["vt"].copy_(x[:, H + KH:].reshape(T, KH * D))
    return s["q"], s["kt"], s["vt"]


def _weights(logits, temperature):
    x = logits.double()
    m = x.amax(-1, keepdim=True)
    return torch.exp((x - m) / temperature)


def _plain_verify(s):
    """The nodes in index order: a node below the current one is tested; accepted, it becomes
    the current one.  The current node's remaining distribution is r (not normalised)."""
    c = s["case"]
    T, V = c["nodes"], c["vocab"]
    tok, par, u = s["tokens"].long(), s["parents_dev"], s["accept_u"].double()
    cur = torch.zeros(1, dtype=torch.int32, device=DEV)
    path = torch.full((T + 1,), -1, dtype=torch.int32, device=DEV)
    emitted = torch.full((T + 1,), -1, dtype=torch.int32, device=DEV)
    count = torch.ones(1, dtype=torch.int32, device=DEV)
    path[0] = 0
    ids = torch.arange(V, device=DEV)
    greedy = c["mode"] == "greedy"
    if greedy:
        m = s["logits"].amax(-1, keepdim=True)
        best = torch.where(s["logits"] == m, ids, V).amin(-1)
    else:
        p = _weights(s["logits"], s["temperature"])
        p = p / p.sum(-1, keepdim=True)
        r = p[0]
        if c["mode"] == "drawn":
            q = _weights(s["draft"], s["temperature"])
            q = q / q.sum(-1, keepdim=True)
            qc = q[0]
    for t in range(1, T):
        child = par[t:t + 1] == cur
        x = tok[t:t + 1]
        if greedy:
            ok = child & (best[cur.long()] == x)
        elif c["mode"] == "point":
            ok = child & (u[t] * r.sum() < r[x])
            rest = torch.where(ids == x, 0.0, r)
            r = torch.where(ok, p[t], torch.where(child, rest, r))
        else:
            ok = child & (u[t] * qc[x] < r[x])
            rest = (r - qc).clamp_min(0.0)
            rest = rest / rest.sum()
            r = torch.where(ok, p[t], torch.where(child, rest, r))
            qc = torch.where(ok, q[t], qc)
        at = torch.where(ok, count, T).long()
        path.scatter_(0, at, torch.full_like(cur, t))
        emitted.scatter_(0, torch.where(ok, count - 1, T).long(), x.int())
        cur = torch.where(ok, torch.full_like(cur, t), cur)
        count = count + ok.int()
    if greedy:
        last = best[cur.long()]
    else:
        cum = torch.cumsum(r, 0)
        last = torch.searchsorted(cum, s["sample_u"].double() * cum[-1:], right=True).clamp_max(V - 1)
    emitted.scatter_(0, (count - 1).long(), last.int())
    s["path"].copy_(path[:T])
    s["emitted"].copy_(emitted[:T])
    s["count"].copy_(count)
    return s["path"], s["emitted"], s["count"]


def _plain_commit(s):
    c = s["case"]
    T, P = c["nodes"], c["prefix"]
    i = torch.arange(T, device=DEV)
    live = i < s["count"]
    src = torch.where(live, s["path"], 0).long()
    for cache, tree in ((s["kc"], s["kt"]), (s["vc"], s["vt"])):
        cache[:, P:P + T] = torch.where(live[None, :, None], tree[:, src], cache[:, P:P + T])
    return s["kc"], s["vc"]


# ------------------------------------------------------------------ work and the definition in 64 bits

def work(case):
    T = case["nodes"]
    if case["kind"] == "attn":
        H, KH, n = case["heads"], case["kv_heads"], case["prefix"] + T
        return {"bytes": 2 * n * KH * D * 2 + 2 * T * H * D * 2 + T * ((T + 63) // 64) * 8,
                "flops": 4 * T * H * n * D}
    if case["kind"] == "rope":
        w = (case["heads"] + 2 * case["kv_heads"]) * D
        return {"bytes": 2 * T * w * 2 + w * 2 + T * 4, "flops": 7 * T * w}
    if case["kind"] == "verify":
        n = T * case["vocab"] * (2 if case["mode"] == "drawn" else 1)
        return {"bytes": 2 * n + 24 * T, "flops": n * (1 if case["mode"] == "greedy" else 3)}
    return {"bytes": 2 * 2 * case["layers"] * case["keep"] * case["heads"] * D * 2, "flops": 0}


def exact(case, seed):
    return {"attn": _exact_attn, "rope": _exact_rope, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](case, seed)


def _exact_attn(case, seed):
    s = _attn_inputs(case, seed)
    T, P, H, KH = case["nodes"], case["prefix"], case["heads"], case["kv_heads"]
    G = H // KH
    row, head = _kv_strides(case)
    rows = torch.arange(P, device=DEV)[:, None] * row + torch.arange(D, device=DEV)[None, :]
    hidden = torch.zeros(T, P + T, dtype=torch.float64, device=DEV)
    for t in range(T):
        hidden[t, P:] = -math.inf
        a = t
        while a >= 0:
            hidden[t, P + a] = 0.0
            a = s["parents"][a]
    out = torch.empty(T, H, D, dtype=torch.float64, device=DEV)
    for h in range(H):
        kh = h // G
        K = torch.cat([s["k"][rows + kh * head], s["kt"][:, kh * D:(kh + 1) * D]]).double()
        V = torch.cat([s["v"][rows + kh * head], s["vt"][:, kh * D:(kh + 1) * D]]).double()
        z = torch.mm(s["q"][:, h * D:(h + 1) * D].double(), K.t().contiguous()) / math.sqrt(D) + hidden
        out[:, h] = torch.mm(torch.softmax(z, 1), V)
    return out.view(T, H * D)


def _exact_rope(case, seed):
    s = _rope_inputs(case, seed)
    T, H, KH = case["nodes"], case["heads"], case["kv_heads"]
    # the biased row is stored in half precision, by definition
    x = (s["qkv"].float() + s["bias"].float()).half().double().cpu().numpy().reshape(T, H + 2 * KH, 2, 64)
    pos = np.float32(case["prefix"]) + np.array(_depths(s["parents"]), np.float32)
    th = (pos[:, None] * _inv_freq()[None, :]).astype(np.float64)[:, None, :]
    out = x.copy()
    out[:, :H + KH, 0] = x[:, :H + KH, 0] * np.cos(th) - x[:, :H + KH, 1] * np.sin(th)
    out[:, :H + KH, 1] = x[:, :H + KH, 1] * np.cos(th) + x[:, :H + KH, 0] * np.sin(th)
    out = torch.from_numpy(out.reshape(T, (H + 2 * KH) * D)).to(DEV)
    return out[:, :H * D], out[:, H * D:(H + KH) * D], out[:, (H + KH) * D:]


def _exact_verify(case, seed):
    """A walk on the host over the rows that it visits."""
    s = _verify_inputs(case, seed)
    T = case["nodes"]
    tok, u = s["tokens"].tolist(), s["accept_u"].double().tolist()
    kids = [[c for c in range(1, T) if s["parents"][c] == t] for t in range(T)]

    def row(x, t):
        z = x[t].cpu().numpy().astype(np.float64)
        if case["mode"] == "greedy":
            return z
        z = np.exp((z - z.max()) / s["temperature"])
        return z / math.fsum(z)

    node, path, out = 0, [0], []
    while True:
        p = row(s["logits"], node)
        q = row(s["draft"], node) if case["mode"] == "drawn" and kids[node] else None
        taken = None
        for c in kids[node]:
            if case["mode"] == "greedy":
                good = tok[c] == int(np.argmax(p))
            elif case["mode"] == "point":
                good = u[c] * math.fsum(p) < p[tok[c]]
                if not good:
                    p[tok[c]] = 0.0
            else:
                good = u[c] * q[tok[c]] < p[tok[c]]
                if not good:
                    p = np.maximum(p - q, 0.0)
                    p /= math.fsum(p)
            if good:
                taken = c
                break
        if taken is None:
            break
        node = taken
        path.append(node)
        out.append(tok[node])
    if case["mode"] == "greedy":
        out.append(int(np.argmax(p)))
    else:
        cum = np.cumsum(p)
        out.append(min(int(np.searchsorted(cum, float(s["sample_u"][0]) * cum[-1], side="right")), case["vocab"] - 1))
    pad = [-1] * (T - len(path))
    mk = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    return mk(path + pad), mk(out + pad), mk([len(path)])


def _exact_commit(case, seed):
    s = _commit_inputs(case, seed)
    res = []
    for cache, tree in ((s["kc"], s["kt"]), (s["vc"], s["vt"])):
        for i, t in enumerate(s["path"].tolist()[:case["keep"]]):
            cache[:, case["prefix"] + i] = tree[:, t]
        res.append(cache.double())
    return tuple(res)
