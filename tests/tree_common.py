"""Float64 references and inputs of the drafted-token tree tests."""
import math

import numpy as np

D = 128


def random_parents(rng, nodes, reach=8):
    return [-1] + [int(rng.integers(max(0, t - reach), t)) for t in range(1, nodes)]


def chain_parents(nodes):
    return [-1] + list(range(nodes - 1))


def ancestors(parents):
    """[nodes][nodes] truth values: node t sees itself and the nodes above it."""
    n = len(parents)
    vis = np.zeros((n, n), bool)
    for t in range(n):
        a = t
        while a >= 0:
            vis[t, a] = True
            a = parents[a]
    return vis


def depths(parents):
    d = []
    for t, p in enumerate(parents):
        d.append(0 if t == 0 else d[p] + 1)
    return d


def mask_words(vis):
    n = vis.shape[0]
    words = (n + 63) // 64
    out = np.zeros((n, words), np.uint64)
    for t in range(n):
        for j in np.flatnonzero(vis[t]):
            out[t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def attention(q, K, V, Kt, Vt, vis, with_bound=False):
    """q [T,H,128], K/V [P,KH,128], Kt/Vt [T,KH,128], vis [T,T] -> out [T,H,128] float64;
    zeros for a node that sees no row.

    The bound (per output) of the kernel's arithmetic, from its roundings alone:
      fp16 output                     2^-11 |out|  (2^-25 in the subnormal range)
      weights rounded to fp16         2^-11 each, in the numerator and in the sum they are
                                      divided by: 2 * 2^-11 * A,  A = sum w |V| / sum w
      fp16 weights below 2^-14        2^-25 each:  2^-25 * sum |V| / sum w,  w relative to
                                      the largest score (sum w >= 1), both sums again
      fp32 scores                     a sum of 128 products is off by at most
                                      128 * 2^-24 * sum |q k| / sqrt(128); that and the
                                      exponential's few fp32 steps scale a weight by
                                      e^delta: 2 delta A,  delta = that + 2^-19 (scores up
                                      to 2^4 in size, exp2 argument rounded to 2^-24 each)
      fp32 sums of the products       n * 2^-24 * A at most."""
    T, H, _ = q.shape
    KH = Kt.shape[1]
    G = H // KH
    out = np.zeros((T, H, D))
    bound = np.zeros((T, H, D))
    for h in range(H):
        k = np.concatenate([K[:, h // G], Kt[:, h // G]]).astype(np.float64)
        v = np.concatenate([V[:, h // G], Vt[:, h // G]]).astype(np.float64)
        for t in range(T):
            see = np.concatenate([np.ones(K.shape[0], bool), vis[t]])
            if not see.any():
                continue
            ks, vs, x = k[see], v[see], q[t, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = ks @ x / math.sqrt(D)
                w = np.exp(s - s.max())
                out[t, h] = w @ vs / w.sum()
            if with_bound:
                A = w @ np.abs(vs) / w.sum()
                delta = 128 * 2.0 ** -24 * (np.abs(ks) @ np.abs(x)).max() / math.sqrt(D) + 2.0 ** -19
                small = 2.0 ** -25 * (np.abs(vs).sum(0) + len(vs) * A) / w.sum()
                bound[t, h] = (2.0 ** -11 * np.abs(out[t, h]) + 2.0 ** -25 + small
                               + (2 * 2.0 ** -11 + 2 * delta + len(vs) * 2.0 ** -24) * A)
    return (out, bound) if with_bound else out


def softmax64(row, temperature):
    x = row.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    m = x.max()
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / temperature))
    return w / w.sum()


def verify(logits, tokens, parents, mode, temperature=1.0, accept_u=None, sample_u=0.0, draft=None,
           max_children=64):
    """The walk of qd_tree_verify in float64: (path, emitted)."""
    T, V = logits.shape
    kids = [[c for c in range(t + 1, T) if parents[c] == t] for t in range(T)]
    node, path, out = 0, [0], []

    def best(row):
        x = row.astype(np.float64)
        x[np.isnan(x)] = -np.inf
        ok = ~np.isnan(row)
        return int(np.flatnonzero(ok & (x == x.max()))[0]) if ok.any() else 0

    while True:
        if mode != "greedy":
            p = softmax64(logits[node], temperature)
            if mode == "drawn" and kids[node]:
                q = softmax64(draft[node], temperature)
        taken = None
        for n, c in enumerate(kids[node]):
            if mode == "drawn" and n == max_children:
                break
            x = int(tokens[c])
            inside = 0 <= x < V
            if mode == "greedy":
                ok = x == best(logits[node])
            elif mode == "point":
                w = p[x] if inside else 0.0
                ok = float(accept_u[c]) * p.sum() < w
                if not ok and inside:
                    p[x] = 0.0
            else:
                pw, qw = (p[x], q[x]) if inside else (0.0, 0.0)
                ok = float(accept_u[c]) * qw < pw
                if not ok:
                    r = np.maximum(p - q, 0.0)
                    if r.sum() > 0.0:
                        p = r / r.sum()
            if ok:
                taken = c
                break
        if taken is None:
            break
        node = taken
        path.append(node)
        out.append(int(tokens[node]))
    if mode == "greedy":
        out.append(best(logits[node]))
    else:
        cum = np.cumsum(p)
        hit = np.flatnonzero((cum > float(sample_u) * cum[-1]) & (p > 0))
        out.append(int(hit[0]) if len(hit) else (int(np.flatnonzero(p > 0)[-1]) if (p > 0).any() else 0))
    return path, out
