"""GPU parity of qd_tree_qkv_rope (bits of qd_qkv_bias_rope_cache) and qd_tree_commit, and one
whole speculative step of all four tree operators."""
import numpy as np
import pytest
import torch

from common import normal_f16
from tree_common import (D, ancestors, attention, chain_parents, depths, mask_words, random_parents, verify)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qdiy():
    import qdiy as m
    torch.cuda.set_device(0)
    m.load()
    return m


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


def same(a, b):
    return np.array_equal(np.asarray(a).view(np.uint16), np.asarray(b).view(np.uint16))


# ------------------------------------------------------------------ RoPE rows

@pytest.mark.parametrize("H", [1, 4, 16])
@pytest.mark.parametrize("T,P", [(1, 0), (5, 3), (33, 100), (70, 929)])
@pytest.mark.parametrize("bias", [True, False])
def test_rope_has_the_decode_steps_bits(qdiy, H, T, P, bias):
    rng = np.random.default_rng(T + P)
    S = P + T
    ctx = qdiy.Context(num_heads=H, max_seqlen=S)
    qkv, b = dev(normal_f16(rng, (T, 3 * H * D))), dev(normal_f16(rng, 3 * H * D)) if bias else None
    before = host(qkv).copy()
    depth = depths(random_parents(rng, T))
    q, k, v = (torch.full((T + 1, H * D), 9.0, dtype=torch.float16, device="cuda") for _ in range(3))
    ctx.tree_qkv_rope(qkv, b, dev(np.array(depth, np.int32)), q, k, v, P, T)
    assert same(host(qkv), before)
    kc, vc = (torch.zeros(S * H * D, dtype=torch.float16, device="cuda") for _ in range(2))
    for t in range(T):
        one, pos = qkv[t].clone(), P + depth[t]
        ctx.qkv_bias_rope_cache(one, b, kc, vc, pos)
        assert same(host(q[t]), host(one[:H * D]))
        assert same(host(k[t]), host(kc[pos * H * D:(pos + 1) * H * D]))
        assert same(host(v[t]), host(vc[pos * H * D:(pos + 1) * H * D]))
    for x in (q, k, v):
        assert np.all(host(x[T]) == 9.0)


@pytest.mark.parametrize("H,KH", [(8, 2), (7, 1), (28, 4)])
@pytest.mark.parametrize("layout", ["packed", "padded", "head_major"])
def test_rope_grouped_heads_and_strides(qdiy, H, KH, layout):
    """Against the rotation in float64 with the table's own fp32 angles: the products and their
    sum round to fp32 (3 * 2^-24 of |x1| + |x2|), the result to fp16; cos and sin are within
    2^-23 of the fp32 angle's."""
    rng = np.random.default_rng(H)
    T, P = 19, 40
    ctx = qdiy.Context(num_heads=KH, max_seqlen=200)
    W = H + 2 * KH
    x, b = normal_f16(rng, (T, W, D)), normal_f16(rng, (W, D))
    depth = np.array(depths(random_parents(rng, T)), np.int32)
    pad = 0 if layout == "packed" else 72
    trow, thead = (KH * D + pad, D) if layout != "head_major" else (D, T * D)
    buf = np.full((T, W * D + pad), np.nan, np.float16)
    buf[:, :W * D] = x.reshape(T, -1)
    q = torch.full((T, H * D + pad), 9.0, dtype=torch.float16, device="cuda")
    n = (T - 1) * trow + (KH - 1) * thead + D
    k, v = (torch.full((n,), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.tree_qkv_rope(dev(buf), dev(b.reshape(-1)), dev(depth), q, k, v, P, T, num_heads=H, qkv_stride=W * D + pad,
                      q_stride=H * D + pad, tree_row_stride=trow, tree_head_stride=thead)
    y = (x.astype(np.float32) + b.astype(np.float32)).astype(np.float16).astype(np.float64)
    inv = (10000.0 ** (-2.0 * np.arange(64) / D)).astype(np.float32)
    th = ((P + depth).astype(np.float32)[:, None] * inv).astype(np.float64)[:, None, :]
    y1, y2 = y[..., :64], y[..., 64:]
    want = np.concatenate([y1 * np.cos(th) - y2 * np.sin(th), y2 * np.cos(th) + y1 * np.sin(th)], -1)
    size = np.concatenate([np.abs(y1) + np.abs(y2)] * 2, -1)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (3 * 2.0 ** -24 + 2 * 2.0 ** -23) * size
    gq = host(q)
    assert np.all(gq[:, H * D:] == 9.0)
    gk = np.stack([[host(k)[t * trow + h * thead:][:D] for h in range(KH)] for t in range(T)])
    gv = np.stack([[host(v)[t * trow + h * thead:][:D] for h in range(KH)] for t in range(T)])
    assert np.all(np.abs(gq[:, :H * D].reshape(T, H, D) - want[:, :H]) <= tol[:, :H])
    assert np.all(np.abs(gk - want[:, H:H + KH]) <= tol[:, H:H + KH])
    assert np.array_equal(gv.astype(np.float64), y[:, H + KH:])


def test_rope_in_place_and_positions_outside(qdiy):
    rng = np.random.default_rng(0)
    H, T = 4, 6
    ctx = qdiy.Context(num_heads=H, max_seqlen=50)
    x = dev(normal_f16(rng, (T, 3 * H * D)))
    depth = dev(np.array([0, 1, -1, 3, 60, 2 ** 31 - 1], np.int32))
    outs = [[torch.empty(T, H * D, dtype=torch.float16, device="cuda") for _ in range(3)] for _ in range(2)]
    ctx.tree_qkv_rope(x, None, depth, *outs[0], 46, T)
    y = x.clone()
    ctx.tree_qkv_rope(y, None, depth, y, outs[1][1], outs[1][2], 46, T, q_stride=3 * H * D)
    assert same(host(y)[:, :H * D], host(outs[0][0]))
    assert same(host(y)[:, H * D:], host(x)[:, H * D:])
    assert same(host(outs[1][1]), host(outs[0][1])) and same(host(outs[1][2]), host(outs[0][2]))
    bad = np.isnan(np.concatenate([host(o) for o in outs[0]], 1))
    assert bad[[2, 4, 5]].all() and not bad[[0, 1, 3]].any()      # 46 + 3 is the last row


def test_rope_refusals(qdiy):
    H, KH, T = 4, 2, 3
    ctx = qdiy.Context(num_heads=KH, max_seqlen=50)
    x = torch.zeros(T, (H + 2 * KH) * D, dtype=torch.float16, device="cuda")
    bias = torch.zeros((H + 2 * KH) * D, dtype=torch.float16, device="cuda")
    q, k, v = (torch.zeros(T, H * D, dtype=torch.float16, device="cuda") for _ in range(3))
    depth = torch.zeros(T + 1, dtype=torch.int32, device="cuda")
    lib = qdiy.load()
    W = (H + 2 * KH) * D
    good = dict(x=x.data_ptr(), xs=W, b=bias.data_ptr(), d=depth.data_ptr(), q=q.data_ptr(), qs=H * D, k=k.data_ptr(),
                v=v.data_ptr(), trow=KH * D, thead=D, P=5, T=T, H=H, hd=128)

    def call(**kw):
        a = dict(good, **kw)
        return lib.qd_tree_qkv_rope(ctx._h, a["x"], a["xs"], a["b"], a["d"], a["q"], a["qs"], a["k"], a["v"],
                                    a["trow"], a["thead"], a["P"], a["T"], a["H"], a["hd"], None)

    bad = [dict(T=0), dict(T=1025), dict(P=-1), dict(P=51), dict(H=3), dict(H=0), dict(hd=64), dict(xs=W - 8),
           dict(xs=W + 4), dict(qs=H * D - 8), dict(trow=0), dict(thead=4), dict(d=good["d"] + 2)]
    bad += [{n: None} for n in ("x", "d", "q", "k", "v")] + [{n: good[n] + 2} for n in ("x", "b", "q", "k", "v")]
    bad += [dict(k=good["x"]), dict(v=good["b"]), dict(k=good["q"]), dict(q=good["x"]), dict(q=good["b"])]
    for kw in bad:
        assert call(**kw) == qdiy.QD_EINVAL, kw
    assert call() == qdiy.QD_OK and call(b=None) == qdiy.QD_OK
    torch.cuda.synchronize()
    with pytest.raises(TypeError):
        ctx.tree_qkv_rope(x, bias, depth.float(), q, k, v, 5, T, num_heads=H)
    with pytest.raises(ValueError):
        ctx.tree_qkv_rope(x, bias, depth, q, k, v, 5, T, num_heads=H, qkv_stride=2 * W)


# ------------------------------------------------------------------ committing a path

def commit_inputs(qdiy, H, L, S, T, seed, layout="engine"):
    rng = np.random.default_rng(seed)
    row, head = (H * D, D) if layout == "engine" else (D, S * D)
    ctx = qdiy.Context(num_heads=H, max_seqlen=S, kv_row_stride=row, kv_head_stride=head)
    caches = [normal_f16(rng, (L, S, H, D)) for _ in range(2)]
    trees = [normal_f16(rng, (L, T, H, D)) for _ in range(2)]
    return rng, ctx, caches, trees


def lay(x, layout):
    return dev(x if layout == "engine" else x.transpose(0, 2, 1, 3))


@pytest.mark.parametrize("layout", ["engine", "head_major"])
@pytest.mark.parametrize("H,L,T,n", [(1, 1, 1, 1), (4, 3, 27, 4), (2, 2, 64, 64), (16, 2, 20, 9), (3, 5, 130, 17)])
def test_commit(qdiy, H, L, T, n, layout):
    S, P = 200, 21
    rng, ctx, caches, trees = commit_inputs(qdiy, H, L, S, T, H + T, layout)
    path = np.full(T, -1, np.int32)
    path[:n] = np.sort(rng.choice(T, n, replace=False))
    gc, gt = [lay(c, layout) for c in caches], [lay(t, layout) for t in trees]
    kw = {} if layout == "engine" else dict(tree_row_stride=D, tree_head_stride=T * D)
    ctx.tree_commit(gt[0], gt[1], gc[0], gc[1], dev(path), dev(np.array([n], np.int32)), P, T, layers=L, **kw)
    for c, t, g in zip(caches, trees, gc):
        c[:, P:P + n] = t[:, path[:n]]
        g = host(g) if layout == "engine" else host(g).transpose(0, 2, 1, 3)
        assert same(np.ascontiguousarray(g).reshape(-1), c.reshape(-1))


@pytest.mark.parametrize("T,path", [(5, [0]), (9, [0, 1, 2, 3]), (9, [0, 2, 3, 8]), (40, list(range(0, 40, 2))),
                                    (40, list(range(40))), (64, [0] + list(range(25, 64))), (3, [2])])
def test_commit_in_place(qdiy, T, path):
    """The node rows are the cache's own behind the prefix."""
    H, L, S, P = 4, 3, 120, 30
    _, ctx, caches, _ = commit_inputs(qdiy, H, L, S, T, T)
    full = np.full(T, -1, np.int32)
    full[:len(path)] = path
    gk, gv = dev(caches[0]), dev(caches[1])
    ctx.tree_commit(gk.view(-1)[P * H * D:], gv.view(-1)[P * H * D:], gk, gv, dev(full),
                    dev(np.array([len(path)], np.int32)), P, T, layers=L, tree_layer_stride=S * H * D)
    for c, g in zip(caches, (gk, gv)):
        c[:, P:P + len(path)] = c[:, P:][:, path].copy()
        assert same(host(g), c)


def test_commit_skips_what_it_cannot_place(qdiy):
    """Entries outside the nodes, rows past the cache, counts beyond the nodes or below zero."""
    H, L, S, T = 2, 2, 40, 12
    for P, n, path in ((35, 12, list(range(12))), (10, 12, [0, -3, 12, 5, 2 ** 31 - 1, -2 ** 31, 11, 1, 2, 3, 4, 6]),
                       (10, 400, list(range(12))), (10, -5, list(range(12))), (10, 0, list(range(12))),
                       (40, 12, list(range(12)))):
        _, ctx, caches, trees = commit_inputs(qdiy, H, L, S, T, 3)
        gc, gt = [dev(c) for c in caches], [dev(t) for t in trees]
        ctx.tree_commit(gt[0], gt[1], gc[0], gc[1], dev(np.array(path, np.int32)), dev(np.array([n], np.int32)), P, T,
                        layers=L)
        for c, t, g in zip(caches, trees, gc):
            for i, x in enumerate(path[:max(0, n)]):
                if 0 <= x < T and P + i < S:
                    c[:, P + i] = t[:, x]
            assert same(host(g), c)


def test_commit_refusals(qdiy):
    H, L, S, T, P = 2, 3, 40, 5, 10
    _, ctx, caches, trees = commit_inputs(qdiy, H, L, S, T, 3)
    gc, gt = [dev(c) for c in caches], [dev(t) for t in trees]
    path, count = dev(np.zeros(T, np.int32)), dev(np.zeros(1, np.int32))
    lib = qdiy.load()
    good = dict(kt=gt[0].data_ptr(), vt=gt[1].data_ptr(), tl=T * H * D, tr=H * D, th=D, kc=gc[0].data_ptr(),
                vc=gc[1].data_ptr(), cl=S * H * D, path=path.data_ptr(), count=count.data_ptr(), P=P, T=T, L=L)

    def call(**kw):
        a = dict(good, **kw)
        return lib.qd_tree_commit(ctx._h, a["kt"], a["vt"], a["tl"], a["tr"], a["th"], a["kc"], a["vc"], a["cl"],
                                  a["path"], a["count"], a["P"], a["T"], a["L"], None)

    at = P * H * D * 2
    bad = [dict(T=0), dict(T=1025), dict(L=0), dict(L=5000), dict(P=-1), dict(P=41), dict(tl=4), dict(tl=0), dict(cl=0),
           dict(tr=0), dict(th=3), dict(path=good["path"] + 2), dict(count=good["count"] + 1),
           dict(kt=good["kc"] + at), dict(kt=good["kc"] + at, vt=good["vc"] + at),      # another layer stride
           dict(kt=good["kc"] + at + 256, vt=good["vc"] + at + 256, tl=good["cl"]),     # not from the prefix on
           dict(kt=good["vc"]), dict(path=good["kc"]), dict(count=good["vc"])]
    bad += [{n: None} for n in ("kt", "vt", "kc", "vc", "path", "count")]
    bad += [{n: good[n] + 8} for n in ("kt", "vt", "kc", "vc")]
    bad += [dict(kt=good["kc"] + (S - 4) * H * D * 2, vt=good["vc"] + (S - 4) * H * D * 2, tl=good["cl"], P=S - 4)]
    for kw in bad:
        assert call(**kw) == qdiy.QD_EINVAL, kw
    assert call() == qdiy.QD_OK
    assert call(kt=good["kc"] + at, vt=good["vc"] + at, tl=good["cl"]) == qdiy.QD_OK
    torch.cuda.synchronize()


# ------------------------------------------------------------------ a whole step

@pytest.mark.parametrize("mode", ["greedy", "point"])
def test_a_speculative_step(qdiy, mode):
    """Two layers of attention over a cache (their Q/K/V rows given), logits from the second
    layer's output, verification and commit, captured as one graph and replayed over three
    steps of a growing cache held by its own inputs; then the committed rows serve a decode
    step.  The float64 walk gets the GPU's own logits; the attention of each layer is within
    its bound; the cache rows have the bits that a token by token decode would write."""
    H, L, V, T, S, P = 4, 2, 611, 23, 160, 70
    row = H * D
    rng = np.random.default_rng(17)
    ctx = qdiy.Context(num_heads=H, max_seqlen=S)
    kc, vc = (dev(normal_f16(rng, (L, S, row))) for _ in range(2))
    kt, vt = (torch.empty(L, T, row, dtype=torch.float16, device="cuda") for _ in range(2))
    parents = random_parents(rng, T, 4)
    mask, depth = qdiy.tree_layout(parents)
    mask, depth_d = mask.cuda(), depth.cuda()
    qkv = torch.empty(L, T, 3 * row, dtype=torch.float16, device="cuda")
    q, out = (torch.empty(L, T, row, dtype=torch.float16, device="cuda") for _ in range(2))
    head = dev(normal_f16(rng, (V, row), 0.3))
    logits = torch.empty(T, V, dtype=torch.float16, device="cuda")
    tokens, par = torch.zeros(T, dtype=torch.int32, device="cuda"), dev(np.array(parents, np.int32))
    au, su = torch.empty(T, device="cuda"), torch.empty(1, device="cuda")
    path, emitted = (torch.empty(T, dtype=torch.int32, device="cuda") for _ in range(2))
    count = torch.empty(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(ctx.tree_attention_workspace_bytes(T), qdiy.tree_verify_workspace_bytes(T, V)),
                     dtype=torch.uint8, device="cuda")
    temp = 0.0 if mode == "greedy" else 0.9

    def step(prefix):
        for l in range(L):
            ctx.tree_qkv_rope(qkv[l], None, depth_d, q[l], kt[l], vt[l], prefix, T)
            ctx.tree_attention(q[l], kc[l], vc[l], kt[l], vt[l], mask, out[l], prefix, T, ws)
        qdiy.gemm_nt(out[L - 1], head, logits, T, V, row)
        qdiy.tree_verify(logits, tokens, par, T, V, ws, path, emitted, count, temperature=temp, accept_u=au,
                         sample_u=su)
        ctx.tree_commit(kt, vt, kc, vc, path, count, prefix, T, layers=L)

    graphs = {}
    prefix = P
    accepted = 0
    for i in range(3):
        x = normal_f16(rng, (L, T, 3 * row))
        qkv.copy_(dev(x))
        au.copy_(dev(rng.random(T, dtype=np.float32) * 0.3))
        su.copy_(dev(rng.random(1, dtype=np.float32)))
        before = [host(kc).copy(), host(vc).copy()]
        # drafts: the most likely tokens after each node, from a first eager pass over a copy
        tokens.zero_()
        step(prefix)
        kc.copy_(dev(before[0]))
        vc.copy_(dev(before[1]))
        lg = host(logits).astype(np.float64)
        rank, tok = {}, np.zeros(T, np.int32)
        for t in range(1, T):
            p = parents[t]
            tok[t] = np.argsort(-lg[p], kind="stable")[rank.get(p, 0)]
            rank[p] = rank.get(p, 0) + 1
        tokens.copy_(dev(tok))
        torch.cuda.synchronize()
        g = graphs[prefix] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(prefix)
        g.replay()
        torch.cuda.synchronize()
        n = int(count)
        want = verify(host(logits), tok, parents, mode, temp, host(au), host(su)[0])
        assert (host(path)[:n].tolist(), host(emitted)[:n].tolist()) == want
        accepted += n - 1
        for l in range(L):
            K, Vv = (b[l, :prefix].reshape(prefix, H, D) for b in before)
            ref, bound = attention(host(q[l]).reshape(T, H, D), K, Vv, host(kt[l]).reshape(T, H, D),
                                   host(vt[l]).reshape(T, H, D), ancestors(parents), with_bound=True)
            assert np.all(np.abs(host(out[l]).reshape(T, H, D) - ref) <= bound)
            # token by token: the same rows
            k1, v1 = dev(before[0][l]), dev(before[1][l])
            for j, t in enumerate(want[0]):
                ctx.qkv_bias_rope_cache(dev(x[l, t]), None, k1, v1, prefix + j)
            assert same(host(kc[l]), host(k1)) and same(host(vc[l]), host(v1))
        prefix += n
    assert accepted > 0
