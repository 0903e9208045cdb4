"""What the tree calls promise beyond their results on whole inputs: memory that need not be
there, infinities that are seen, captured calls, long scans in several splits."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import Case as Attention
from test_gpu_tree_verify import Case as Verify, dev
from tree_common import ancestors, attention, chain_parents, verify
from tree_plan import attention_plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qdiy():
    import qdiy as m
    torch.cuda.set_device(0)
    m.load()
    return m


# ------------------------------------------------------------------ verification

@pytest.mark.parametrize("parents", [[-1], [-1, 0, 0, 0], [-1, 0, 1, 0, 1, 2, 2, 5, 5, 5]])
@pytest.mark.parametrize("V", [40, 9001])
def test_draft_rows_of_leaves_need_not_be_there(qdiy, parents, V):
    """The drafter's buffer ends with the last node that has children; the workspace follows it
    at once, in the same allocation."""
    T = len(parents)
    for seed in range(3):
        c = Verify(T, V, "drawn", seed=seed, parents=parents)
        c.upload()
        c.outputs(qdiy)
        inner = 1 + max(parents)
        n = (2 * inner * V + 15) // 16 * 16
        arena = torch.full((n + c.ws.numel(),), 0xFF, dtype=torch.uint8, device="cuda")
        arena[:2 * inner * V].view(torch.float16).copy_(dev(c.draft[:inner].reshape(-1)))
        g, p = c.g, ctypes.c_void_p
        at = lambda t: p(t.data_ptr())
        rc = qdiy.load().qd_tree_verify(
            at(g["target"]), V, p(arena.data_ptr()), V, at(g["tokens"]), at(g["parents"]), at(g["au"]), at(g["su"]),
            c.temperature, T, V, c.max_children, p(arena.data_ptr() + n), c.ws.numel(), at(c.path), at(c.emitted),
            at(c.count), p(torch.cuda.current_stream().cuda_stream))
        assert rc == qdiy.QD_OK
        assert c.got() == c.want()
        # the binding, over a tensor without the last node's row
        c.outputs(qdiy)
        g["draft"] = dev(c.draft[:T - 1])
        c.call(qdiy)
        assert c.got() == c.want()


# ------------------------------------------------------------------ attention: infinities that are seen

def far_below(c, t_far=0):
    """Cache row `t_far` scores some 226 above every other row, whose weights are far below what
    fp32 holds."""
    base = np.where(np.arange(128) % 3 == 0, 1.0, -1.0)
    c.q[:] = base.astype(np.float16)
    c.K[:] = 0.0
    c.Kt[:] = 0.0
    c.K[t_far] = (20.0 * base).astype(np.float16)
    c.gq = dev(c.q.reshape(c.T, -1))


@pytest.mark.parametrize("H,KH,P,T", [(2, 2, 40, 20), (2, 2, 2000, 20), (1, 1, 9000, 3), (2, 1, 3000, 40),
                                      (2, 2, 5000, 100)])
@pytest.mark.parametrize("gap", [False, True])
def test_a_nodes_infinity_reaches_those_that_see_it(qdiy, H, KH, P, T, gap):
    """However small its weight, and whichever of the splits holds it; nothing else changes."""
    vis = ancestors(chain_parents(T))
    vis[:, 1] = False
    vis[1, 1] = vis[T - 1, 1] = True
    c = Attention(qdiy, H, KH, P, T, seed=P + T, vis=vis, kscale=0.2)
    if gap:
        far_below(c)
    c.upload()
    a = c.result().copy()
    assert np.all(np.isfinite(a))
    c.Vt[1, :, 5] = np.inf
    c.Vt[1, :, 77] = -np.inf
    c.Vt[1, :, 126] = np.nan
    c.upload()
    b = c.result().copy()
    see = [1, T - 1]
    assert np.all(b[see][:, :, 5] == np.inf) and np.all(b[see][:, :, 77] == -np.inf)
    assert np.all(np.isnan(b[see][:, :, 126]))
    for d in (5, 77, 126):
        a[see, :, d] = b[see, :, d] = 0
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("H,KH,P,T", [(2, 2, 40, 5), (2, 2, 2000, 20), (1, 1, 9000, 3), (2, 1, 3000, 24),
                                      (2, 2, 5000, 100), (2, 2, 9, 64), (16, 16, 1203, 70)])
@pytest.mark.parametrize("gap", [False, True])
def test_a_cached_infinity_reaches_every_node(qdiy, H, KH, P, T, gap):
    """Cache rows are seen by all, however small their weight: infinities and NaN reach their
    column of every output, and no other column changes."""
    c = Attention(qdiy, H, KH, P, T, seed=P + T, kscale=0.2)
    if gap:
        far_below(c)
    c.upload()
    a = c.result().copy()
    assert np.all(np.isfinite(a))
    far = [1, P // 3, P // 2, P - 2, P - 1]
    for i, (j, bad) in enumerate(zip(far, (np.inf, -np.inf, np.nan, np.inf, -np.inf))):
        c.V[j, :, 20 + 25 * i] = bad
    c.V[1, :, 0] = np.inf
    c.V[P - 1, :, 0] = -np.inf
    c.upload()
    b = c.result().copy()
    for i, bad in enumerate((np.inf, -np.inf, np.nan, np.inf, -np.inf)):
        assert np.array_equal(b[:, :, 20 + 25 * i], np.full((T, H), bad, np.float16), equal_nan=True)
    assert np.all(np.isnan(b[:, :, 0]))                      # inf - inf
    for d in (0, 20, 45, 70, 95, 120):
        a[:, :, d] = b[:, :, d] = 0
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_infinities_in_the_cache_and_in_nodes(qdiy):
    """Those of the cache reach all nodes, a node's those that see it."""
    T = 30
    vis = ancestors(chain_parents(T))
    vis[:, 4] = False
    vis[9, 4] = True
    c = Attention(qdiy, 2, 2, 700, T, seed=3, vis=vis, kscale=0.2)
    a = c.result().copy()
    c.V[333, :, 8] = np.inf
    c.Vt[4, :, 9] = np.inf
    c.Vt[4, 0, 8] = -np.inf
    c.Kt[4] = np.nan                                         # unseen but by node 9, which sees its NaN score
    c.upload()
    b = c.result().copy()
    others = [t for t in range(T) if t != 9]
    assert np.all(b[others][:, :, 8] == np.inf) and np.all(np.isnan(b[9]))
    a[9] = b[9] = 0
    a[:, :, 8] = b[:, :, 8] = 0
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_scores_that_are_no_numbers_stay_with_their_row(qdiy):
    """A NaN in one node's q leaves the other nodes' bits as they are."""
    for P, T in ((50, 7), (3000, 40), (3000, 130)):
        c = Attention(qdiy, 2, 2, P, T, seed=P)
        a = c.result().copy()
        c.q[3, 1, 17] = np.nan
        c.gq = dev(c.q.reshape(T, -1))
        b = c.result().copy()
        assert np.all(np.isnan(b[3, 1]))
        a[3, 1] = b[3, 1] = 0
        assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


# ------------------------------------------------------------------ what outputs may overlap

def test_rope_refuses_node_rows_over_each_other(qdiy):
    """K rows over V rows, rows over rows and heads over heads would race; rows that only share
    their buffer are taken."""
    H, KH, T = 4, 2, 3
    ctx = qdiy.Context(num_heads=KH, max_seqlen=50)
    W = (H + 2 * KH) * 128
    x = dev(np.random.default_rng(1).standard_normal((T, W)).astype(np.float16))
    depth, q = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(T, H * 128, dtype=torch.float16, device="cuda")
    want = [torch.zeros(T, KH, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    ctx.tree_qkv_rope(x, None, depth, q, *want, 5, T, num_heads=H)
    buf = torch.zeros(1 << 14, dtype=torch.float16, device="cuda")
    row = KH * 128

    def call(at, trow, thead):
        ctx.tree_qkv_rope(x, None, depth, q, buf, buf[at:], 5, T, num_heads=H, tree_row_stride=trow,
                          tree_head_stride=thead)

    for at, trow, thead in ((0, row, 128), (128, row, 128), (row, row, 128), (2 * row, row, 128), (64, 2 * row, 256),
                            (8192, 8, 128), (8192, row - 8, 128), (8192, row, 120), (8192, row, 8),
                            (8192, 128, 3 * 128 - 8), (8192, 128, 128), (row, 2 * row - 8, 128)):
        with pytest.raises(qdiy.QdError) as e:
            call(at, trow, thead)
        assert e.value.code == qdiy.QD_EINVAL, (at, trow, thead)
    for at, trow, thead in ((row, 2 * row, 128), (128, 2 * row, 256), (8192, row, 128), (8192, 128, 3 * 128),
                            (3 * row, row, 128), (3 * 128, 128, 6 * 128), (KH * 128 + 64, 3 * row, 128)):
        buf.zero_()
        call(at, trow, thead)
        for w, base in zip(want, (0, at)):
            got = torch.as_strided(buf, (T, KH, 128), (trow, thead, 1), base)
            assert torch.equal(got, w), (at, trow, thead)


def test_commit_refuses_cache_rows_over_each_other(qdiy):
    H, L, S, T, P = 2, 3, 40, 5, 10
    ctx = qdiy.Context(num_heads=H, max_seqlen=S)
    row = H * 128
    rng = np.random.default_rng(2)
    kt, vt = (dev(rng.standard_normal((L, T, row)).astype(np.float16)) for _ in range(2))
    path, count = dev(np.array([0, 2, 3, -1, -1], np.int32)), dev(np.array([3], np.int32))
    buf = torch.zeros(4 * L * S * row, dtype=torch.float16, device="cuda")

    def call(at, layer):
        ctx.tree_commit(kt, vt, buf, buf[at:], path, count, P, T, layers=L, cache_layer_stride=layer)

    for at, layer in ((0, S * row), (row, S * row), (128, S * row), (L * S * row, 8), (L * S * row, row),
                      (L * S * row, (T - 1) * row), (S * row, S * row)):
        with pytest.raises(qdiy.QdError) as e:
            call(at, layer)
        assert e.value.code == qdiy.QD_EINVAL, (at, layer)
    for at, layer in ((L * S * row, S * row), (S * row, 2 * S * row), (3 * S * row, S * row)):
        buf.zero_()
        call(at, layer)
        for t, base in ((kt, 0), (vt, at)):
            got = torch.as_strided(buf, (L, S, row), (layer, row, 1), base)
            assert torch.equal(got[:, P:P + 3], t[:, [0, 2, 3]])


def test_commit_takes_a_cache_that_ends_with_its_rows(qdiy):
    """A cache shorter than the context's max_seqlen, which holds every row that the call can
    write: what lies behind it in the same buffer is not the cache."""
    H, L, S, T, P = 2, 2, 400, 5, 10
    ctx = qdiy.Context(num_heads=H, max_seqlen=S)
    row, rows = H * 128, P + T
    rng = np.random.default_rng(4)
    n, m = L * rows * row, L * T * row
    buf = torch.zeros(2 * n + 2 * m + 64, dtype=torch.float16, device="cuda")
    kc, vc, kt, vt = buf[:n], buf[n:2 * n], buf[2 * n:2 * n + m], buf[2 * n + m:2 * n + 2 * m]
    path, count = buf[2 * n + 2 * m:][:2 * T].view(torch.int32), buf[2 * n + 2 * m + 32:][:2].view(torch.int32)
    x = dev(rng.standard_normal(2 * m).astype(np.float16))
    buf[2 * n:2 * n + 2 * m].copy_(x)
    path.copy_(dev(np.array([0, 1, 4, -1, -1], np.int32)))
    count.fill_(3)
    ctx.tree_commit(kt, vt, kc, vc, path, count, P, T, layers=L)
    for c, t in ((kc, x[:m]), (vc, x[m:])):
        got, want = c.view(L, rows, row), t.view(L, T, row)
        assert torch.equal(got[:, P:P + 3], want[:, [0, 1, 4]])
        assert not got[:, :P].any() and not got[:, P + 3:].any()
    assert torch.equal(buf[2 * n:2 * n + 2 * m], x)
    for bad in (dict(path=kc[:2 * T].view(torch.int32)), dict(count=vc[n - 8:].view(torch.int32)), dict(k_tree=vc)):
        a = dict(k_tree=kt, v_tree=vt, k_cache=kc, v_cache=vc, path=path, count=count)
        a.update(bad)
        with pytest.raises(qdiy.QdError):
            ctx.tree_commit(**a, prefix=P, nodes=T, layers=L, tree_layer_stride=T * row)


# ------------------------------------------------------------------ attention: long scans in several splits

# H, KH, P, T, then the blocks' rows, splits and rounds that they are there for (256 CUs): several
# splits of three rounds and more, odd and even, so that LDS buffers are written again while others
# still read, tiles loaded ahead are used, and a split's tiles lie a hop apart.
LONG = [(64, 64, 3001, 5, 16, 4, 3), (64, 64, 3999, 13, 16, 4, 4), (16, 4, 50000, 3, 16, 49, 4), (64, 32, 9001, 8, 16, 8, 5),
        (64, 64, 3001, 27, 32, 4, 3), (64, 32, 8101, 15, 32, 8, 4), (2, 1, 99990, 11, 32, 196, 2),
        (128, 128, 701, 40, 64, 2, 3), (64, 64, 1917, 64, 64, 4, 4), (64, 16, 3331, 12, 64, 14, 2), (32, 8, 6100, 48, 64, 10, 5),
        (64, 64, 601, 128, 128, 4, 3), (64, 64, 701, 100, 128, 4, 4), (32, 8, 4801, 64, 128, 16, 5), (16, 16, 4001, 250, 128, 8, 9)]


@pytest.mark.parametrize("H,KH,P,T,block,splits,rounds", LONG)
def test_long_scans_in_several_splits(qdiy, H, KH, P, T, block, splits, rounds):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    plan = attention_plan(T, H, KH, P, cus)
    if cus == 256:
        assert (plan[0], plan[3], plan[4]) == (block, splits, rounds)
    c = Attention(qdiy, H, KH, P, T, seed=P)
    assert c.ws.numel() == plan[2] * KH * plan[5] * plan[0] * 130 * 4
    a = c.result().copy()
    assert np.all(np.isfinite(a))
    G = H // KH
    for kh in sorted({0, KH // 2, KH - 1}):                  # a float64 sample of the heads, all nodes
        hs = slice(kh * G, kh * G + G)
        want, bound = attention(c.q[:, hs], c.K[:, kh:kh + 1], c.V[:, kh:kh + 1], c.Kt[:, kh:kh + 1], c.Vt[:, kh:kh + 1],
                                c.vis, with_bound=True)
        err = np.abs(a[:, hs].astype(np.float64) - want)
        assert np.all(err <= bound), np.max(err / bound)
    for _ in range(4):                                       # a race would show in some call's bits
        assert np.array_equal(a.view(np.uint16), c.result().view(np.uint16))


# ------------------------------------------------------------------ host tensors

def test_host_tensors_are_refused_by_every_call(qdiy):
    """One argument after the other on the host; nothing is launched."""
    ctx = qdiy.Context(num_heads=1, max_seqlen=64)
    h, i, f = (torch.zeros(4096, dtype=t, device="cuda") for t in (torch.float16, torch.int32, torch.float32))
    m, ws = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    calls = [(ctx.tree_qkv_rope, dict(qkv=h, bias=h, depth=i, q_out=h, k_tree=h, v_tree=h, prefix=3, nodes=2)),
             (ctx.tree_attention, dict(q=h, k_layer=h, v_layer=h, k_tree=h, v_tree=h, mask=m, out=h, prefix=3, nodes=2,
                                       workspace=ws)),
             (ctx.tree_commit, dict(k_tree=h, v_tree=h, k_cache=h, v_cache=h, path=i, count=i, prefix=3, nodes=2)),
             (qdiy.tree_verify, dict(target_logits=h, tokens=i, parents=i, nodes=2, vocab=9, workspace=ws, path=i,
                                     emitted=i, count=i, temperature=1.0, accept_u=f, sample_u=f, draft_logits=h,
                                     max_children=1))]
    n = 0
    for call, args in calls:
        for name, x in args.items():
            if isinstance(x, torch.Tensor):
                with pytest.raises(ValueError, match=f"{name} is on cpu"):
                    call(**dict(args, **{name: x.cpu()}))
                n += 1
    assert n == 6 + 8 + 6 + 10


# ------------------------------------------------------------------ a captured step

def test_a_captured_step_holds_for_its_prefix(qdiy):
    """A step of two layers captured at one prefix and replayed with other activations, drafts,
    random numbers and caches of that length, with eager work between: every replay gives the
    eager step's bits.  (Prefix is the host's number: a step at another prefix is another graph.)"""
    H, L, V, T, S, P = 4, 2, 611, 23, 160, 70
    row = H * 128
    rng = np.random.default_rng(23)
    ctx = qdiy.Context(num_heads=H, max_seqlen=S)
    half = lambda *n: torch.empty(*n, dtype=torch.float16, device="cuda")
    kc, vc, kt, vt = half(L, S, row), half(L, S, row), half(L, T, row), half(L, T, row)
    qkv, q, out, logits = half(L, T, 3 * row), half(L, T, row), half(L, T, row), half(T, V)
    parents = [-1] + [int(rng.integers(max(0, t - 3), t)) for t in range(1, T)]
    mask, depth = (x.cuda() for x in qdiy.tree_layout(parents))
    head = dev((0.3 * rng.standard_normal((V, row))).astype(np.float16))
    tokens, par = torch.zeros(T, dtype=torch.int32, device="cuda"), dev(np.array(parents, np.int32))
    au, su = torch.empty(T, device="cuda"), torch.empty(1, device="cuda")
    path, emitted = (torch.empty(T, dtype=torch.int32, device="cuda") for _ in range(2))
    count = torch.empty(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(ctx.tree_attention_workspace_bytes(T), qdiy.tree_verify_workspace_bytes(T, V)),
                     dtype=torch.uint8, device="cuda")

    def step():
        for l in range(L):
            ctx.tree_qkv_rope(qkv[l], None, depth, q[l], kt[l], vt[l], P, T)
            ctx.tree_attention(q[l], kc[l], vc[l], kt[l], vt[l], mask, out[l], P, T, ws)
        qdiy.gemm_nt(out[L - 1], head, logits, T, V, row)
        qdiy.tree_verify(logits, tokens, par, T, V, ws, path, emitted, count, temperature=0.9, accept_u=au, sample_u=su)
        ctx.tree_commit(kt, vt, kc, vc, path, count, P, T, layers=L)

    def results():
        torch.cuda.synchronize()
        return [x.cpu().numpy().copy() for x in (kc, vc, kt, vt, out, logits, path, emitted, count)]

    def inputs(seed):
        r = np.random.default_rng(seed)
        for x in (kc, vc, qkv):
            x.copy_(dev(r.standard_normal(tuple(x.shape)).astype(np.float16)))
        start = kc.clone(), vc.clone()
        au.copy_(dev(0.02 * r.random(T, dtype=np.float32)))
        su.copy_(dev(r.random(1, dtype=np.float32)))
        tokens.zero_()
        step()                                               # drafts: what the target finds likely
        order = torch.argsort(logits.float(), dim=1, descending=True, stable=True)
        tokens[1:] = order[par[1:].long(), torch.arange(1, T, device="cuda") % 3].int()
        for x, x0 in zip((kc, vc), start):                   # without the rows that step committed
            x.copy_(x0)
        return start

    inputs(1)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    counts = []
    for seed in (10, 20, 30, 40, 50):
        k0, v0 = inputs(seed)                                # (clones)
        step()
        want = results()
        kc.copy_(k0)
        vc.copy_(v0)
        for x in (kt, vt, out, logits):
            x.fill_(7.0)
        path.fill_(77)
        g.replay()
        for a, b in zip(want, results()):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
        n = int(count)
        walk = verify(logits.cpu().numpy(), tokens.cpu().numpy(), parents, "point", 0.9, au.cpu().numpy(), float(su))
        assert (path.tolist()[:n], emitted.tolist()[:n]) == walk
        counts.append(n)
    assert max(counts) > 1                                   # (the drafts weigh some 0.02 each)


# ------------------------------------------------------------------ one context, several streams; far strides

def test_calls_of_one_context_on_two_streams(qdiy):
    """The context gives them its sizes and its cos/sin table only."""
    ctx = qdiy.Context(num_heads=8, max_seqlen=2100)
    cs = [Attention(qdiy, 8, 8, 2000 + 77 * i, 30, seed=60 + i) for i in range(2)]
    rope = []
    for i, c in enumerate(cs):
        c.ctx = ctx
        x = dev(np.random.default_rng(70 + i).standard_normal((30, 24 * 128)).astype(np.float16))
        depth = torch.arange(30, dtype=torch.int32, device="cuda") // 2
        rope.append((x, depth, [torch.empty(30, 1024, dtype=torch.float16, device="cuda") for _ in range(3)]))

    def call(i, stream=None):
        cs[i].call(stream=stream)
        x, depth, outs = rope[i]
        ctx.tree_qkv_rope(x, None, depth, *outs, 100 + i, 30, stream=stream)

    def got(i):
        return [t.cpu().numpy().copy() for t in (cs[i].out, *rope[i][2])]

    for i in range(2):
        call(i)
    torch.cuda.synchronize()
    want = [got(i) for i in range(2)]
    for i in range(2):
        for t in (cs[i].out[:30], *rope[i][2]):
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(20):
        for i, s in enumerate(streams):
            call(i, s)
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(want[i], got(i)):
            assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_heads_and_layers_past_32_bits(qdiy):
    """Heads and layers 2^31 + 64 elements apart, 4 GiB and a little, in the cache and in the node rows."""
    far, P, T, S = (1 << 31) + 64, 40, 12, 60
    c = Attention(qdiy, 2, 2, P, T, seed=80)
    want = c.result().copy()
    c.ctx = qdiy.Context(num_heads=2, max_seqlen=S, kv_row_stride=128, kv_head_stride=far)
    c.trow, c.thead = 128, far
    big = [torch.empty(2 * far, dtype=torch.float16, device="cuda") for _ in range(4)]
    c.kc, c.vc, c.kt, c.vt = big
    rows = lambda x, n: torch.as_strided(x, (n, 2, 128), (128, far, 1))
    for x, src, n in ((c.kc, c.K, P), (c.vc, c.V, P), (c.kt, c.Kt, T), (c.vt, c.Vt, T)):
        rows(x, n).copy_(dev(src))
    assert np.array_equal(want.view(np.uint16), c.result().view(np.uint16))
    # the path 0, 3, 4 into the cache
    path, count = dev(np.array([0, 3, 4] + [-1] * (T - 3), np.int32)), dev(np.array([3], np.int32))
    c.ctx.tree_commit(c.kt, c.vt, c.kc, c.vc, path, count, P, T, tree_row_stride=128, tree_head_stride=far)
    for x, src, old in ((c.kc, c.Kt, c.K), (c.vc, c.Vt, c.V)):
        assert np.array_equal(rows(x, P + 3).cpu().numpy(), np.concatenate([old, src[[0, 3, 4]]]))
    # heads near, layers far
    ctx = qdiy.Context(num_heads=1, max_seqlen=S)
    for x in (c.kc, c.vc):
        torch.as_strided(x, (2, S, 128), (far, 128, 1)).zero_()
    ctx.tree_commit(c.kt, c.vt, c.kc, c.vc, path, count, P, T, layers=2, tree_layer_stride=far, cache_layer_stride=far)
    for x, src in ((c.kc, c.Kt), (c.vc, c.Vt)):
        layers = torch.as_strided(x, (2, S, 128), (far, 128, 1))
        for l in range(2):
            assert torch.equal(layers[l, P:P + 3], dev(src[[0, 3, 4], l]))
            assert not layers[l, :P].any() and not layers[l, P + 3:].any()
    # node rows from RoPE, heads far
    x = dev(np.random.default_rng(81).standard_normal((T, 6 * 128)).astype(np.float16))
    depth = torch.arange(T, dtype=torch.int32, device="cuda") // 3
    near = [torch.empty(T, 256, dtype=torch.float16, device="cuda") for _ in range(3)]
    q = torch.empty(T, 256, dtype=torch.float16, device="cuda")
    c.ctx.tree_qkv_rope(x, None, depth, *near, 7, T)
    c.ctx.tree_qkv_rope(x, None, depth, q, c.kt, c.vt, 7, T, tree_row_stride=128, tree_head_stride=far)
    assert torch.equal(q, near[0])
    for a, b in ((c.kt, near[1]), (c.vt, near[2])):
        assert torch.equal(rows(a, T), b.view(T, 2, 128))


# ------------------------------------------------------------------ the largest calls

@pytest.mark.parametrize("H,T,P", [(4095, 1024, 33), (4096, 1023, 700)])
def test_the_most_query_rows(qdiy, H, T, P):
    """Four million query rows of one cache head; a float64 sample of nodes and heads, within the
    bound of the kernel's roundings."""
    g = torch.Generator(device="cuda")
    g.manual_seed(H)
    half = lambda *n: torch.randn(*n, generator=g, device="cuda").half()
    q = torch.empty(T, H * 128, dtype=torch.float16, device="cuda")
    for t0 in range(0, T, 128):
        q[t0:t0 + 128] = half(min(128, T - t0), H * 128)
    k, v, kt, vt = half(P, 128), half(P, 128), half(T, 128), half(T, 128)
    parents = [-1] + [max(0, t - 1 - t % 7) for t in range(1, T)]
    mask = qdiy.tree_layout(parents)[0].cuda()
    ctx = qdiy.Context(num_heads=1, max_seqlen=P)
    ws = torch.empty(ctx.tree_attention_workspace_bytes(T, H), dtype=torch.uint8, device="cuda")
    out = torch.full((T, H * 128), 7.0, dtype=torch.float16, device="cuda")
    ctx.tree_attention(q, k, v, kt, vt, mask, out, P, T, ws, num_heads=H)
    assert bool(torch.isfinite(out).all())
    vis = ancestors(parents)
    nodes = sorted({0, 1, T // 3, T // 2, T - 2, T - 1})
    host = lambda x: x.cpu().numpy()
    for h in sorted({0, 1, 63, 64, H // 2, H - 2, H - 1}):
        cols = slice(h * 128, h * 128 + 128)
        # (a node's row of vis names all node rows that it sees)
        for t in nodes:
            want, bound = attention(host(q[t:t + 1, cols])[:, None], host(k)[:, None], host(v)[:, None], host(kt)[:, None],
                                    host(vt)[:, None], vis[t:t + 1], with_bound=True)
            err = np.abs(host(out[t, cols]).astype(np.float64) - want[0, 0])
            assert np.all(err <= bound[0, 0]), (h, t)


@pytest.mark.parametrize("mode", ["greedy", "point", "drawn"])
@pytest.mark.parametrize("T,V", [(300, 40001), (1024, 9000)])
def test_many_rows_whose_chunks_share_workgroups(qdiy, mode, T, V):
    for seed in range(2):
        Verify(T, V, mode, seed=seed).check(qdiy)
