"""GPU parity of qd_tree_attention against float64 attention of the same fp16 inputs, within
the bound that tree_common.attention derives from the kernel's roundings."""
import numpy as np
import pytest
import torch

from common import normal_f16
from tree_common import D, ancestors, attention, chain_parents, mask_words, random_parents

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qdiy():
    import qdiy as m
    torch.cuda.set_device(0)
    m.load()
    return m


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Case:
    """Random nodes over a cache in the chosen layout; everything no call may read is NaN."""

    def __init__(self, qdiy, H, KH, P, T, seed=0, layout="engine", tree="engine", q_pad=0, out_pad=0, vis=None,
                 kscale=1.0, spare=3):
        rng = np.random.default_rng(seed)
        self.H, self.KH, self.P, self.T = H, KH, P, T
        self.q = normal_f16(rng, (T, H, D), 1.5)
        self.K, self.V = normal_f16(rng, (P, KH, D), kscale), normal_f16(rng, (P, KH, D))
        self.Kt, self.Vt = normal_f16(rng, (T, KH, D), kscale), normal_f16(rng, (T, KH, D))
        self.vis = ancestors(random_parents(rng, T)) if vis is None else vis
        S = P + spare
        self.ctx, self.kc, self.vc = self._rows(qdiy, S, layout)
        self.trow, self.thead = (KH * D, D) if tree == "engine" else (D, (T + 2) * D) if tree == "head_major" else (
            KH * D + 24, D)
        self.q_stride, self.out_stride = H * D + q_pad, H * D + out_pad
        qb = np.full((T, self.q_stride), np.nan, np.float16)
        qb[:, :H * D] = self.q.reshape(T, -1)
        self.gq = dev(qb)
        self.out = torch.full((T + 1, self.out_stride), 7.0, dtype=torch.float16, device="cuda")
        self.mask = dev(mask_words(self.vis))
        self.ws = torch.full((self.ctx.tree_attention_workspace_bytes(T, H),), 0xFF, dtype=torch.uint8, device="cuda")
        self.upload()

    def _rows(self, qdiy, S, layout):
        if layout == "head_major":
            self.row, self.head = D, S * D
            self.cache_shape = (self.KH, S, D)
        else:
            self.row, self.head = self.KH * D + (40 if layout == "padded" else 0), D
            self.cache_shape = (S, self.row)
        ctx = qdiy.Context(num_heads=self.KH, max_seqlen=S, kv_row_stride=self.row, kv_head_stride=self.head)
        return ctx, None, None

    def _lay(self, x, shape_rows, row, head, n):
        flat = np.full(max(1, (shape_rows - 1) * row + (self.KH - 1) * head + D), np.nan, np.float16)
        for h in range(self.KH):
            for r in range(n):
                flat[r * row + h * head:r * row + h * head + D] = x[r, h]
        return dev(flat)

    def upload(self):
        S = self.P + 3
        self.kc, self.vc = (self._lay(x, S, self.row, self.head, self.P) for x in (self.K, self.V))
        self.kt, self.vt = (self._lay(x, self.T + 2, self.trow, self.thead, self.T) for x in (self.Kt, self.Vt))

    def call(self, stream=None):
        self.ctx.tree_attention(self.gq, self.kc, self.vc, self.kt, self.vt, self.mask, self.out, self.P, self.T,
                                self.ws, num_heads=self.H, q_stride=self.q_stride, out_stride=self.out_stride,
                                tree_row_stride=self.trow, tree_head_stride=self.thead, stream=stream)

    def result(self):
        self.call()
        torch.cuda.synchronize()
        o = self.out.cpu().numpy()
        assert np.all(o[self.T] == 7.0) and np.all(o[:, self.H * D:] == 7.0)    # rows and gaps left as they were
        return o[:self.T, :self.H * D].reshape(self.T, self.H, D)

    def check(self):
        got = self.result().astype(np.float64)
        want, bound = attention(self.q, self.K, self.V, self.Kt, self.Vt, self.vis, with_bound=True)
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("T", [1, 2, 5, 15, 16, 17, 31, 33, 48, 63, 64, 65, 100])
@pytest.mark.parametrize("P", [0, 1, 31, 32, 33, 130])
def test_lengths(qdiy, P, T):
    Case(qdiy, 4, 4, P, T, seed=1000 * P + T).check()


@pytest.mark.parametrize("H,KH", [(1, 1), (2, 1), (7, 1), (32, 8), (12, 4), (16, 2), (28, 4), (16, 16), (20, 20), (71, 1)])
def test_heads(qdiy, H, KH):
    Case(qdiy, H, KH, 77, 9, seed=H).check()


@pytest.mark.parametrize("H,KH,P,T", [(2, 2, 700, 13), (16, 16, 600, 5), (8, 2, 1029, 40), (1, 1, 4099, 3),
                                      (2, 2, 2050, 130), (1, 1, 513, 257), (1, 1, 0, 1024), (4, 1, 300, 300)])
def test_longer(qdiy, H, KH, P, T):
    Case(qdiy, H, KH, P, T, seed=P + T).check()


@pytest.mark.parametrize("layout", ["engine", "padded", "head_major"])
@pytest.mark.parametrize("tree", ["engine", "padded", "head_major"])
def test_strides(qdiy, layout, tree):
    Case(qdiy, 8, 4, 210, 21, seed=5, layout=layout, tree=tree, q_pad=56, out_pad=8).check()


@pytest.mark.parametrize("P", [0, 40])
def test_any_mask(qdiy, P):
    """Masks that are no tree's, rows that see nothing: zeros over an empty prefix."""
    rng = np.random.default_rng(8)
    vis = rng.random((70, 70)) < 0.3
    vis[::7] = False
    c = Case(qdiy, 4, 2, P, 70, seed=2, vis=vis)
    c.check()
    if P == 0:
        assert np.all(c.result()[::7] == 0)


def test_bits_past_the_nodes_are_ignored(qdiy):
    c = Case(qdiy, 4, 2, 33, 37, seed=4)
    a = c.result().copy()
    words = c.mask.cpu().numpy().copy()
    words |= np.int64(-1) << np.int64(37)
    c.mask = dev(words)
    assert np.array_equal(a.view(np.uint16), c.result().view(np.uint16))


@pytest.mark.parametrize("P", [0, 45])
def test_what_masked_rows_hold_does_not_matter(qdiy, P):
    """Infinities and NaN in node rows that a node does not see leave its bits as they are."""
    T = 40
    vis = ancestors(chain_parents(T))
    vis[10:, 3] = vis[10:, 17] = vis[10:, 39] = False
    vis[39, 39] = True
    c = Case(qdiy, 4, 2, P, T, seed=6, vis=vis)
    a = c.result().copy()
    for j, bad in ((3, np.nan), (17, np.inf), (39, -np.inf)):
        c.Kt[j], c.Vt[j] = bad, bad
    c.Vt[39, :, ::2] = np.nan
    c.upload()
    b = c.result()
    blind = [t for t in range(T) if not (vis[t, 3] or vis[t, 17] or vis[t, 39])]
    assert len(blind) > 20
    assert np.array_equal(a[blind].view(np.uint16), b[blind].view(np.uint16))


def test_infinite_values_that_are_seen(qdiy):
    """A visible infinity in V reaches exactly the outputs of the nodes that see it."""
    T = 20
    vis = ancestors(chain_parents(T))
    vis[:, 12] = False
    vis[12, 12] = vis[15, 12] = True
    c = Case(qdiy, 2, 2, 50, T, seed=9, vis=vis, kscale=0.2)
    a = c.result().copy()
    c.Vt[12, :, 5] = np.inf
    c.upload()
    b = c.result()
    assert np.all(b[[12, 15]][:, :, 5] == np.inf)
    a[[12, 15], :, 5] = b[[12, 15], :, 5]
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("kscale", [0.0, 8.0, 60.0])
def test_score_spreads(qdiy, kscale):
    """Equal scores, and scores far apart (one row takes nearly all the weight).  Scores of
    60 pass the size that the bound's exponential step assumes, so there the largest weight
    is checked: rows whose best score leads by more than 40 are that row's V, rounded."""
    c = Case(qdiy, 4, 4, 300, 18, seed=11, kscale=kscale)
    if kscale < 60:
        c.check()
        return
    got = c.result()
    n = 0
    for t in range(c.T):
        for h in range(c.H):
            k = np.concatenate([c.K[:, h], c.Kt[c.vis[t], h]]).astype(np.float64)
            v = np.concatenate([c.V[:, h], c.Vt[c.vis[t], h]])
            s = np.sort(k @ c.q[t, h].astype(np.float64) / np.sqrt(D))
            if s[-1] - s[-2] > 40:
                i = int(np.argmax(k @ c.q[t, h].astype(np.float64)))
                assert np.array_equal(got[t, h], v[i])
                n += 1
    assert n > 5


def test_rising_scores(qdiy):
    """Every later row scores higher, so that a running maximum keeps moving."""
    c = Case(qdiy, 2, 2, 400, 12, seed=12)
    ramp = np.linspace(0.0, 3.0, 412, dtype=np.float32)
    base = np.where(c.q.mean(0, keepdims=True) > 0, 0.6, -0.6)
    c.q[:] = (base + 0.1 * c.q).astype(np.float16)
    c.K[:] = (ramp[:400, None, None] * base).astype(np.float16)
    c.Kt[:] = (ramp[400:, None, None] * base).astype(np.float16)
    c.gq = dev(c.q.reshape(c.T, -1))
    c.upload()
    c.check()


def test_matches_decode_attention(qdiy):
    """A chain of one node is a decode step: within the sum of both bounds."""
    c = Case(qdiy, 16, 16, 500, 1, seed=13)
    got = c.result().astype(np.float64)
    kc = torch.cat([c.kc.view(-1)[:500 * 2048], c.kt.view(-1)[:2048]])
    vc = torch.cat([c.vc.view(-1)[:500 * 2048], c.vt.view(-1)[:2048]])
    out = torch.empty(16 * D, dtype=torch.float16, device="cuda")
    c.ctx.decode_attention(c.gq, kc, vc, out, 501)
    assert np.max(np.abs(got.reshape(-1) - out.cpu().numpy().astype(np.float64))) <= 4e-3


def test_same_bits_from_call_to_call_and_on_another_stream(qdiy):
    c = Case(qdiy, 16, 16, 1500, 27, seed=14)
    a = c.result().copy()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            c.call()
    s.synchronize()
    o = c.out.cpu().numpy()[:c.T, :c.H * D].reshape(c.T, c.H, D)
    assert np.array_equal(a.view(np.uint16), o.view(np.uint16))


def test_two_streams_at_once(qdiy):
    """Two calls of one context with their own workspaces and outputs."""
    cs = [Case(qdiy, 8, 8, 2000 + 77 * i, 30, seed=20 + i) for i in range(2)]
    want = [c.result().copy() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for c, s in zip(cs, streams):
            c.call(stream=s)
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        o = c.out.cpu().numpy()[:c.T, :c.H * D].reshape(c.T, c.H, D)
        assert np.array_equal(w.view(np.uint16), o.view(np.uint16))


@pytest.mark.parametrize("H,KH,P,T", [(16, 16, 1200, 27), (4, 4, 40, 5)])
def test_captured_and_replayed(qdiy, H, KH, P, T):
    c = Case(qdiy, H, KH, P, T, seed=30)
    c.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.call()
    for seed in (31, 32, 33):
        rng = np.random.default_rng(seed)
        c.q = normal_f16(rng, (T, H, D), 1.5)
        c.gq.copy_(dev(c.q.reshape(T, -1)))
        want = c.result().copy()                       # eager, between the replays
        c.out[:T].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        o = c.out.cpu().numpy()[:T, :H * D].reshape(T, H, D)
        assert np.array_equal(want.view(np.uint16), o.view(np.uint16))


def test_rows_of_the_cache_itself_as_node_rows(qdiy):
    """The node rows may be the cache's rows behind the prefix."""
    c = Case(qdiy, 4, 4, 90, 11, seed=40, spare=11)
    want = c.result().copy()
    row = 4 * D
    kc = torch.cat([c.kc[:90 * row], c.kt[:11 * row]])
    vc = torch.cat([c.vc[:90 * row], c.vt[:11 * row]])
    c.ctx.tree_attention(c.gq, kc, vc, kc[90 * row:], vc[90 * row:], c.mask, c.out, 90, 11, c.ws)
    o = c.out.cpu().numpy()[:11].reshape(11, 4, D)
    assert np.array_equal(want.view(np.uint16), o.view(np.uint16))


def test_offsets_past_32_bits(qdiy):
    """Node rows 2^25 elements apart, the most that the call takes: row 64 starts at 4 GiB.  (A
    cache is held below 4 GiB by its context.)"""
    T, row = 70, 1 << 25
    c = Case(qdiy, 1, 1, 40, T, seed=41)
    big = torch.zeros((T - 1) * row + D, dtype=torch.float16, device="cuda")
    want = c.result().copy()
    at = (torch.arange(T, device="cuda")[:, None] * row + torch.arange(D, device="cuda")[None, :]).reshape(-1)
    big[at] = dev(c.Kt.reshape(-1))
    c.kt = big
    bigv = torch.zeros_like(big)
    bigv[at] = dev(c.Vt.reshape(-1))
    c.vt = bigv
    c.trow = row
    assert np.array_equal(want.view(np.uint16), c.result().view(np.uint16))


def test_refusals(qdiy):
    c = Case(qdiy, 8, 4, 20, 6, seed=50)
    lib = qdiy.load()
    good = dict(q=c.gq.data_ptr(), qs=c.q_stride, k=c.kc.data_ptr(), v=c.vc.data_ptr(), kt=c.kt.data_ptr(),
                vt=c.vt.data_ptr(), trow=c.trow, thead=c.thead, mask=c.mask.data_ptr(), out=c.out.data_ptr(),
                os=c.out_stride, P=20, T=6, H=8, hd=128, ws=c.ws.data_ptr(), wsb=c.ws.numel())

    def call(**kw):
        a = dict(good, **kw)
        return lib.qd_tree_attention(c.ctx._h, a["q"], a["qs"], a["k"], a["v"], a["kt"], a["vt"], a["trow"],
                                     a["thead"], a["mask"], a["out"], a["os"], a["P"], a["T"], a["H"], a["hd"],
                                     a["ws"], a["wsb"], None)

    bad = [dict(T=0), dict(T=1025), dict(P=-1), dict(P=24), dict(H=0), dict(H=6), dict(H=8192), dict(hd=64),
           dict(qs=8 * D - 8), dict(qs=8 * D + 4), dict(os=8 * D - 8), dict(os=8 * D + 2), dict(trow=0),
           dict(trow=12), dict(trow=(1 << 25) + 8), dict(thead=-8), dict(thead=1 << 41), dict(wsb=c.ws.numel() - 1),
           dict(mask=good["mask"] + 4), dict(ws=good["ws"] + 8)]
    bad += [{n: None} for n in ("q", "k", "v", "kt", "vt", "mask", "out", "ws")]
    bad += [{n: good[n] + 8} for n in ("q", "k", "v", "kt", "vt", "out")]
    bad += [dict(out=good[n]) for n in ("q", "k", "v", "kt", "vt")] + [dict(ws=good[n]) for n in ("q", "k", "vt", "out")]
    for kw in bad:
        assert call(**kw) == qdiy.QD_EINVAL, kw
    assert call() == qdiy.QD_OK
    torch.cuda.synchronize()
    with pytest.raises(qdiy.QdError):
        c.ctx.tree_attention_workspace_bytes(0, 8)
    with pytest.raises(ValueError):
        c.ctx.tree_attention(c.gq, c.kc[:64], c.vc, c.kt, c.vt, c.mask, c.out, 20, 6, c.ws, num_heads=8)
    with pytest.raises(TypeError):
        c.ctx.tree_attention(c.gq, c.kc, c.vc, c.kt, c.vt, c.mask.int(), c.out, 20, 6, c.ws, num_heads=8)
    with pytest.raises(ValueError):
        c.ctx.tree_attention(c.gq, c.kc, c.vc, c.kt, c.vt, c.mask[:3], c.out, 20, 6, c.ws, num_heads=8)
