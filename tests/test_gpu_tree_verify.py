"""GPU parity of qd_tree_verify: path, emitted tokens and count equal those of the float64
walk of tree_common.verify."""
import numpy as np
import pytest
import torch

from tree_common import chain_parents, random_parents, softmax64, verify

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
    def __init__(self, T, V, mode, seed=0, parents=None, temperature=0.8, spread=2.0, pad=0):
        rng = np.random.default_rng(seed)
        self.T, self.V, self.mode, self.pad = T, V, mode, pad
        self.temperature = 0.0 if mode == "greedy" else temperature
        self.parents = random_parents(rng, T) if parents is None else list(parents)
        x = rng.standard_normal((T, V)) * spread
        for _ in range(3):
            x[np.arange(T), rng.integers(0, V, T)] += 6.0
        self.logits = x.astype(np.float16)
        self.draft = (x + 0.6 * rng.standard_normal((T, V))).astype(np.float16) if mode == "drawn" else None
        self.tokens = np.zeros(T, np.int32)
        rank = {}
        for t in range(1, T):
            p = self.parents[t]
            if mode == "drawn":
                self.tokens[t] = rng.choice(V, p=softmax64(self.draft[p], self.temperature))
            else:
                order = np.argsort(-x[p], kind="stable")
                self.tokens[t] = order[min(rank.get(p, 0), V - 1)]
                rank[p] = rank.get(p, 0) + 1
        self.au = rng.random(T, dtype=np.float32)
        self.su = rng.random(1, dtype=np.float32)
        self.max_children = max([1] + [self.parents.count(t) for t in range(T)])

    def upload(self):
        def rows(x):
            b = np.full((self.T, self.V + self.pad), np.float16(60000.0))
            b[:, :self.V] = x
            return dev(b)
        self.g = dict(target=rows(self.logits), draft=None if self.draft is None else rows(self.draft),
                      tokens=dev(self.tokens), parents=dev(np.array(self.parents, np.int32)), au=dev(self.au),
                      su=dev(self.su))

    def outputs(self, qdiy):
        n = qdiy.tree_verify_workspace_bytes(self.T, self.V, self.max_children)
        self.ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
        self.path, self.emitted = (torch.full((self.T + 1,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        self.count = torch.full((2,), 77, dtype=torch.int32, device="cuda")

    def call(self, qdiy, stream=None):
        g = self.g
        qdiy.tree_verify(g["target"], g["tokens"], g["parents"], self.T, self.V, self.ws, self.path, self.emitted,
                         self.count, temperature=self.temperature, accept_u=g["au"], sample_u=g["su"],
                         draft_logits=g["draft"], max_children=self.max_children, ldt=self.V + self.pad,
                         ldd=self.V + self.pad, stream=stream)

    def got(self):
        torch.cuda.synchronize()
        path, out, n = self.path.tolist(), self.emitted.tolist(), self.count.tolist()
        assert path[self.T] == 77 and out[self.T] == 77 and n[1] == 77
        n = n[0]
        assert path[n:self.T] == [-1] * (self.T - n) and out[n:self.T] == [-1] * (self.T - n)
        return path[:n], out[:n]

    def want(self):
        return verify(self.logits, self.tokens, self.parents, self.mode, self.temperature, self.au, self.su[0],
                      self.draft, self.max_children)

    def check(self, qdiy):
        self.upload()
        self.outputs(qdiy)
        self.call(qdiy)
        got, want = self.got(), self.want()
        assert got == want
        return got


MODES = ["greedy", "point", "drawn"]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,V", [(1, 1), (1, 50), (2, 1), (3, 7), (8, 1000), (17, 8191), (17, 8192), (9, 8193),
                                 (40, 503), (64, 32003), (5, 151936), (129, 300)])
def test_trees(qdiy, mode, T, V):
    for seed in range(4):
        Case(T, V, mode, seed=seed).check(qdiy)


@pytest.mark.parametrize("mode", MODES)
def test_chains(qdiy, mode):
    lens = [len(Case(12, 700, mode, seed=s, parents=chain_parents(12)).check(qdiy)[0]) for s in range(8)]
    assert max(lens) > 2


@pytest.mark.parametrize("mode", MODES)
def test_the_largest_tree(qdiy, mode):
    Case(1024, 64, mode, seed=3, parents=random_parents(np.random.default_rng(5), 1024, 40)).check(qdiy)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_row_strides(qdiy, mode, pad):
    """Rows that start at any 2-byte address; what lies between them is not read as a logit."""
    Case(14, 9001, mode, seed=6, pad=pad).check(qdiy)


@pytest.mark.parametrize("mode", ["point", "drawn"])
@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24])
def test_random_numbers_at_their_ends(qdiy, mode, u):
    """0 accepts every draft of positive probability and takes the first token with weight; the
    largest float below 1 rejects most and takes the last."""
    for seed in range(3):
        c = Case(20, 900, mode, seed=seed)
        c.au[:] = u
        c.su[:] = u
        path, _ = c.check(qdiy)
        if u == 0.0:
            assert c.parents.count(path[-1]) == 0     # down to a leaf
    flat = Case(3, 20000, mode, seed=9, spread=0.01)
    flat.au[:] = 1.0 - 2.0 ** -24
    flat.su[:] = u
    flat.check(qdiy)


def test_all_children_rejected(qdiy):
    """Siblings that all fail leave the rest of the distribution, also where they held nearly all
    of it and where two carry the same token."""
    T, V = 6, 12000
    c = Case(T, V, "point", seed=2, parents=[-1, 0, 0, 0, 0, 0])
    c.logits[0] = np.float16(-4.0)
    c.logits[0, [5, 8191, 8192, 11999]] = np.float16(12.0)
    c.tokens[1:] = [5, 8191, 5, 8192, 11999]
    c.au[:] = 1.0 - 2.0 ** -24
    for u in (0.0, 0.3, 0.9999):
        c.su[:] = u
        path, out = c.check(qdiy)
        assert path == [0] and out[0] not in (5, 8191, 8192, 11999)


def test_nothing_left(qdiy):
    """All tokens of a tiny vocabulary rejected (random numbers of 1, outside their range): the
    call ends, with token 0."""
    c = Case(3, 2, "point", seed=1, parents=[-1, 0, 0])
    c.tokens[1:] = [0, 1]
    c.au[:] = 1.0
    c.check(qdiy)


@pytest.mark.parametrize("mode", MODES)
def test_logits_that_are_no_numbers(qdiy, mode):
    T, V = 7, 8300
    for fill in ("nan", "ninf", "pinf", "mixed"):
        c = Case(T, V, mode, seed=4, parents=[-1, 0, 1, 2, 3, 4, 5])
        rng = np.random.default_rng(11)
        for x in [c.logits] + ([c.draft] if c.draft is not None else []):
            if fill == "nan":
                x[0] = np.nan
            elif fill == "ninf":
                x[0] = -np.inf
            elif fill == "pinf":
                x[0, [3, 8200]] = np.inf
            else:
                x[:, rng.integers(0, V, 4000)] = -np.inf
                x[:, rng.integers(0, V, 400)] = np.nan
        c.check(qdiy)


def test_argmax_ties_and_signed_zeros(qdiy):
    c = Case(3, 20000, "greedy", seed=1, parents=chain_parents(3))
    c.logits[:] = np.float16(-1.0)
    c.logits[0, [9000, 400, 19999]] = np.float16(2.0)
    c.logits[1, 77] = np.float16(-0.0)
    c.logits[1, 12000] = np.float16(0.0)
    c.tokens[1:] = [400, 77]
    path, out = c.check(qdiy)
    assert path == [0, 1, 2] and out == [400, 77, 0]


@pytest.mark.parametrize("mode", MODES)
def test_tokens_and_parents_out_of_range(qdiy, mode):
    """Drafted tokens outside the vocabulary are rejected; nodes without a proper parent are
    never reached."""
    c = Case(9, 600, mode, seed=5, parents=[-1, 0, 0, 0, 1, 2, 3, 3, 3])
    c.tokens[[1, 2]] = [-1, 600]
    c.au[:] = 0.0
    c.check(qdiy)
    c.tokens[1] = 2 ** 31 - 1
    c.tokens[2] = -2 ** 31
    c.parents[6:] = [7, -5, 8]
    path, _ = c.check(qdiy)
    assert not set(path) & {1, 2, 6, 7, 8}


def test_max_children(qdiy):
    """Only the first children of a node are tested against drawn drafts."""
    for seed in range(6):
        c = Case(8, 300, "drawn", seed=seed, parents=[-1, 0, 0, 0, 0, 0, 0, 0])
        c.au[1:3] = 1.0 - 2.0 ** -24
        c.au[3:] = 0.0
        c.max_children = 2
        path, _ = c.check(qdiy)
        assert path in ([0], [0, 1], [0, 2])


def test_draft_equal_to_target(qdiy):
    """q == p: every drawn child of positive probability stands; one that could not be drawn is
    rejected and leaves p as it was."""
    c = Case(4, 500, "drawn", seed=7, parents=[-1, 0, 0, 1])
    c.draft[:] = c.logits
    path, _ = c.check(qdiy)
    assert path[:2] == [0, 1]
    c.logits[0, 11] = c.draft[0, 11] = -np.inf
    c.tokens[[1, 2]] = 11
    path, out = c.check(qdiy)
    assert path == [0] and out[0] != 11


@pytest.mark.parametrize("temperature", [1e-6, 0.05, 1.0, 30.0, 1e30])
@pytest.mark.parametrize("mode", ["point", "drawn"])
def test_temperatures(qdiy, mode, temperature):
    if mode == "drawn" and temperature == 1e-6:
        c = Case(10, 400, mode, seed=3, temperature=0.01)
        c.temperature = 1e-6
        c.draft[:] = c.logits
    else:
        c = Case(10, 400, mode, seed=3, temperature=temperature)
    c.check(qdiy)


@pytest.mark.parametrize("mode", ["point", "drawn"])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 100.0])
def test_large_logits(qdiy, mode, temperature):
    """Logits near the ends of their type: neighbours differ by 32, far more than the temperature."""
    c = Case(9, 3000, "point", seed=2)
    rng = np.random.default_rng(12)
    c.mode, c.temperature = mode, temperature
    c.logits = (rng.standard_normal((9, 3000)) * 20000).clip(-65000, 65000).astype(np.float16)
    c.logits[:, 7] = np.float16(65504)
    c.logits[:, 1500] = np.float16(65472)
    if mode == "drawn":
        c.draft = c.logits.copy()
        c.draft[:, 1500] = np.float16(65504)
    c.tokens[1:] = np.where(rng.random(8) < 0.5, 7, 1500)
    c.check(qdiy)


@pytest.mark.parametrize("mode", MODES)
def test_captured_and_replayed(qdiy, mode):
    c = Case(27, 9000, mode, seed=0)
    c.upload()
    c.outputs(qdiy)
    c.call(qdiy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.call(qdiy)
    for seed in (1, 2, 3, 4):
        n = Case(27, 9000, mode, seed=seed, parents=c.parents)
        for name in ("logits", "tokens", "au", "su", "draft"):
            setattr(c, name, getattr(n, name))
        c.g["target"].copy_(dev(n.logits))
        c.g["tokens"].copy_(dev(n.tokens))
        c.g["au"].copy_(dev(n.au))
        c.g["su"].copy_(dev(n.su))
        if n.draft is not None:
            c.g["draft"].copy_(dev(n.draft))
        c.path[:27] = 5
        torch.cuda.synchronize()
        graph.replay()
        assert c.got() == c.want()


def test_two_streams_at_once(qdiy):
    cs = [Case(30, 20011, m, seed=8) for m in ("point", "drawn")]
    streams = [torch.cuda.Stream() for _ in cs]
    for c in cs:
        c.upload()
        c.outputs(qdiy)
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s in zip(cs, streams):
            c.call(qdiy, stream=s)
    torch.cuda.synchronize()
    for c in cs:
        assert c.got() == c.want()


@pytest.mark.parametrize("mode", MODES)
def test_a_vocabulary_of_many_chunks(qdiy, mode):
    """More chunks than a wave's lanes, in the short and in the long chunks."""
    Case(2, 300001, mode, seed=2, parents=[-1, 0]).check(qdiy)
    Case(3, 4500000, mode, seed=3, parents=[-1, 0, 0]).check(qdiy)


def test_rejected_by_a_random_number_of_one(qdiy):
    """u = 1 rejects every child of a point draft, also where one token holds all but 1e-17 of
    the weight, so that nothing representable is left of 1 after it."""
    c = Case(5, 300, "point", seed=9, parents=[-1, 0, 0, 0, 1], temperature=1.0)
    c.logits[:] = np.float16(0.0)
    c.logits[:, 7] = np.float16(45.0)
    c.logits[:, 11] = np.float16(3.0)
    c.tokens[1:] = [7, 11, 12, 7]
    c.au[:] = 1.0
    path, out = c.check(qdiy)
    assert path == [0] and out[0] not in (7, 11, 12)
