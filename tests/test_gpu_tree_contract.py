"""What the tree calls promise beyond their results on whole inputs: memory that need not be
there, infinities that are seen, captured calls, long scans in several splits."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import Case as Attention
from test_gpu_tree_verify import Case as Verify, dev
from tree_common import ancestors, chain_parents

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
