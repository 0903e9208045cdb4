"""What the tree calls promise beyond their results on whole inputs: memory that need not be
there, infinities that are seen, captured calls, long scans in several splits."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_tree_verify import Case as Verify, dev

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
