"""What the tree calls promise about their arguments, on the CPU: which memory the host checks
count as read or written, and what the Python binding lets through to the C call."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def qdiy():
    import qdiy as m
    if not os.path.exists(m.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    m.load()
    return m


class Recorder:
    """In place of the library: keeps the arguments of each call and answers QD_OK."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def binding(qdiy, monkeypatch):
    """The binding over host tensors: CPU stands for the current device (get_device() is -1)."""
    rec = Recorder()
    monkeypatch.setattr(qdiy, "load", lambda: rec)
    monkeypatch.setattr(qdiy, "_current_device", lambda: -1)
    monkeypatch.setattr(qdiy, "_stream", lambda s: 0)
    return rec


def halves(n):
    return torch.zeros(n, dtype=torch.float16)


def ints(n):
    return torch.zeros(n, dtype=torch.int32)


# ------------------------------------------------------------------ rows of the drafter that are not there

def test_draft_rows_of_leaves_are_no_ones_memory(qdiy):
    """A drafter's buffer may end with its last row that has children; what lies behind it, the
    workspace here, is not the call's input.  (The call is refused for another reason, path over
    count, which is looked at later: nothing is launched.)"""
    lib = qdiy.load()
    nodes, vocab = 4, 100
    buf = ctypes.create_string_buffer(1 << 17)
    at = (ctypes.addressof(buf) + 255) & ~255
    V = ctypes.c_void_p
    wsb = lib.qd_tree_verify_workspace_bytes(nodes, vocab, 3)
    target, rest, draft = at, at + 4096, at + 8192
    p = lambda i: V(rest + 64 * i)

    def call(ws):
        return lib.qd_tree_verify(V(target), vocab, V(draft), vocab, p(0), p(1), p(2), p(3), 0.5, nodes, vocab, 3, V(ws),
                                  wsb, p(4), p(5), p(4), None)

    row = 2 * vocab
    assert call(draft + 2 * row // 16 * 16 + 16) == qdiy.QD_EINVAL     # behind the rows of nodes 0 and 1
    assert b"must not overlap" in lib.qd_last_error()
    assert call(draft + 16) == qdiy.QD_EINVAL                          # within node 0's
    assert b"overlaps an input" in lib.qd_last_error()


@pytest.mark.parametrize("nodes", [1, 2, 7])
def test_binding_takes_draft_logits_without_the_last_row(qdiy, binding, nodes):
    """The last node has no children; every other one may have."""
    V, ldd = 50, 60
    need = (nodes - 2) * ldd + V if nodes > 1 else 0
    i = ints(nodes)
    args = (halves(nodes * V), i, i, nodes, V, torch.zeros(1 << 16, dtype=torch.uint8), i, i, i)
    kw = dict(temperature=1.0, accept_u=torch.zeros(nodes), sample_u=torch.zeros(1), max_children=2, ldd=ldd)
    qdiy.tree_verify(*args, draft_logits=halves(need), **kw)
    assert len(binding.calls) == 1
    if need:
        with pytest.raises(ValueError, match="draft_logits holds"):
            qdiy.tree_verify(*args, draft_logits=halves(need - 1), **kw)
        assert len(binding.calls) == 1
