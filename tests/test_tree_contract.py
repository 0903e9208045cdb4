"""What the tree calls promise about their arguments, on the CPU: which memory the host checks
count as read or written, and what the Python binding lets through to the C call."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT


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


# ------------------------------------------------------------------ numbers that a C int cannot hold

WIDE = [2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1]


@pytest.mark.parametrize("prefix", WIDE)
def test_binding_refuses_a_prefix_past_32_bits(qdiy, binding, prefix):
    """ctypes keeps the low 32 bits of such a number: 2^32 + 5 would run as a prefix of 5 (and
    with a prefix of -2^32 + 5 no cache row would have been asked for)."""
    ctx = qdiy.Context.__new__(qdiy.Context)
    ctx.num_heads, ctx.max_seqlen, ctx.kv_row_stride, ctx.kv_head_stride, ctx._h = 1, 64, 128, 128, None
    x, i = halves(4096), ints(4)
    ws = torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(OverflowError, match="prefix"):
        ctx.tree_qkv_rope(x, None, i, x, x, x, prefix, 2)
    with pytest.raises(OverflowError, match="prefix"):
        ctx.tree_attention(x, x, x, x, x, torch.zeros(2, dtype=torch.int64), x, prefix, 2, ws)
    with pytest.raises(OverflowError, match="prefix"):
        ctx.tree_commit(x, x, x, x, i, i, prefix, 2)
    assert not binding.calls
    ctx.tree_qkv_rope(x, None, i, x, x, x, 5, 2)
    assert len(binding.calls) == 1


@pytest.mark.parametrize("n", WIDE)
def test_binding_refuses_counts_past_32_bits(qdiy, binding, n):
    ctx = qdiy.Context.__new__(qdiy.Context)
    ctx.num_heads, ctx.max_seqlen, ctx.kv_row_stride, ctx.kv_head_stride, ctx._h = 1, 64, 128, 128, None
    x, i, ws = halves(4096), ints(4), torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(OverflowError, match="max_children"):
        qdiy.tree_verify(x, i, i, 2, 9, ws, i, i, i, max_children=n)
    with pytest.raises(OverflowError, match="nodes"):
        qdiy.tree_verify(x, i, i, n, 9, ws, i, i, i)
    with pytest.raises(OverflowError, match="vocab"):
        qdiy.tree_verify(x, i, i, 2, n, ws, i, i, i)
    with pytest.raises(OverflowError, match="nodes"):
        ctx.tree_attention(x, x, x, x, x, torch.zeros(2, dtype=torch.int64), x, 5, n, ws)
    with pytest.raises(OverflowError, match="num_heads"):
        ctx.tree_qkv_rope(x, None, i, x, x, x, 5, 2, num_heads=n)
    with pytest.raises((OverflowError, ValueError), match="layers"):
        ctx.tree_commit(x, x, x, x, i, i, 5, 2, layers=n, tree_layer_stride=0, cache_layer_stride=0)
    for call in (lambda: ctx.tree_attention_workspace_bytes(n), lambda: ctx.tree_attention_workspace_bytes(2, n),
                 lambda: qdiy.tree_verify_workspace_bytes(n, 9), lambda: qdiy.tree_verify_workspace_bytes(2, n),
                 lambda: qdiy.tree_verify_workspace_bytes(2, 9, n)):
        with pytest.raises(OverflowError):
            call()
    assert not binding.calls


@pytest.mark.parametrize("stride", [2 ** 63, -2 ** 63 - 1, -2 ** 64 + 1024])
def test_binding_refuses_strides_past_64_bits(qdiy, binding, stride):
    """(A stride below zero makes the extents small, which are checked with Python's numbers.)"""
    ctx = qdiy.Context.__new__(qdiy.Context)
    ctx.num_heads, ctx.max_seqlen, ctx.kv_row_stride, ctx.kv_head_stride, ctx._h = 1, 64, 128, 128, None
    x, i, ws = halves(4096), ints(4), torch.zeros(4096, dtype=torch.uint8)
    m = torch.zeros(2, dtype=torch.int64)
    for kw in ("qkv_stride", "q_stride", "tree_row_stride", "tree_head_stride"):
        with pytest.raises(OverflowError, match=kw):
            ctx.tree_qkv_rope(x, None, i, x, x, x, 5, 2, **{kw: stride})
    for kw in ("q_stride", "out_stride", "tree_row_stride", "tree_head_stride"):
        with pytest.raises(OverflowError, match=kw):
            ctx.tree_attention(x, x, x, x, x, m, x, 5, 2, ws, **{kw: stride})
    for kw in ("tree_layer_stride", "tree_row_stride", "tree_head_stride", "cache_layer_stride"):
        with pytest.raises(OverflowError, match=kw):
            ctx.tree_commit(x, x, x, x, i, i, 5, 2, **{kw: stride})
    for kw in ("ldt", "ldd"):
        with pytest.raises(OverflowError, match=kw):
            qdiy.tree_verify(x, i, i, 2, 9, ws, i, i, i, **{kw: stride})
    assert not binding.calls


def test_binding_refuses_fractions(qdiy, binding):
    x, i, ws = halves(4096), ints(4), torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(TypeError, match="whole numbers"):
        qdiy.tree_verify(x, i, i, 2, 9.5, ws, i, i, i)
    assert not binding.calls


# ------------------------------------------------------------------ layouts

@pytest.mark.parametrize("parents", [[-1, 2 ** 32], [2 ** 31, 0], [-1, 0, -2 ** 32 + 1]])
def test_layout_refuses_parents_past_32_bits(qdiy, parents):
    with pytest.raises(OverflowError):
        qdiy.tree_layout(parents)


@pytest.mark.parametrize("parents", [[-1, 0.5], [-1, "0"], [-1, None]])
def test_layout_refuses_what_is_no_whole_number(qdiy, parents):
    with pytest.raises(TypeError):
        qdiy.tree_layout(parents)


def test_layout_of_too_many_nodes_allocates_nothing(qdiy, monkeypatch):
    """The masks of 200000 nodes would take 5 GB; the count is refused before they are made."""
    sizes = []
    empty = torch.empty
    monkeypatch.setattr(qdiy.torch, "empty", lambda *a, **kw: sizes.append(a) or empty(0, **kw))
    with pytest.raises(qdiy.QdError) as e:
        qdiy.tree_layout([-1] + [0] * 199999)
    assert e.value.code == qdiy.QD_EINVAL and not sizes


def test_layout_takes_arrays_and_tensors(qdiy):
    import numpy as np
    want = qdiy.tree_layout([-1, 0, 0, 2])
    for p in (np.array([-1, 0, 0, 2], np.int64), torch.tensor([-1, 0, 0, 2], dtype=torch.int32), (-1, 0, 0, 2)):
        mask, depth = qdiy.tree_layout(p)
        assert torch.equal(mask, want[0]) and torch.equal(depth, want[1])


# ------------------------------------------------------------------ attention's plan

def test_the_restated_plan_is_the_librarys(tmp_path):
    """tests/tree_plan.py chooses the GPU tests' sizes by block, splits and rounds."""
    from tree_plan import attention_plan
    src, lib = tmp_path / "shim.cpp", tmp_path / "shim.so"
    src.write_text("""
#include "qd_tree.h"
extern "C" void plan(int nodes, int heads, int kv_heads, int prefix, int cus, int* out) {
  const qd::TreeAttnPlan p = qd::tree_attn_plan(nodes, heads, kv_heads, prefix, cus, out + 5);
  out[0] = p.block_rows, out[1] = p.key_waves, out[2] = p.blocks, out[3] = p.splits, out[4] = p.rounds;
}
""")
    csrc = os.path.join(ROOT, "llm-inference-diy_amd", "csrc")
    subprocess.run(["hipcc", "-x", "c++", "-D__HIP_PLATFORM_AMD__", "-std=c++17", "-shared", "-fPIC", "-I", csrc, "-I",
                    "/opt/rocm/include", "-o", str(lib), str(src)], check=True)
    plan = ctypes.CDLL(str(lib)).plan
    out = (ctypes.c_int * 6)()
    for nodes in (1, 5, 16, 17, 32, 33, 64, 65, 100, 128, 129, 250, 1024):
        for heads, kv_heads in ((1, 1), (16, 16), (32, 8), (28, 4), (71, 1), (64, 64), (300, 300)):
            for prefix in (0, 1, 32, 33, 512, 700, 2000, 8191, 32700):
                plan(nodes, heads, kv_heads, prefix, 256, out)
                assert tuple(out) == attention_plan(nodes, heads, kv_heads, prefix, 256), (nodes, heads, kv_heads, prefix)


# ------------------------------------------------------------------ max_children

@pytest.mark.parametrize("max_children", [-1, 0, 65, 1000])
@pytest.mark.parametrize("mode", ["greedy", "point", "drawn, one node"])
def test_max_children_is_not_read_without_drawn_siblings(qdiy, mode, max_children):
    """Refused for path over count, which is looked at after max_children and the workspace's size."""
    lib = qdiy.load()
    nodes, vocab = 1 if mode.startswith("drawn") else 4, 100
    buf = ctypes.create_string_buffer(1 << 17)
    at = (ctypes.addressof(buf) + 255) & ~255
    V = ctypes.c_void_p
    p = lambda i: V(at + 8192 + 64 * i)
    wsb = lib.qd_tree_verify_workspace_bytes(nodes, vocab, 0)
    draft = V(at + 4096) if mode.startswith("drawn") else None
    rc = lib.qd_tree_verify(V(at), vocab, draft, vocab, p(0), p(1), p(2), p(3), 0.0 if mode == "greedy" else 0.5, nodes,
                            vocab, max_children, V(at + 16384), wsb, p(4), p(5), p(4), None)
    assert rc == qdiy.QD_EINVAL and b"must not overlap" in lib.qd_last_error()


# ------------------------------------------------------------------ tensors that no kernel may be given

def test_tensors_of_another_device_are_refused(qdiy):
    """A host tensor where device 0 is current, without asking any device."""
    h = halves(4)
    with pytest.raises(ValueError, match="x is on cpu, the current device is cuda:0"):
        qdiy._arg(h, "x", torch.float16, 0, 1)
    with pytest.raises(ValueError, match="workspace is on cpu, the current device is cuda:0"):
        qdiy._workspace(h, 0)
    assert qdiy._arg(h, "x", torch.float16, -1, 4) == h.data_ptr()
    assert qdiy._workspace(h, -1) == (h.data_ptr(), 8)


def test_other_tensors_are_refused(qdiy):
    h = halves(16).view(4, 4)
    with pytest.raises(TypeError, match="x must be torch.float32"):
        qdiy._arg(h, "x", torch.float32, -1, 1)
    with pytest.raises(ValueError, match="x must be contiguous"):
        qdiy._arg(h.t(), "x", torch.float16, -1, 1)
    with pytest.raises(ValueError, match="x holds 16 elements, needs 17"):
        qdiy._arg(h, "x", torch.float16, -1, 17)
    for x in ([1.0], None, 3):
        with pytest.raises(TypeError, match="x must be a torch.Tensor"):
            qdiy._arg(x, "x", torch.float16, -1, 1)
    for x in (h.t(), 5):
        with pytest.raises(TypeError, match="workspace"):
            qdiy._workspace(x, -1)
