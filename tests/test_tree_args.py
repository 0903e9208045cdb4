"""Drafted-token trees, on the CPU: qd_tree_layout against a plain walk, and the refusals
of every entry point, which answer before any GPU work."""
import ctypes
import os

import numpy as np
import pytest
import torch

from tree_common import ancestors, chain_parents, depths, mask_words, random_parents, softmax64, verify


@pytest.fixture(scope="module")
def qdiy():
    import qdiy as m
    if not os.path.exists(m.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    m.load()
    return m


@pytest.mark.parametrize("nodes", [1, 2, 63, 64, 65, 129, 1024])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_layout(qdiy, nodes, kind):
    parents = chain_parents(nodes) if kind == "chain" else random_parents(np.random.default_rng(nodes), nodes, 20)
    mask, depth = qdiy.tree_layout(parents)
    assert np.array_equal(mask.numpy(), mask_words(ancestors(parents)))
    assert depth.tolist() == depths(parents)


@pytest.mark.parametrize("parents", [[0], [1], [-1, 1], [-1, -1], [-1, 0, 3], [], [-1] + [0] * 1024])
def test_layout_refuses(qdiy, parents):
    with pytest.raises(qdiy.QdError) as e:
        qdiy.tree_layout(parents)
    assert e.value.code == qdiy.QD_EINVAL


def test_layout_outputs_are_optional(qdiy):
    lib = qdiy.load()
    par = (ctypes.c_int * 3)(-1, 0, 1)
    depth = (ctypes.c_int * 3)()
    mask = (ctypes.c_uint64 * 3)()
    assert lib.qd_tree_layout(par, 3, None, depth) == 0 and list(depth) == [0, 1, 2]
    assert lib.qd_tree_layout(par, 3, mask, None) == 0 and list(mask) == [1, 3, 7]
    assert lib.qd_tree_layout(None, 3, mask, depth) == qdiy.QD_EINVAL


def test_workspace_sizes_refuse(qdiy):
    lib = qdiy.load()
    for a in ((0, 100, 1), (1025, 100, 1), (4, 0, 1), (4, (1 << 24) + 1, 1), (4, 100, -1), (4, 100, 65)):
        assert lib.qd_tree_verify_workspace_bytes(*a) == 0
        with pytest.raises(ValueError):
            qdiy.tree_verify_workspace_bytes(*a)
    assert lib.qd_tree_verify_workspace_bytes(1, 1, 0) > 0
    assert lib.qd_tree_attention_workspace_bytes(None, 4, 16) == 0


def _verify_args():
    buf = ctypes.create_string_buffer(1 << 20)
    base = (ctypes.addressof(buf) + 255) & ~255
    at = lambda i: base + i * 32768
    return buf, dict(target=at(0), ldt=100, draft=at(1), ldd=100, tokens=at(2), parents=at(3), au=at(4), su=at(5),
                     temp=0.5, nodes=4, vocab=100, kids=3, ws=at(6), wsb=32768, path=at(8), emitted=at(9),
                     count=at(10))


def test_verify_refuses(qdiy):
    lib = qdiy.load()
    keep, good = _verify_args()
    V = ctypes.c_void_p

    def call(**kw):
        a = dict(good, **kw)
        return lib.qd_tree_verify(V(a["target"]), a["ldt"], V(a["draft"]), a["ldd"], V(a["tokens"]), V(a["parents"]),
                                  V(a["au"]), V(a["su"]), a["temp"], a["nodes"], a["vocab"], a["kids"], V(a["ws"]),
                                  a["wsb"], V(a["path"]), V(a["emitted"]), V(a["count"]), None)

    bad = [dict(nodes=0), dict(nodes=1025), dict(vocab=0), dict(vocab=1 << 25), dict(temp=-1.0),
           dict(temp=float("nan")), dict(temp=float("inf")), dict(temp=1e-9), dict(kids=0), dict(kids=65),
           dict(kids=-1), dict(ldt=99), dict(ldd=99), dict(wsb=16), dict(target=good["target"] + 1),
           dict(draft=good["draft"] + 1), dict(ws=good["ws"] + 8)]
    bad += [{n: None} for n in ("target", "tokens", "parents", "au", "su", "ws", "path", "emitted", "count")]
    bad += [{n: good[n] + 2} for n in ("tokens", "parents", "au", "su", "path", "emitted", "count")]
    # outputs over inputs, and over each other
    bad += [dict(path=good["target"]), dict(emitted=good["draft"] + 64), dict(count=good["tokens"] + 4),
            dict(path=good["parents"]), dict(ws=good["au"]), dict(count=good["su"]),
            dict(path=good["emitted"] + 4), dict(count=good["path"]), dict(ws=good["path"])]
    for kw in bad:
        assert call(**kw) == qdiy.QD_EINVAL, kw
        assert lib.qd_last_error()


def test_calls_refuse_a_null_context(qdiy):
    lib = qdiy.load()
    buf = ctypes.create_string_buffer(4096)
    b = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255)
    assert lib.qd_tree_qkv_rope(None, b, 384, None, b, b, 128, b, b, 128, 128, 0, 1, 1, 128, None) == qdiy.QD_EINVAL
    assert lib.qd_tree_attention(None, b, 128, b, b, b, b, 128, 128, b, b, 128, 0, 1, 1, 128, b, 256,
                                 None) == qdiy.QD_EINVAL
    assert lib.qd_tree_commit(None, b, b, 0, 128, 128, b, b, 0, b, b, 0, 1, 1, None) == qdiy.QD_EINVAL


def test_cpu_tensors_are_refused(qdiy):
    h = torch.zeros(4, 100, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    if not torch.cuda.is_available():
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            qdiy.tree_verify(h, i, i, 4, 100, torch.zeros(4096, dtype=torch.uint8), i, i, i)


@pytest.mark.parametrize("mode", ["point", "drawn"])
def test_the_definition_keeps_the_targets_distribution(mode):
    """The first emitted token of the tests' own float64 walk is distributed as the target's
    softmax, whatever the drafts: 40000 walks over 6 tokens, each count within 5 standard
    deviations (a false alarm in 1 of 10^5 runs; the draws are fixed)."""
    rng = np.random.default_rng(3)
    V, n, temp = 6, 40000, 0.7
    logits = rng.standard_normal((4, V)).astype(np.float16)
    draft = rng.standard_normal((4, V)).astype(np.float16)
    parents = [-1, 0, 0, 0]
    q = softmax64(draft[0], temp)
    hits = np.zeros(V)
    tokens = np.array([0, 1, 4, 1])
    for _ in range(n):
        if mode == "drawn":
            tokens = np.concatenate([[0], rng.choice(V, 3, p=q)])
        _, out = verify(logits, tokens, parents, mode, temp, rng.random(4), rng.random(), draft)
        hits[out[0]] += 1
    p = softmax64(logits[0], temp)
    assert np.all(np.abs(hits - n * p) < 5 * np.sqrt(n * p * (1 - p)))
