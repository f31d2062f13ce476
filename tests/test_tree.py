"""Host side of drafted trees and the refusals of the new C entry points: no GPU needed."""
import ctypes
import os
import random

import pytest
import torch

from metagross_b200.tree import tree_depths, tree_mask

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metagross_b200", "libmgb200.so")


def walk(parents):
    T = len(parents)
    m = torch.zeros(T, T, dtype=torch.bool)
    for t in range(T):
        u = t
        while u >= 0:
            m[t, u] = True
            u = parents[u]
    return m


@pytest.mark.parametrize("T", [1, 2, 3, 7, 16, 33, 100])
def test_mask_follows_the_parents(T):
    r = random.Random(T)
    trees = [[-1] + [r.randrange(-1, t) for t in range(1, T)], list(range(-1, T - 1)), [-1] * T, [-1] + [0] * (T - 1)]
    want = torch.stack([walk(p) for p in trees])
    assert torch.equal(tree_mask(trees), want)
    for p, m in zip(trees, want):
        assert torch.equal(tree_mask(p), m)
        assert tree_depths(m).tolist() == [int(x) for x in m.sum(1) - 1]


def test_a_parent_above_its_token_is_refused():
    with pytest.raises(ValueError, match="smaller index"):
        tree_mask([-1, 1, 0])


class Layout(ctypes.Structure):
    _fields_ = [("kv_dtype", ctypes.c_int32), ("staging_dtype", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("num_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("max_blocks", ctypes.c_int32),
                ("num_pages", ctypes.c_int64), ("scale_layout", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Ptrs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_pool", "v_pool", "k_scales", "v_scales", "staging_k", "staging_v")]


class Draft(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q_stride", ctypes.c_int64 * 3),
                ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3), ("mask", ctypes.c_void_p),
                ("mask_stride", ctypes.c_int64), ("max_draft", ctypes.c_int32), ("num_q_heads", ctypes.c_int32)]


@pytest.fixture
def lib():
    so = ctypes.CDLL(LIB)
    so.mg_last_error.restype = ctypes.c_char_p
    for f in ("mg_tree_plan_bytes", "mg_tree_workspace_bytes", "mg_fork_workspace_bytes"):
        getattr(so, f).restype = ctypes.c_int64
    return so


A = 1 << 20  # an address that is never dereferenced: every call below is refused before its launch


@pytest.mark.parametrize("hkv,d,hq,draft,text", [(4, 96, 32, 8, b"head_dim 64 or 128"), (4, 64, 30, 8, b"multiple"),
                                                 (4, 64, 32, -1, b"max_draft")])
def test_unsupported_tree_shapes_have_no_size(lib, hkv, d, hq, draft, text):
    lay = Layout(0, 1, 16, hkv, d, 64, 1024)
    assert lib.mg_tree_plan_bytes(ctypes.byref(lay), 2, draft, hq) == 0
    assert text in lib.mg_last_error()
    assert lib.mg_tree_workspace_bytes(ctypes.byref(lay), 2, draft, hq) == 0


def tree_call(lib, lay, draft, plan=A, plan_bytes=1 << 40, scale=0.125, ws=A, ws_bytes=1 << 40, ptrs=None):
    ptrs = ptrs or Ptrs(*([A] * 6))
    rc = lib.mg_tree_attention(ctypes.byref(lay), ctypes.byref(ptrs), ctypes.c_void_p(A), 2, ctypes.byref(draft),
                               ctypes.c_void_p(plan), ctypes.c_int64(plan_bytes), ctypes.c_float(scale),
                               ctypes.c_void_p(A), ctypes.c_void_p(ws), ctypes.c_int64(ws_bytes), None, None)
    return rc, lib.mg_last_error()


def test_tree_attention_refusals(lib):
    lay = Layout(0, 1, 16, 4, 64, 64, 1024)
    st = (ctypes.c_int64 * 3)(1024, 128, 64)
    ok = lambda **k: Draft(**{**dict(q=A, k=A, v=A, q_stride=st, k_stride=st, v_stride=st, max_draft=4,  # noqa: E731
                                     num_q_heads=32), **k})
    for kw, text in ((dict(plan_bytes=64), b"plan needs"), (dict(plan=A + 8), b"plan needs"),
                     (dict(ws_bytes=64), b"workspace needs"), (dict(scale=-1.0), b"scale"),
                     (dict(scale=float("inf")), b"scale"), (dict(ptrs=Ptrs(A, A, A, A, None, None)), b"null layer")):
        rc, err = tree_call(lib, lay, ok(), **kw)
        assert rc == 1 and text in err, (kw, err)
    for d, text in ((ok(q=None), b"null"), (ok(v=A + 4), b"8-byte"),
                    (ok(k_stride=(ctypes.c_int64 * 3)(1024, 126, 64)), b"strides"), (ok(num_q_heads=30), b"multiple")):
        rc, err = tree_call(lib, lay, d)
        assert rc == 1 and text in err, err
    rc, err = tree_call(lib, Layout(0, 0, 16, 4, 64, 64, 1024), ok())
    assert rc == 1 and b"fp16 staging" in err


def test_fork_refusals(lib):
    class Alloc(ctypes.Structure):
        _fields_ = [("free_stack", ctypes.c_void_p), ("n_free", ctypes.c_void_p), ("in_use", ctypes.c_void_p),
                    ("num_pages", ctypes.c_int64)]

    lay, ptrs = Layout(0, 1, 16, 4, 64, 64, 1024), Ptrs(*([A] * 6))

    def call(al=Alloc(A, A, A, 1024), layers=2, src=A, ws=A, ws_bytes=1 << 20, ptrs=ptrs, pairs=3):
        rc = lib.mg_fork_sequences(ctypes.byref(al), ctypes.byref(lay), ctypes.byref(ptrs), layers, ctypes.c_void_p(A),
                                   ctypes.c_void_p(A), 8, ctypes.c_void_p(src), ctypes.c_void_p(A), None, pairs,
                                   ctypes.c_void_p(ws), ctypes.c_int64(ws_bytes), None, None)
        return rc, lib.mg_last_error()

    assert lib.mg_fork_workspace_bytes(3) == 20
    for kw, text in ((dict(al=Alloc(A, A, A, 1000)), b"page counts"), (dict(al=Alloc(A, None, A, 1024)), b"allocator"),
                     (dict(layers=0), b"num_layers"), (dict(src=None), b"null"), (dict(ws_bytes=16), b"workspace"),
                     (dict(ptrs=Ptrs(A + 8, A, A, A, A, A)), b"16-byte"), (dict(pairs=-1), b"num_pairs")):
        rc, err = call(**kw)
        assert rc == 1 and text in err, (kw, err)
    assert call(pairs=0)[0] == 0


def test_qk_norm_refusals(lib):
    def call(stride=640, rows=2, hq=4, hkv=3, d=64, table=8, eps=1e-5, q=A):
        p = ctypes.c_void_p(A)
        rc = lib.mg_qk_norm_rope_f16(p, ctypes.c_int64(stride), p, p, p, p, p, ctypes.c_int64(table),
                                     ctypes.c_float(eps), ctypes.c_void_p(q), p, None, ctypes.c_int64(rows), hq, hkv, d,
                                     None, None)
        return rc, lib.mg_last_error()

    for kw, text in ((dict(stride=639), b"row stride"), (dict(d=63), b"even"), (dict(rows=-1), b"rows"),
                     (dict(table=0), b"tables"), (dict(eps=-1.0), b"eps"), (dict(q=None), b"null"),
                     (dict(hkv=0), b"head counts")):
        rc, err = call(**kw)
        assert rc == 1 and text in err, (kw, err)
    assert call(rows=0)[0] == 0


@pytest.mark.parametrize("page,blocks,fits", [(16, (1 << 22) - 2, True), (16, (1 << 22) - 1, False), (64, 1 << 20, False)])
def test_contexts_of_2_to_the_26_tokens_are_refused(lib, page, blocks, fits):
    lay = Layout(0, 1, page, 4, 64, blocks, 1 << 23)
    size = lib.mg_tree_plan_bytes(ctypes.byref(lay), 2, 4, 32)
    assert (size > 0) == fits
    assert fits or b"2^26" in lib.mg_last_error()
