"""What the draft trees' entry points refuse, by the C ABI and by the Python
wrappers.  No call reaches a kernel, so these run without a GPU."""
import ctypes

import pytest
import torch

from tinygiant_amd import _lib
from tinygiant_amd.draft import DraftTree, _Trees
from tests.test_attn_args import INVALID, P, batch, said
from tests.test_attn_calls import WIDE, batch_over, cache


@pytest.fixture(scope="module")
def lib():
    return _lib.require_lib()


def trees(**kw):
    d = dict(cu=P, parent=P, n_seqs=1, n_tokens=3, max_nodes=64)
    d.update(kw)
    return _Trees(*[d[n] for n, _ in _Trees._fields_])


BAD_TREES = [(dict(cu=None), "cu is NULL"), (dict(n_seqs=-1), "n_seqs -1"), (dict(n_tokens=-1), "n_tokens -1"),
             (dict(max_nodes=0), "max_nodes 0"), (dict(max_nodes=1025), "max_nodes 1025")]


@pytest.mark.parametrize("kw,msg", BAD_TREES)
def test_trees_are_refused(lib, kw, msg):
    assert lib.tg_draft_tree_dev(ctypes.byref(trees(**kw)), P, P, P, None) == INVALID and msg in said(lib)


def test_tree_refuses(lib):
    t = trees()
    assert lib.tg_draft_tree_dev(None, P, P, P, None) == INVALID and "trees is NULL" in said(lib)
    assert lib.tg_draft_tree_dev(ctypes.byref(t), None, P, P, None) == INVALID
    assert lib.tg_draft_tree_dev(ctypes.byref(t), P, None, P, None) == INVALID
    assert lib.tg_draft_tree_dev(ctypes.byref(t), P, P, None, None) == INVALID and "links is NULL" in said(lib)
    for kw in (dict(n_seqs=0), dict(n_tokens=0)):
        assert lib.tg_draft_tree_dev(ctypes.byref(trees(**kw)), P, P, P, None) == 0


def test_append_and_attend_of_trees_refuse(lib):
    """Their own arguments; the others are those of the calls without trees."""
    b = ctypes.byref(batch())
    rows = (2, P, 1024, P, 256, P, 256, P, 1024, 8, None, None, 1e-6, P, P, 64, None)
    assert lib.tg_kv_append_tree_q4_dev(b, None, *rows) == INVALID and "depth is NULL" in said(lib)
    assert lib.tg_kv_append_tree_q4_dev(b, P, 3, *rows[1:]) == INVALID and "tg_kv_append_tree_q4_dev: element type 3" in said(lib)
    rows = (1, P, 1024, 8, 0.1, 2 * P, 1024, 0, P, 1 << 40, None)
    assert lib.tg_attn_tree_q4_dev(b, None, 2, *rows) == INVALID and "bits is NULL" in said(lib)
    for words in (0, 33, -1):
        assert lib.tg_attn_tree_q4_dev(b, P, words, *rows) == INVALID and f"{words} words" in said(lib)
    assert lib.tg_attn_tree_q4_dev(b, P, 2, 0, *rows[1:]) == INVALID and "tg_attn_tree_q4_dev: element type 0" in said(lib)
    for kw in (dict(n_tokens=0), dict(n_seqs=0)):
        assert lib.tg_attn_tree_q4_dev(ctypes.byref(batch(**kw)), P, 2, *rows) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(n_layers=-1), "-1 layers"), (dict(layer_bytes=18 * 128 * 8 - 16), "layers"), (dict(layer_bytes=18 * 128 * 8 + 8), "layers"),
    (dict(path=None), "path or count"), (dict(count=None), "path or count"), (dict(cols=0), "0 columns"), (dict(stride=3), "3 apart"),
    (dict(n_layers=65537, layer_bytes=1 << 30), "65537 layers")])
def test_keep_refuses(lib, kw, msg):
    d = dict(n_layers=2, layer_bytes=18 * 128 * 8, path=P, stride=4, cols=4, count=P, kv_len=None)
    d.update(kw)
    args = (d["n_layers"], d["layer_bytes"], d["path"], d["stride"], d["cols"], d["count"], d["kv_len"], None)
    assert lib.tg_kv_keep_q4_dev(ctypes.byref(batch()), *args) == INVALID and msg in said(lib)
    assert lib.tg_kv_keep_q4_dev(None, *args) == INVALID and "batch is NULL" in said(lib)
    assert lib.tg_kv_keep_q4_dev(ctypes.byref(batch(n_seqs=0)), 2, 18 * 128 * 8, P, 4, 4, P, None, None) == 0


def test_keep_refuses_more_than_a_launch_takes(lib):
    b = batch(n_seqs=1 << 20, n_kv_heads=8)
    assert lib.tg_kv_keep_q4_dev(ctypes.byref(b), 48, 1 << 40, P, 4, 4, P, None, None) == INVALID and "than a launch takes" in said(lib)


def test_python_refuses():
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError, match="cu must be"):
        DraftTree(i, 4)
    kv, b = cache(), batch_over(WIDE[:1])

    class Tree:
        device, n_seqs, n_tokens = b.device, 1, 2

    q = torch.zeros(3, 2, 64)
    for call in (lambda t: kv.attend(0, q.half(), b, tree=t), lambda t: kv.append(0, None, q, q, b, tree=t)):
        for change in (dict(n_tokens=2), dict(n_seqs=2, n_tokens=3), dict(device=torch.device("meta"), n_tokens=3)):
            t = Tree()
            t.__dict__.update(change)
            with pytest.raises(ValueError, match="tree of"):
                call(t)
    with pytest.raises(TypeError, match="path must be"):
        kv.keep(b, WIDE[:1], i[:1])
    for layer, n in ((-1, 1), (0, 2), (2, None), (1, -1)):
        with pytest.raises(ValueError, match="layers"):
            kv.keep(b, WIDE[:1], i[:1], layer=layer, n_layers=n)


# ---------------------------------------------------------------- verify
def verify_args(lib, t=None, **kw):
    d = dict(links=P, type=0, logits=P, stride=100, draft=P, dstride=100, vocab=100, tokens=P, u=P, temp=1.0, temps=None, out=P, path=P,
             count=P, ws=P, n=1 << 40)
    d.update(kw)
    return lib.tg_verify_dev(ctypes.byref(t if t is not None else trees()), *[d[n] for n in (
        "links", "type", "logits", "stride", "draft", "dstride", "vocab", "tokens", "u", "temp", "temps", "out", "path", "count", "ws", "n")], None)


@pytest.mark.parametrize("kw,msg", BAD_TREES)
def test_verify_refuses_trees(lib, kw, msg):
    t = trees(**kw)
    assert verify_args(lib, t) == INVALID and msg in said(lib)
    assert lib.tg_verify_workspace(ctypes.byref(t), 100) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "element type 3"), (dict(links=None), "NULL"), (dict(logits=None), "NULL"), (dict(tokens=None), "NULL"), (dict(u=None), "NULL"),
    (dict(out=None), "NULL"), (dict(path=None), "NULL"), (dict(count=None), "NULL"), (dict(vocab=0), "vocab 0"),
    (dict(vocab=(1 << 20) + 1, stride=1 << 25), "vocab 1048577"), (dict(stride=99), "overlap"), (dict(dstride=99), "overlap"),
    (dict(logits=P + 2), "aligned"), (dict(draft=P + 1, type=1), "aligned"), (dict(temp=float("inf")), "temperature inf"),
    (dict(ws=None), "workspace"), (dict(n=8), "workspace"), (dict(ws=P + 8), "workspace")])
def test_verify_refuses(lib, kw, msg):
    assert verify_args(lib, **kw) == INVALID and msg in said(lib)


def test_verify_refuses_more_than_a_launch_takes(lib):
    t = trees(n_tokens=1 << 20, n_seqs=1 << 14)
    assert lib.tg_verify_workspace(ctypes.byref(t), 1 << 18) == 0
    assert verify_args(lib, t, vocab=1 << 18, stride=1 << 18, draft=None) == INVALID and "than a launch takes" in said(lib)


def test_verify_of_nothing(lib):
    assert verify_args(lib, trees(n_seqs=0)) == 0


def test_python_verify_refuses():
    from tinygiant_amd.draft import verify

    with pytest.raises(TypeError, match="logits must be"):
        verify(torch.zeros(3, 9), None, None, None)
