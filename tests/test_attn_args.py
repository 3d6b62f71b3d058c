"""What the attention block's entry points refuse, by the C ABI and by the
Python wrappers.  No call reaches a kernel, so these run without a GPU."""
import ctypes

import pytest
import torch

from tinygiant_amd import _lib
from tinygiant_amd.attn import KVBatch, PagedKV, _Batch
from tinygiant_amd.linear import matmul_i8

P = 1 << 20  # an address that is aligned and never read
INVALID = -1


@pytest.fixture(scope="module")
def lib():
    return _lib.require_lib()


def batch(**kw):
    d = dict(pages=P, table=P, cu=P, kv_len=P, n_pages=4, page_tokens=16, n_kv_heads=2, head_dim=128, table_cols=2,
             table_stride=2, n_seqs=1, n_tokens=3)
    d.update(kw)
    return _Batch(*[d[n] for n, _ in _Batch._fields_])


BAD = [(dict(head_dim=96), "head_dim 96"), (dict(page_tokens=8), "page_tokens 8"), (dict(page_tokens=40), "page_tokens 40"),
       (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(n_pages=0), "n_pages 0"), (dict(table_cols=0), "table_cols 0"),
       (dict(table_cols=1 << 27, table_stride=1 << 27), "table_cols"), (dict(table_stride=1), "1 apart"),
       (dict(pages=None), "NULL pointer"), (dict(table=None), "NULL pointer"), (dict(cu=None), "NULL pointer"),
       (dict(kv_len=None), "NULL pointer"), (dict(pages=P + 8), "16-byte aligned"), (dict(n_seqs=-1), "n_seqs -1"),
       (dict(n_tokens=-1), "n_tokens -1")]


def append(lib, b, **kw):
    d = dict(type=2, q=P, qs=1024, k=P, ks=256, v=P, vs=256, qo=P, qos=1024, heads=8, qn=None, kn=None, eps=1e-6, c=P, s=P,
             max_pos=64)
    d.update(kw)
    return lib.tg_kv_append_q4_dev(ctypes.byref(b) if b else None, d["type"], d["q"], d["qs"], d["k"], d["ks"], d["v"], d["vs"],
                                   d["qo"], d["qos"], d["heads"], d["qn"], d["kn"], d["eps"], d["c"], d["s"], d["max_pos"], None)


def attend(lib, b, **kw):
    d = dict(type=1, q=P, qs=1024, heads=8, scale=0.1, out=P, os=1024, max_len=0, ws=P, n=1 << 40)
    d.update(kw)
    return lib.tg_attn_q4_dev(ctypes.byref(b) if b else None, d["type"], d["q"], d["qs"], d["heads"], d["scale"], d["out"],
                              d["os"], d["max_len"], d["ws"], d["n"], None)


def product(lib, **kw):
    d = dict(x=P, xt=0, xs=64, norm=None, w=P, ws=P, res=None, rs=0, out=P, ot=0, os=32, M=2, N=32, K=64, work=P, n=1 << 40)
    d.update(kw)
    return lib.tg_matmul_i8_dev(d["x"], d["xt"], d["xs"], d["norm"], 1e-6, d["w"], d["ws"], d["res"], d["rs"], d["out"], d["ot"],
                                d["os"], d["M"], d["N"], d["K"], d["work"], d["n"], None)


def said(lib):
    return lib.tg_last_error().decode()


@pytest.mark.parametrize("kw,msg", BAD)
def test_batch_is_refused_everywhere(lib, kw, msg):
    for call in (append, attend, lambda L, b: L.tg_kv_read_q4_dev(ctypes.byref(b), P, P, None)):
        assert call(lib, batch(**kw)) == INVALID
        assert msg in said(lib)
    assert lib.tg_attn_q4_workspace(ctypes.byref(batch(**kw)), 8, 0) == 0


def test_null_batch(lib):
    assert append(lib, None) == INVALID and "batch is NULL" in said(lib)
    assert attend(lib, None) == INVALID and lib.tg_kv_read_q4_dev(None, P, P, None) == INVALID
    assert lib.tg_attn_q4_workspace(None, 8, 0) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "element type 3"), (dict(heads=0), "n_heads 0"), (dict(q=None), "q NULL"), (dict(qo=None), "q_out is NULL"),
    (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(qs=1000), "q rows"), (dict(ks=258), "k rows"),
    (dict(v=P + 2), "v rows"), (dict(k=P + 4), "k rows"), (dict(type=0, k=P + 8), "k rows"), (dict(c=None), "rope_cos and rope_sin"),
    (dict(max_pos=0), "max_pos 0"), (dict(qn=P + 4), "16-byte aligned"), (dict(qos=512), "q_out rows"),
    (dict(heads=-1), "n_heads -1")])
def test_append_refuses(lib, kw, msg):
    assert append(lib, batch(), **kw) == INVALID
    assert msg in said(lib)


@pytest.mark.parametrize("kw,msg", [
    (dict(type=0), "element type 0"), (dict(heads=7), "n_heads 7"), (dict(heads=0), "n_heads 0"), (dict(q=None), "q is NULL"),
    (dict(out=None), "out is NULL"), (dict(qs=1028), "q rows"), (dict(q=P + 8), "q rows"), (dict(os=512), "out rows"),
    (dict(scale=0.0), "scale 0"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(max_len=-1), "max_len -1")])
def test_attend_refuses(lib, kw, msg):
    assert attend(lib, batch(), **kw) == INVALID
    assert msg in said(lib)


def test_attend_refuses_a_small_workspace(lib):
    b = batch(n_pages=10000, table_cols=8192, table_stride=8192, page_tokens=64)
    need = lib.tg_attn_q4_workspace(ctypes.byref(b), 8, 0)
    if need:
        assert attend(lib, b, n=need - 1) == INVALID and "workspace" in said(lib)
        assert attend(lib, b, ws=None) == INVALID and "workspace" in said(lib)
        assert attend(lib, b, ws=P + 8) == INVALID and "workspace" in said(lib)


def test_read_refuses(lib):
    b = batch()
    for k, v in ((None, P), (P, None), (P + 2, P), (P, P + 8)):
        assert lib.tg_kv_read_q4_dev(ctypes.byref(b), k, v, None) == INVALID


@pytest.mark.parametrize("kw,msg", [
    (dict(M=-1), "M -1"), (dict(N=0), "N 0"), (dict(K=0), "K 0"), (dict(K=40, xs=64), "K 40"), (dict(K=131088, xs=1 << 20), "K 131088"),
    (dict(xt=3), "type 3"), (dict(ot=-1), "type -1"), (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(out=None), "NULL"), (dict(w=P + 4), "aligned"), (dict(xs=63), "overlap"), (dict(os=31), "overlap"),
    (dict(res=P, rs=31), "overlap")])
def test_product_refuses(lib, kw, msg):
    assert product(lib, **kw) == INVALID
    assert msg in said(lib)
    if kw.keys() & {"N", "K"}:
        assert lib.tg_matmul_i8_workspace(kw.get("M", 2), kw.get("N", 32), kw.get("K", 64)) == 0


def test_empty_calls_do_nothing(lib):
    """No rows or no sequences: OK before any device is looked for."""
    for kw in (dict(n_tokens=0), dict(n_seqs=0)):
        assert append(lib, batch(**kw)) == 0 and attend(lib, batch(**kw)) == 0
        assert lib.tg_kv_read_q4_dev(ctypes.byref(batch(**kw)), P, P, None) == 0
    assert product(lib, M=0) == 0


def test_python_refuses_host_tensors_and_shapes():
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError, match="cu"):
        KVBatch(i, i[:2], i.view(1, 3))
    for kw in (dict(head_dim=80), dict(page_tokens=24), dict(n_pages=0), dict(n_layers=0), dict(n_kv_heads=0)):
        d = dict(n_layers=1, n_pages=2, page_tokens=16, n_kv_heads=1, head_dim=64)
        d.update(kw)
        with pytest.raises(ValueError):
            PagedKV(device="cpu", **d)
    with pytest.raises(TypeError, match="pages"):
        PagedKV(1, 2, 16, 1, 64, pages=torch.zeros(1, 2, 1, 1, 18 * 64, dtype=torch.uint8))
    with pytest.raises(TypeError, match="x must be"):
        matmul_i8(torch.zeros(2, 64), torch.zeros(32, 64, dtype=torch.int8), torch.zeros(32))


def test_results_in_the_place_of_their_operands_are_refused(lib):
    assert attend(lib, batch()) == INVALID and "out is q" in said(lib)
    assert product(lib) == INVALID and "out is x" in said(lib)
