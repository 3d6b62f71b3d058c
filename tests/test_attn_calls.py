"""How the attention block's Python side hands its tensors to the C ABI.  No call reaches a kernel, so these run without
a GPU; objects are made of host tensors around the constructors, which take only the device's."""
import ctypes

import pytest
import torch

from tinygiant_amd import _lib
from tinygiant_amd.attn import KVBatch, PagedKV, table_stride


def cache(head_dim=64, n_kv=2, page=16, n_pages=4):
    kv = PagedKV.__new__(PagedKV)
    kv.pages = torch.zeros(1, n_pages, n_kv, page // 16, 18 * head_dim, dtype=torch.uint8)
    kv.device, kv.n_layers, kv.n_pages, kv.page_tokens, kv.n_kv_heads, kv.head_dim = kv.pages.device, 1, n_pages, page, n_kv, head_dim
    kv.layer_bytes = kv.pages.stride(0)
    return kv


def batch_over(table):
    b = KVBatch.__new__(KVBatch)
    n = table.shape[0]
    b.cu, b.kv_len, b.table = torch.arange(n + 1, dtype=torch.int32), torch.ones(n, dtype=torch.int32), table
    b.max_len, b.n_seqs, b.device = 0, n, table.device
    return b


WIDE = torch.arange(60, dtype=torch.int32).view(5, 12)


@pytest.mark.parametrize("table", [
    WIDE, WIDE[:, :4], WIDE[::2, 3:7], WIDE[1:2], WIDE[0].expand(3, 12), WIDE[0, :4].expand(5, 4), WIDE[2:3, :4].expand(1, 4),
    WIDE[:, :1], WIDE[0, :1].expand(7, 1)], ids=lambda t: f"{tuple(t.shape)}x{t.stride()}")
def test_every_entry_of_the_table_is_where_the_kernels_look(table):
    """Entry (s, c) at table + s * table_stride + c, whatever view the table is."""
    b = cache()._batch(0, batch_over(table), 3)
    flat = torch.as_strided(table, (table.untyped_storage().nbytes() // 4 - table.storage_offset(),), (1,))
    assert b.table == table.data_ptr() and b.table_cols == table.shape[1]
    for s in range(table.shape[0]):
        for c in range(table.shape[1]):
            at = s * b.table_stride + c
            assert at < len(flat) and flat[at] == table[s, c], (s, c, b.table_stride)


def test_a_table_whose_rows_overlap_is_refused():
    for rows in (2, 3):
        t = torch.as_strided(WIDE, (rows, 4), (2, 1))
        with pytest.raises(ValueError, match="overlap"):
            table_stride(t)
    assert table_stride(torch.as_strided(WIDE, (1, 4), (2, 1))) >= 4  # one row overlaps nothing


def test_one_row_for_every_sequence_is_taken_by_the_c_side():
    lib = _lib.require_lib()
    b = cache()._batch(0, batch_over(WIDE[0].expand(3, 12)), 0)  # no rows: checked, nothing launched
    P = 1 << 20
    assert b.table_stride == 0 and lib.tg_kv_read_q4_dev(ctypes.byref(b), P, P, None) == 0
    b.table_stride = 5
    assert lib.tg_kv_read_q4_dev(ctypes.byref(b), P, P, None) == -1 and "5 apart" in lib.tg_last_error().decode()


@pytest.mark.parametrize("M,N,K", [(1, (1 << 31) - 1, 16), ((1 << 31) - 1, 1, 16), ((1 << 30) + 1, 16, 16), (7, (1 << 30) + 1, 128),
                                   (1 << 27, 16, 16), (1 << 24, 16, 1024), (1 << 20, 1 << 21, 64)])
def test_products_that_no_launch_takes_are_refused(M, N, K):
    """Before a device is looked for: rows or channels beyond 32-bit indexes, or beyond a launch's threads."""
    lib = _lib.require_lib()
    P = 1 << 20
    assert lib.tg_matmul_i8_workspace(M, N, K) == 0
    assert lib.tg_matmul_i8_dev(P, 1, K, None, 1e-6, P, P, None, 0, 2 * P, 1, N, M, N, K, P, 1 << 60, None) == -1
    assert "than a launch takes" in lib.tg_last_error().decode()


@pytest.mark.parametrize("M,N,K", [(1, 1 << 29, 16), ((1 << 26) - 4, 16, 512), ((1 << 24) - 1, 16, 1024), (0, 1 << 30, 16), (1 << 15, 1 << 15, 4096)])
def test_the_largest_products_are_taken(M, N, K):
    assert _lib.require_lib().tg_matmul_i8_workspace(M, N, K) >= M * K


def test_gradients_are_refused_where_torch_records_them():
    """And only there: without them the calls go on, here to the layer that there is not."""
    kv, b = cache(), batch_over(WIDE[:1])
    z = lambda *shape: torch.zeros(*shape)
    attend = dict(q=z(1, 2, 64).half(), out=z(1, 2, 64).half())
    append = dict(q=z(1, 2, 64), k=z(1, 2, 64), v=z(1, 2, 64), cos=z(9, 32), sin=z(9, 32), q_norm=z(64), k_norm=z(64), out=z(1, 2, 64))
    for args, name in ((attend, "attend"), (append, "append")):
        for one in args:
            leaf = dict(args, **{one: args[one].clone().requires_grad_()})
            with pytest.raises(RuntimeError, match=f"{name} has no gradients"):
                getattr(kv, name)(7, batch=b, **leaf)
            with torch.no_grad(), pytest.raises(ValueError, match="layer 7"):
                getattr(kv, name)(7, batch=b, **leaf)
        with pytest.raises(ValueError, match="layer 7"):
            getattr(kv, name)(7, batch=b, **args)


def test_one_row_has_no_row_stride():
    """A row of a tensor of any width: there is no next one, so its stride is never what a call is refused for."""
    kv = cache()
    for width in (131, 130, 5 * 64):
        x = torch.zeros(3, width)[1:2, :128]
        for t in (x, x.view(1, 2, 64)):
            assert kv._rows(t, "k", 2, torch.float32, 1) == 128
    assert kv._rows(torch.zeros(3, 192)[:, :128], "k", 2, torch.float32, 3) == 192
