"""What attention asks for beside its tensors.  Sizes alone, so these run without a GPU."""
import ctypes

import pytest

from tinygiant_amd import _lib
from tests.test_attn_args import INVALID, P, attend, batch, said


@pytest.fixture(scope="module")
def lib():
    return _lib.require_lib()


# (n_seqs, rows, key heads, heads, dims, tokens), column tiles, places of partial results for a key head and their columns
CASES = [((16, 192, 4, 32, 128, 8192), 112, 256, 16),   # 12 rows each: 96 columns a sequence, the few-column kernel's
         ((1, 1, 4, 32, 128, 8192), 1, 256, 16),
         ((64, 64, 8, 32, 64, 4096), 80, 128, 16),
         ((4, 400, 4, 32, 128, 8192), 16, 128, 256)]    # 800 columns a sequence: wide tiles


@pytest.mark.parametrize("case,tiles,parts,cols", CASES, ids=str)
def test_ordinary_calls_ask_for_what_they_use(lib, case, tiles, parts, cols):
    """Of each key head partial results of `cols` columns (dims, largest score, sum), twice as many as the blocks that a
    launch has for it, and 16 bytes for each column tile that is joined."""
    seqs, rows, kv, heads, D, tokens = case
    b = batch(n_seqs=seqs, n_tokens=rows, n_kv_heads=kv, head_dim=D, page_tokens=64, table_cols=tokens // 64, table_stride=tokens // 64)
    need = lib.tg_attn_q4_workspace(ctypes.byref(b), heads, tokens)
    partial = parts * kv * cols * (D + 2) * 4
    assert partial <= need <= partial + tiles * kv * 16 + 256, (need, partial)


def test_trees_ask_for_their_own(lib):
    """A tree's sizes may choose the other kernel, which needs more: that is what its own function says, and what its call
    asks for."""
    b = batch(n_seqs=16, n_tokens=192, n_kv_heads=4, head_dim=128, page_tokens=64, table_cols=128, table_stride=128)
    ref = ctypes.byref(b)
    few, tree = lib.tg_attn_q4_workspace(ref, 32, 8192), lib.tg_attn_tree_q4_workspace(ref, 32, 8192)
    assert 0 < few < tree
    assert attend(lib, b, heads=32, qs=4096, os=4096, max_len=8192, n=few - 1) == INVALID and f"{few} and" in said(lib)
    assert lib.tg_attn_tree_q4_dev(ref, P, 2, 1, P, 4096, 32, 0.1, 2 * P, 4096, 8192, P, tree - 1, None) == INVALID
    assert f"tg_attn_tree_q4_dev: workspace of {tree - 1} bytes, {tree} and" in said(lib)
    assert lib.tg_attn_tree_q4_workspace(ctypes.byref(batch(head_dim=96)), 8, 0) == 0
    assert lib.tg_attn_tree_q4_workspace(None, 8, 0) == 0
