"""Calls of the attention block that its documentation allows, each of which
once went wrong: views of page tables, blocks that are not finite next to
others, rows that are not all there, scores beyond ordinary sizes.  Bounds are
those of test_gpu_attn.py."""
import numpy as np
import pytest
import torch

from oracle import attn as A
from tests.conftest import gpu_note
from tests.test_gpu_attn import DT, Setup, check_attend, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 40, 100]])
@pytest.mark.parametrize("view", ["expanded", "columns", "every other row"])
def test_views_of_page_tables(view, news):
    """One row expanded to all sequences (a prefix that they share), columns and rows of a wider table."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"table views {view} {news}")
    lens = [70, 90, 110]
    s = Setup(51, 128, 2, 16, lens, news)
    if view == "expanded":
        s.table[:] = s.table[2]
        table = dev(s.table[2]).expand(3, -1)
    elif view == "columns":
        table = torch.full((3, s.table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")[:, 2:-3]
    else:
        table = torch.full((5, s.table.shape[1]), -9, dtype=torch.int32, device="cuda")[::2]
    if view != "expanded":
        table.copy_(dev(s.table))
    batch = KVBatch(s.batch.cu, s.batch.kv_len, table, max_len=110)
    q, qn = s.rows(8, "bf16")
    check_attend(s, q, qn, s.kv.attend(0, q, batch))
    k, v = s.kv.read(0, batch, s.T)
    for i, (n, new) in enumerate(zip(lens, news)):
        kr, vr = s.cache.rows(s.table[i], n)
        for got, ref in ((k, kr), (v, vr)):
            assert np.array_equal(got[s.cu[i]:s.cu[i + 1]].cpu().numpy(), ref[:, n - new:].transpose(1, 0, 2).astype(np.float16))


def test_overlapping_rows_of_a_page_table_are_refused():
    from tinygiant_amd.attn import KVBatch
    s = Setup(52, 64, 1, 16, [40, 40], [1, 1])
    with pytest.raises(ValueError, match="overlap"):
        KVBatch(s.batch.cu, s.batch.kv_len, torch.as_strided(s.batch.table, (2, 3), (1, 1)))
