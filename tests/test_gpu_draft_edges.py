"""Draft trees at the edges of what a cache holds, on the GPU: trees that go on behind the page table's end, pages that are
not there, in the tokens before a tree and inside it, and entries kept in more layers than a wave takes at once."""
import numpy as np
import pytest
import torch

from oracle import attn as A
from oracle import draft as R
from tests.conftest import gpu_note
from tests.test_gpu_attn import Setup, dev
from tests.test_gpu_draft import check_tree_attend, random_tree, tree_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


# (D, n_kv, group, page, tokens, nodes, type): few columns, whole and split over the tokens; wide tiles, whole and split
SIZES = [(64, 1, 4, 16, 120, 40, "f16"), (128, 4, 8, 16, 52, 30, "bf16"), (256, 1, 2, 32, 500, 60, "f16"), (128, 2, 8, 64, 5000, 70, "bf16"),
         (128, 8, 8, 16, 260, 200, "f16"), (64, 8, 8, 32, 330, 300, "bf16"), (256, 8, 8, 64, 400, 250, "bf16"), (128, 8, 8, 64, 3000, 300, "f16")]


def without(parent, lost):
    """The tree in which the nodes of `lost`, and what follows them, are none: what such rows have in common with those
    whose tokens are not there is that they are NaN."""
    return [-5 if j in lost else p for j, p in enumerate(parent)]


@pytest.mark.parametrize("case", SIZES, ids=str)
@pytest.mark.parametrize("late", [False, True])
def test_a_tree_behind_the_tables_end(case, late):
    """Rows at a place behind the table's end are NaN, whether or not they follow the node that is the first there, and whether
    or not they are nodes; all others are as they are with a longer table."""
    from tinygiant_amd.attn import KVBatch
    D, n_kv, G, page, n, new, dt = case
    gpu_note(f"attend tree behind the table {case} {late}")
    s = Setup(n + late, D, n_kv, page, [n, n // 2], [new, 7])
    q, qn = s.rows(n_kv * G, dt)
    base = n - new
    cols = (n - 4) // page if late else base // page + 1  # some of sequence 0's nodes have their places
    cap = cols * page
    assert base < cap <= n - 4
    for bad in (False, True):
        parents = [random_tree(s.rng, new), random_tree(s.rng, 7)]
        # all kinds: nodes that follow the first one behind the end, others that follow nodes before it
        at = cap - base
        for j in range(at + 1, new):
            parents[0][j] = int(s.rng.integers(0, at)) if j % 3 else int(s.rng.integers(at, j))
        if bad:
            parents[0][at + 2] = at + 2
            parents[0][at] = -3
        # sequence 1 may be longer than the short table too
        end1 = max(0, cap - (n // 2 - 7))
        for hint in (n, 1):
            b = KVBatch(s.batch.cu, s.batch.kv_len, dev(s.table[:, :cols]), max_len=hint)
            out = s.kv.attend(0, q, b, tree=tree_of(s, parents, 320))
            assert torch.isnan(out[at:new]).all()
            check_tree_attend(s, [without(parents[0], range(at, new)), without(parents[1], range(end1, 7))], q, qn, out, max_nodes=320)


@pytest.mark.parametrize("case", SIZES, ids=str)
def test_pages_that_are_not_there(case):
    """Before a tree: all of its rows need them.  Inside it: the rows whose own place or ancestors they are; the
    others, and the other sequence, are as exact as ever."""
    from tinygiant_amd.attn import KVBatch
    D, n_kv, G, page, n, new, dt = case
    gpu_note(f"attend tree without pages {case}")
    s = Setup(n + 9, D, n_kv, page, [n, n // 2], [new, 7])
    q, qn = s.rows(n_kv * G, dt)
    parents = [random_tree(s.rng, new), random_tree(s.rng, 7)]
    tree = tree_of(s, parents, 320)
    base = n - new
    for col in sorted({0, (base + new // 2) // page, (n - 1) // page}):
        for none in (-1, len(s.cache.pages)):
            table = s.table.copy()
            table[0, col] = none
            out = s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=n), tree=tree)
            first, end = col * page - base, col * page + page - base
            lost = range(new) if first < 0 else range(first, min(end, new))
            check_tree_attend(s, [without(parents[0], lost), parents[1]], q, qn, out, max_nodes=320)


def test_a_second_tree_behind_a_table_of_768_tokens():
    """800 tokens, of which the table holds 768: those of the second tree's 150 nodes that are behind it do not follow the
    first of them, and are NaN all the same."""
    from tinygiant_amd.attn import KVBatch, PagedKV
    from tinygiant_amd.draft import DraftTree
    gpu_note("attend tree, 768 of 800 tokens")
    D, n_kv, G, page, n = 256, 8, 16, 128, 300
    rng = np.random.default_rng(9)
    kv = PagedKV(1, 12, page, n_kv, D)
    table = rng.permutation(12).reshape(2, 6).astype(np.int32)
    lens, news = np.array([600, 500 + n], np.int32), np.array([n, n // 2], np.int32)
    cu0, cu = (np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (lens - news, news))
    parent = np.concatenate([random_tree(rng, k) for k in news]).astype(np.int32)
    bits = R.seen(parent[cu[1]:])
    first = 768 - 650
    assert not bits[first + 1:, first].any()
    tree = DraftTree(dev(cu), int(cu[-1]), dev(parent), max_nodes=n)
    torch.manual_seed(3)
    rows = lambda k, h: torch.randn(int(k), h, D, device="cuda").to(torch.bfloat16)  # noqa: E731
    past, new, q = rows(cu0[-1], n_kv), rows(cu[-1], n_kv), rows(cu[-1], n_kv * G)
    kv.append(0, None, past, past, KVBatch(dev(cu0), dev(lens - news), dev(table)))
    b = KVBatch(dev(cu), dev(lens), dev(table))
    kv.append(0, None, new, new, b, tree=tree)
    nan = torch.isnan(kv.attend(0, q, b, tree=tree).float()).flatten(1)
    assert nan[cu[1] + first:].all() and not nan[:cu[1] + first].any()


@pytest.mark.parametrize("D,n_kv,page,lens,news,layers,layer,n_layers", [
    (128, 4, 16, [60, 9], [16, 3], 5, 0, 5), (64, 3, 32, [200, 70, 40, 33], [33, 9, 0, 30], 8, 0, 8), (256, 1, 16, [90, 300], [64, 5], 9, 0, 9),
    (128, 2, 48, [100 + 3 * i for i in range(20)], [1 + i % 9 for i in range(20)], 7, 1, 6), (64, 2, 16, [50, 31], [9, 4], 11, 2, 7)], ids=str)
def test_keep_of_many_layers(D, n_kv, page, lens, news, layers, layer, n_layers):
    """More layers than a wave has at once, groups that are full and that are not; the layers beside them stay as they were."""
    gpu_note(f"keep {layers} layers from {layer} on {n_layers}")
    s = Setup(layers, D, n_kv, page, lens, news, layers=layers)
    paths, count = np.full((len(lens), max(news)), 999, np.int32), np.zeros(len(lens), np.int32)
    for i, n in enumerate(news):
        kept = sorted(s.rng.choice(n, size=s.rng.integers(1, n + 1), replace=False)) if n else []
        paths[i, :len(kept)], count[i] = kept, len(kept)
    s.kv.keep(s.batch, dev(paths), dev(count), layer=layer, n_layers=n_layers)
    for at in range(layer, layer + n_layers):
        c = A.Cache(len(s.cache.pages), page, n_kv, D, s.all[at])
        for i, n in enumerate(lens):
            R.keep(c, s.table[i], n, news[i], paths[i, :count[i]])
    assert np.array_equal(s.kv.pages.cpu().numpy(), s.all)


@pytest.mark.parametrize("case", SIZES + [(128, 4, 8, 64, 9000, 40, "bf16")], ids=str)
def test_the_same_tree_gives_the_same_bits(case):
    D, n_kv, G, page, n, new, dt = case
    gpu_note(f"attend tree again {case}")
    s = Setup(n, D, n_kv, page, [n, n // 2, 11], [new, 7, 3])
    q, _ = s.rows(n_kv * G, dt)
    tree = tree_of(s, [random_tree(s.rng, k) for k in (new, 7, 3)], 320)
    want = s.kv.attend(0, q, s.batch, tree=tree)
    for _ in range(4):
        s.rows(n_kv * G, dt)[0].sum().item()
        assert torch.equal(s.kv.attend(0, q, s.batch, tree=tree), want)


def test_one_column_of_any_stride():
    """Of a path of one column, or a page table of one, the columns' stride counts for nothing."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("keep and attend, one column")
    s = Setup(8, 64, 2, 64, [40, 33, 64], [6, 9, 1])
    table, path = (dev(x).reshape(1, -1).t() for x in (s.table, np.zeros(3, np.int32)))
    assert table.stride() == path.stride() == (1, 3)
    b = KVBatch(s.batch.cu, s.batch.kv_len, table, max_len=64)
    q, _ = s.rows(4, "f16")
    assert torch.equal(s.kv.attend(0, q, b), s.kv.attend(0, q, s.batch))
    got = s.kv.keep(b, path, dev(np.ones(3, np.int32)), kv_len=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert got.tolist() == [35, 25, 64]
