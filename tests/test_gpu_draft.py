"""Draft trees on the GPU, against oracle/draft.py: which nodes see which, rows
appended by their depth, attention of a tree's rows, and the cache after a
step.

Trees, cache bytes and rotated rows are compared exactly; attention by the
bounds of test_gpu_attn.py, which count the same kernels' roundings."""
import zlib

import numpy as np
import pytest
import torch

from oracle import attn as A
from oracle import draft as R
from tests.conftest import gpu_note
from tests.test_gpu_attn import DT, Setup, check_attend, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


def random_tree(rng, n, power=1.5):
    return [-1] + [int(j * rng.random() ** power) for j in range(1, n)] if n else []


def tree_of(s, parents, max_nodes=64):
    from tinygiant_amd.draft import DraftTree
    flat = np.concatenate([np.asarray(p, np.int32) for p in parents] + [np.full(s.T - s.cu[-1], 7, np.int32)])
    return DraftTree(s.batch.cu, s.T, dev(flat.astype(np.int32)), max_nodes=max_nodes)


def check_tree_attend(s, parents, q, qn, out, scale=None, max_nodes=1024):
    """Sequence by sequence, like check_attend but over what the trees let a row see; rows that are no nodes are NaN."""
    got = out.float().cpu().numpy().astype(np.float64)
    half, u = torch.finfo(out.dtype).eps / 2, 2.0 ** -11
    for i, (n, parent) in enumerate(zip(s.lens, parents)):
        new = len(parent)
        if not new:
            continue
        k, v = s.cache.rows(s.table[i], n)
        rows = slice(s.cu[i], s.cu[i + 1])
        node = np.array([a is not None for a in R.ancestors(parent, max_nodes)]) | (np.arange(new) < new - n)
        ref, size, top, vstep, kstep = A.attend(qn[rows], k, v, new, s.D ** -0.5 if scale is None else scale,
                                                steps=s.cache.rows(s.table[i], n, steps=True), seen=R.seen(parent, max_nodes))
        assert np.isnan(got[rows][~node]).all()
        delta = 2 * u * top + 2.0 ** -18 * (top + 1) + 2.0 ** -11 * kstep
        tol = size * (np.expm1(2 * delta) + 2 * u) + 2.0 ** -10 * vstep + half * np.abs(ref) * (1 + 1e-3) + 2.0 ** -24
        off = np.abs(got[rows] - ref)[node]
        assert (off <= tol[node]).all(), (i, n, new, np.argwhere(off > tol[node])[:5], float((off / tol[node]).max()))


# ---------------------------------------------------------------- trees
@pytest.mark.parametrize("sizes,max_nodes", [([1], 1), ([5], 64), ([31, 32, 33, 0, 1], 40), ([64, 65, 63], 64), ([1024, 3], 1024),
                                             ([1000], 1000), ([7] * 300, 9), ([20, 100], 33)], ids=str)
def test_trees(sizes, max_nodes):
    from tinygiant_amd.draft import DraftTree
    gpu_note(f"trees {sizes[:5]} {max_nodes}")
    rng = np.random.default_rng(len(sizes) + max_nodes)
    cu = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    for kind in ("random", "chain", "bush", "roots", "bad", "none"):
        parents = []
        for n in sizes:
            p = random_tree(rng, n)
            if kind in ("chain", "none"):
                p = list(range(-1, n - 1))
            elif kind == "bush":
                p = [-1] + [0] * (n - 1) if n else []
            elif kind == "roots":
                p = [-1 if rng.random() < 0.3 else x for x in p]
            elif kind == "bad":
                p = [int(rng.choice([j, j + 1, -2, 10 ** 9, -10 ** 9, n])) if rng.random() < 0.1 else x for j, x in enumerate(p)]
            parents.append(p)
        T = int(cu[-1]) + 3
        flat = np.concatenate([np.asarray(p, np.int64) for p in parents] + [np.zeros(3, np.int64)]).astype(np.int32)
        tree = DraftTree(dev(cu), T, None if kind == "none" else dev(flat), max_nodes=max_nodes)
        tree.bits.fill_(77)
        tree.depth.fill_(77)
        tree.links.fill_(77)
        tree.build()
        links = tree.links.cpu().numpy()
        bits, depth = tree.bits.cpu().numpy().view(np.uint32), tree.depth.cpu().numpy()
        for i, p in enumerate(parents):
            want = R.words(p, max_nodes)
            assert np.array_equal(bits[cu[i]:cu[i + 1]], want[0]), (kind, i)
            assert np.array_equal(depth[cu[i]:cu[i + 1]], want[1]), (kind, i)
            follow = [j in [q for k, q in enumerate(p[:max_nodes]) if 0 <= q < k] for j in range(len(p))]
            assert links[cu[i]:cu[i + 1]].tolist() == [-1 if want[1][j] < 0 else 2 * i + follow[j] for j in range(len(p))], (kind, i)
        assert (bits[cu[-1]:] == 77).all() and (depth[cu[-1]:] == 77).all() and (links[cu[-1]:] == -1).all()


def test_trees_of_fewer_rows_than_counted():
    from tinygiant_amd.draft import DraftTree
    gpu_note("trees cut off")
    p = [-1, 0, 1, 1, 3, 0]
    tree = DraftTree(dev(np.array([0, 6, 9], np.int32)), 4, dev(np.array(p[:4], np.int32)))
    assert np.array_equal(tree.depth.cpu().numpy(), R.words(p[:4], 64)[1])


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("case", [
    (128, 4, 8, 16, [60], [16], "bf16"), (64, 2, 3, 32, [200, 9, 70, 40], [33, 9, 0, 1], "f32"), (256, 1, 4, 16, [90, 300], [64, 5], "f16"),
    (128, 2, 16, 64, [100 + 3 * i for i in range(70)], [1 + i % 9 for i in range(70)], "f16")], ids=str)
def test_append(case):
    """Each node at its place, rotated by its depth; places behind the rotation tables' end are no positions."""
    D, n_kv, G, page, lens, news, dt = case
    gpu_note(f"append tree {case[:6]}")
    s = Setup(zlib.crc32(str(case).encode()) % 1000, D, n_kv, page, lens, news, pad=2, layers=2, layer=1)
    parents = [random_tree(s.rng, n) for n in news]
    tree = tree_of(s, parents)
    heads = n_kv * G
    x, xn = s.rows(heads + 2 * n_kv, dt)
    q, k, v = x.split([heads, n_kv, n_kv], 1)
    qh, kh, vh = np.split(xn, [heads, heads + n_kv], 1)
    depth = np.concatenate([R.words(p, 64)[1] for p in parents])
    base = np.concatenate([np.full(len(p), n - len(p)) for n, p in zip(lens, parents)])
    max_pos = int((base + depth).max()) + 1
    ang = s.rng.uniform(0, 1e3, (max_pos, D // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    w = [s.rng.uniform(0.5, 1.5, D).astype(np.float32) for _ in range(2)]
    out = torch.full((s.T, heads, D), 3.0, dtype=DT[dt], device="cuda")
    s.kv.append(1, q, k, v, s.batch, dev(cos), dev(sin), dev(w[0]), dev(w[1]), out=out, tree=tree)
    T = len(depth)
    turned = [A.rotate(A.norm_rows(t[:T], g, 1e-6), cos[base + depth][:, None], sin[base + depth][:, None]) for t, g in ((qh, w[0]), (kh, w[1]))]
    assert torch.equal(out[:T], torch.from_numpy(turned[0]).to(DT[dt]).cuda()) and (out[T:] == 3).all()
    for i, (n, p) in enumerate(zip(lens, parents)):
        for j in range(len(p)):
            for h in range(n_kv):
                s.cache.put(s.table[i, (n - len(p) + j) // page], h, (n - len(p) + j) % page, turned[1][s.cu[i] + j, h], vh[s.cu[i] + j, h])
    assert np.array_equal(s.kv.pages[1].cpu().numpy(), s.cache.pages)
    assert np.array_equal(s.kv.pages[0].cpu().numpy(), s.all[0])


def test_append_leaves_out_what_is_no_node():
    gpu_note("append tree bad nodes")
    s = Setup(3, 64, 1, 16, [30], [6])
    tree = tree_of(s, [[-1, 0, 5, 2, 1, 9]])
    (q, _), (k, _) = s.rows(2, "f16"), s.rows(1, "f16")
    ang = dev(np.zeros((27, 32), np.float32))        # positions up to 26: node 4, of depth 2, is the last
    out = s.kv.append(0, q, k, k, s.batch, ang + 1, ang, tree=tree).float().cpu().numpy()
    bad = [2, 3, 5]
    assert np.isnan(out[bad]).all() and np.array_equal(np.delete(out, bad, 0), np.delete(q.float().cpu().numpy(), bad, 0))
    kn = k.float().cpu().numpy()
    for j in (0, 1, 4):
        s.cache.put(s.table[0, (24 + j) // 16], 0, (24 + j) % 16, kn[j, 0], kn[j, 0])
    assert np.array_equal(s.kv.pages[0].cpu().numpy(), s.cache.pages)
    out = s.kv.append(0, q, k, k, s.batch, ang[:26] + 1, ang[:26], tree=tree).float().cpu().numpy()
    assert np.isnan(out[bad + [4]]).all() and np.isfinite(out[[0, 1]]).all()


# ---------------------------------------------------------------- attention
# (D, n_kv, group, page, lens, nodes, type, max_nodes)
ATTEND = [
    (128, 4, 8, 16, [1], [1], "bf16", 1),
    (128, 4, 8, 16, [15, 16, 17, 31, 32, 33, 48], [3, 16, 9, 31, 32, 2, 17], "f16", 64),   # trees that end at tile and step ends
    (128, 4, 16, 64, [700, 20, 64, 65, 0, 333], [16, 20, 1, 0, 0, 40], "bf16", 40),
    (64, 2, 1, 32, [129, 40], [17, 33], "f16", 64),
    (256, 1, 5, 16, [257, 130, 3], [7, 60, 3], "f16", 64),
    (256, 2, 16, 48, [500], [24], "bf16", 24),
    (128, 1, 24, 128, [300, 77], [5, 30], "f16", 64),
    (128, 4, 8, 64, [190], [190], "bf16", 200),                     # a tree that is all there is
    (128, 2, 8, 16, [300, 17, 128], [300, 17, 100], "f16", 320),
    (64, 2, 4, 32, [1000], [257], "f16", 257),
    (64, 1, 1, 16, [400], [400], "bf16", 400),
    (256, 1, 2, 64, [333, 64], [200, 64], "bf16", 200),
    (128, 1, 7, 16, [1, 5], [40, 9], "bf16", 64),                   # more nodes than tokens: the first see nothing
    (64, 8, 2, 16, [12 + i % 37 for i in range(80)] + [3000, 1700], [1 + i % 12 for i in range(82)], "f16", 16),
    (128, 2, 8, 16, [3000, 40], [64, 40], "bf16", 64),
    (64, 4, 4, 64, [5000], [33], "bf16", 64),
    (128, 2, 8, 32, [900, 700, 33, 0, 1500, 64, 5, 6, 7, 8], [600, 1, 33, 0, 1, 2, 1, 1, 1, 1], "bf16", 640),
    (128, 1, 16, 48, [1777, 1300], [1024, 300], "f16", 1024),
    (64, 1, 4, 16, [1000, 50], [100, 50], "bf16", 33),              # nodes behind max_nodes are NaN
    # in wide tiles
    (128, 8, 8, 16, [190, 100], [190, 60], "bf16", 200),
    (128, 8, 8, 64, [300, 17, 128], [300, 17, 100], "f16", 320),
    (64, 16, 4, 32, [1000], [400], "bf16", 400),
    (64, 8, 8, 16, [300, 150], [280, 150], "f16", 300),
    (256, 8, 8, 64, [333, 64], [200, 64], "bf16", 200),
    (128, 8, 8, 64, [3000, 40], [300, 40], "bf16", 512),            # split
    (64, 8, 8, 32, [2500], [300], "f16", 300),
    (128, 8, 8, 16, [100, 5], [200, 9], "bf16", 200),
    (64, 8, 8, 16, [400, 50], [300, 50], "bf16", 33),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend(case):
    D, n_kv, G, page, lens, news, dt, most = case
    gpu_note(f"attend tree {case}")
    s = Setup(zlib.crc32(str(case).encode()) % 1000, D, n_kv, page, lens, news, pad=2)
    parents = [random_tree(s.rng, n) for n in news]
    q, qn = s.rows(n_kv * G, dt)
    out = torch.full((s.T, n_kv * G, D), 5.0, dtype=DT[dt], device="cuda")
    s.kv.attend(0, q, s.batch, out=out, tree=tree_of(s, parents, most))
    assert (out[s.cu[-1]:] == 5).all()
    check_tree_attend(s, parents, q, qn, out, max_nodes=most)


@pytest.mark.parametrize("lens,news,G,dt,same", [([300, 9, 70], [20, 9, 1], 8, "bf16", True), ([900, 300], [200, 100], 8, "f16", False),
                                                 ([5000], [5], 16, "f16", True), ([2100] * 8, [100] * 8, 8, "bf16", True)])
def test_a_chain_is_ordinary_attention(lens, news, G, dt, same):
    """Bit for bit where the same kernel takes either, whichever way the chain is given."""
    from tinygiant_amd.draft import DraftTree
    gpu_note(f"attend chain {lens}")
    s = Setup(61, 128, 2, 16, lens, news)
    q, qn = s.rows(2 * G, dt)
    want = s.kv.attend(0, q, s.batch)
    chains = [list(range(-1, n - 1)) for n in news]
    a, b = (s.kv.attend(0, q, s.batch, tree=tree) for tree in (tree_of(s, chains, 200), DraftTree(s.batch.cu, s.T, max_nodes=256)))
    assert torch.equal(a, b)
    assert not same or torch.equal(a, want)
    check_tree_attend(s, chains, q, qn, a)


@pytest.mark.parametrize("news,n_kv,G", [([6, 5], 1, 4), ([150, 140], 1, 4), ([190, 180], 8, 8)])
def test_attend_rows_that_are_no_nodes(news, n_kv, G):
    """They are NaN, and tokens that a row does not see may hold anything."""
    gpu_note(f"attend no nodes {news}")
    s = Setup(62, 64, n_kv, 16, [200, 190], news)
    parents = [random_tree(s.rng, n) for n in news]
    parents[0][3] = 3
    parents[1][4] = -5
    # the keys and values of the nodes that are none are not finite
    sc = s.cache.pages[..., 16 * 64:].view(np.float16)
    for i in (0, 1):
        for j, a in enumerate(R.ancestors(parents[i])):
            if a is None:
                t = s.lens[i] - news[i] + j
                places = s.cache._places(t % 16)
                tile = s.cache.pages[s.table[i, t // 16], :, 0].view(np.uint16)
                tile[:, places[4]] = 0x7E00
                tile[:, places[5]] = 0x7C00
    s.kv.pages.copy_(dev(s.all))
    q, qn = s.rows(n_kv * G, "f16")
    out = s.kv.attend(0, q, s.batch, tree=tree_of(s, parents, 160))
    clean = [[a is not None for a in R.ancestors(p)] for p in parents]
    # the oracle multiplies hidden values by 0: give it finite ones
    sc[~np.isfinite(sc)] = 0
    assert not all(clean[0]) and not all(clean[1])
    check_tree_attend(s, parents, q, qn, out, max_nodes=160)


def test_attend_fewer_rows_than_counted():
    gpu_note("attend tree cut off")
    s = Setup(63, 128, 2, 16, [100, 60], [30, 12])
    parents = [random_tree(s.rng, n) for n in (30, 12)]
    tree = tree_of(s, parents)
    q, qn = s.rows(8, "bf16")
    want = s.kv.attend(0, q, s.batch, tree=tree)
    for T in (37, 30, 11):
        got = s.kv.attend(0, q[:T].contiguous(), s.batch, tree=tree)
        # the same nodes at the same places; how rows are split into columns may differ, and so the sums' order
        assert torch.allclose(got.float(), want[:T].float(), rtol=2 ** -7, atol=2 ** -8)


# ---------------------------------------------------------------- keep
@pytest.mark.parametrize("case", [
    (128, 4, 16, [60], [16], 3), (64, 2, 32, [200, 9, 70, 40], [33, 9, 0, 1], 2), (256, 1, 16, [90, 300], [64, 5], 1),
    (128, 5, 64, [100 + 3 * i for i in range(70)], [1 + i % 9 for i in range(70)], 4), (128, 1, 48, [1500], [1024], 2)], ids=str)
def test_keep(case):
    D, n_kv, page, lens, news, layers = case
    gpu_note(f"keep {case[:4]}")
    s = Setup(zlib.crc32(str(case).encode()) % 1000, D, n_kv, page, lens, news, layers=layers)
    P = max(news) + 2
    paths = np.full((len(lens), P), 999, np.int32)
    count = np.zeros(len(lens), np.int32)
    for i, n in enumerate(news):
        if not n:
            continue
        kept = R.ancestors(random_tree(s.rng, n))[s.rng.integers(n)]
        if i % 3 == 1:
            kept = sorted(s.rng.choice(n, size=s.rng.integers(1, n + 1), replace=False))  # any ascending nodes
        paths[i, :len(kept)], count[i] = kept, len(kept)
    kv_len = torch.full((len(lens),), -1, dtype=torch.int32, device="cuda")
    got = s.kv.keep(s.batch, dev(paths), dev(count), kv_len=kv_len)
    assert got is kv_len and np.array_equal(kv_len.cpu().numpy(), np.array(lens) - news + count)
    for layer in range(layers):
        c = A.Cache(len(s.cache.pages), page, n_kv, D, s.all[layer])
        for i, n in enumerate(lens):
            R.keep(c, s.table[i], n, news[i], paths[i, :count[i]])
    assert np.array_equal(s.kv.pages.cpu().numpy(), s.all)


def test_keep_of_some_layers_in_place_of_the_lengths():
    gpu_note("keep some layers")
    s = Setup(70, 64, 2, 16, [50, 31], [9, 4], layers=4)
    path = dev(np.array([[0, 3, 4, 8], [0, 2, 0, 0]], np.int32))
    count = dev(np.array([4, 2], np.int32))
    s.kv.keep(s.batch, path[:, :4], count, kv_len=s.batch.kv_len, layer=1, n_layers=2)
    assert s.batch.kv_len.tolist() == [45, 29]
    for layer in (1, 2):
        c = A.Cache(len(s.cache.pages), 16, 2, 64, s.all[layer])
        R.keep(c, s.table[0], 50, 9, [0, 3, 4, 8])
        R.keep(c, s.table[1], 31, 4, [0, 2])
    assert np.array_equal(s.kv.pages.cpu().numpy(), s.all)


def test_keep_of_what_is_not_there():
    """Entries that are no later node make NaN of their places; pages outside the pool are not written; counts are cut."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("keep bad entries")
    s = Setup(71, 128, 1, 16, [40, 40, 40], [20, 20, 4])
    table = s.table.copy()
    table[1, 1] = len(s.cache.pages)                      # tokens 16..31 of sequence 1: where its nodes 0..11 are
    path = np.array([[0, 0, 20, 7, -3, 19], [0, 2, 13, 14, 15, 16], [0, 1, 2, 3, 9, 9]], np.int32)
    b = KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=40)
    ln = s.kv.keep(b, dev(path), dev(np.array([6, 6, 60], np.int32)), kv_len=torch.empty(3, dtype=torch.int32, device="cuda"))
    assert ln.tolist() == [26, 26, 40]
    before = s.cache.pages.copy()
    R.keep(s.cache, s.table[0], 40, 20, path[0])
    # sequence 1: every destination is in the missing page
    assert np.array_equal(s.kv.pages[0].cpu().numpy(), s.cache.pages)
    k, _ = s.kv.read(0, KVBatch(dev(np.array([0, 20], np.int32)), dev(np.array([40], np.int32)), dev(s.table[:1])), 20)
    nan = torch.isnan(k.float()).flatten(1).all(1).cpu().numpy()
    assert nan.tolist() == [i in (1, 2, 4) for i in range(20)]
    # sources in a missing page: NaN too
    table[1, 1], table[1, 2] = s.table[1, 1], -1          # tokens 32..39: nodes 12..
    s.kv.pages.copy_(dev(before[None]))
    s.kv.keep(KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=40), dev(path), dev(np.array([0, 6, 0], np.int32)))
    k, _ = s.kv.read(0, KVBatch(dev(np.array([0, 20], np.int32)), dev(np.array([40], np.int32)), dev(s.table[1:2])), 20)
    nan = torch.isnan(k.float()).flatten(1).all(1).cpu().numpy()
    assert nan.tolist() == [i in (2, 3, 4, 5) for i in range(20)]
