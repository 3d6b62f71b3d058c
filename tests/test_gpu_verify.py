"""Verification of drafted tokens on the GPU, against oracle/draft.py's walk in
64 bits.  Tokens, paths and counts are whole numbers and compared exactly: the
random numbers of these tests lie where rounding in 64 bits decides nothing, also
those that are put next to a border."""
import zlib

import numpy as np
import pytest
import torch

from oracle import draft as R
from tests.conftest import gpu_note
from tests.test_gpu_attn import DT, dev
from tests.test_gpu_draft import random_tree

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


class Step:
    """A random batch of trees with logits, drafts and random numbers; `pad` rows behind the last sequence."""

    def __init__(self, seed, nodes, V, dtype, with_draft, t, kind="tree", max_nodes=64, pad=0, spread=2.0, ban=0.05):
        self.rng = rng = np.random.default_rng(seed)
        self.nodes, self.V, self.dt, self.max_nodes = nodes, V, DT[dtype], max_nodes
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        T = self.T = int(self.cu[-1]) + pad
        self.parents = [random_tree(rng, n) if kind == "tree" else list(range(-1, n - 1)) for n in nodes]
        x = spread * rng.standard_normal((T, V))
        banned = rng.random(V) < ban
        banned[rng.integers(V)] = False
        y = x + 0.5 * rng.standard_normal((T, V))
        self.logits, self.draft = (torch.from_numpy(np.where(banned, -np.inf, a)).to(self.dt) for a in (x, y))
        if not with_draft:
            draft, self.draft = self.draft, None
        else:
            draft = self.draft
        self.t = np.full(len(nodes), t, np.float32) if np.isscalar(t) else np.asarray(t, np.float32)
        self.tokens = rng.integers(0, V, T).astype(np.int32)
        for i, p in enumerate(self.parents):
            for j in range(1, nodes[i]):
                row = draft[self.cu[i] + p[j]]
                q = R.chances(row.double().numpy(), max(self.t[i], 0.3))
                if with_draft:
                    self.tokens[self.cu[i] + j] = rng.choice(V, p=q)
                else:
                    self.tokens[self.cu[i] + j] = np.argsort(-q, kind="stable")[p[:j].count(p[j]) % V]
        self.u = rng.random(T)

    def want(self, i):
        a, b = self.cu[i], self.cu[i + 1]
        return R.walk(self.logits[a:b].double().numpy(), self.tokens[a:b], self.u[a:b], self.parents[i], float(self.t[i]),
                      None if self.draft is None else self.draft[a:b].double().numpy(), self.max_nodes)

    def tree(self):
        from tinygiant_amd.draft import DraftTree
        flat = np.concatenate([np.asarray(p, np.int64) for p in self.parents] + [np.zeros(self.T - self.cu[-1], np.int64)])
        return DraftTree(dev(self.cu), self.T, dev(flat.astype(np.int32)), max_nodes=self.max_nodes)

    def run(self, **kw):
        from tinygiant_amd.draft import verify
        args = dict(logits=self.logits.cuda(), tokens=dev(self.tokens), u=dev(self.u), tree=None,
                    draft=None if self.draft is None else self.draft.cuda(),
                    temperature=dev(self.t) if len(set(self.t.tolist())) > 1 else float(self.t[0]))
        args.update(kw)
        args["tree"] = args["tree"] or self.tree()
        return verify(**args)

    def check(self, got):
        tokens, path, count = (x.cpu().numpy() for x in got)
        for i in range(len(self.nodes)):
            p, t = self.want(i)
            assert count[i] == len(p), (i, count[i], path[i][:count[i]], p, tokens[i][:count[i]], t)
            assert path[i].tolist() == p + [-1] * (self.max_nodes - len(p)), (i, p)
            assert tokens[i].tolist() == t + [-1] * (self.max_nodes - len(t)), (i, tokens[i][:len(t)], t)
        return count


# (nodes, vocab, type, draft, temperature, kind, max_nodes)
CASES = [
    ([1], 1, "f32", False, 1.0, "tree", 1),
    ([3, 1, 0, 5], 2, "f32", True, 1.0, "tree", 5),
    ([9] * 40, 7, "bf16", True, 0.8, "tree", 16),
    ([9] * 40, 7, "f16", False, 0.8, "tree", 16),
    ([6] * 30, 100, "f32", True, 1.0, "chain", 64),
    ([17] * 20, 2047, "f16", True, 1.0, "tree", 17),
    ([8, 3, 30], 2048, "bf16", False, 1.0, "tree", 33),
    ([8, 3, 30], 2049, "f32", True, 0.6, "tree", 33),
    ([12, 40, 1, 2], 8191, "f32", False, 1.0, "tree", 64),
    ([5, 6, 7, 8], 8192, "bf16", True, 1.0, "chain", 8),
    ([5, 60, 7, 8], 8193, "f16", True, 1.3, "tree", 64),
    ([200, 64, 65], 513, "f32", False, 1.0, "tree", 256),
    ([1000], 33, "f32", True, 1.0, "tree", 1024),
    ([20, 30], 300, "bf16", True, 1.0, "tree", 11),          # nodes behind max_nodes are not asked
    ([7] * 6, 50021, "f32", True, 0.7, "chain", 7),
    ([26, 9], 50021, "bf16", False, 1.0, "tree", 26),
    ([6, 13], 151936, "bf16", True, 1.0, "tree", 13),
    ([5, 5], 151936, "f32", True, 0.7, "chain", 5),
    ([4] * 300, 50, "f32", True, 1.0, "tree", 4),            # more sequences than lanes
    ([9, 30, 1, 16], 3001, "f32", True, 0.0, "tree", 30),    # greedy
    ([9, 30, 1, 16], 3001, "bf16", False, -1.0, "tree", 30),
    ([9, 12, 1, 16], 20000, "f16", True, [0.0, 1.0, float("nan"), 0.5], "tree", 16),
    ([12, 12], 1000, "f32", True, 1e-6, "tree", 12),
    ([12, 12], 1000, "f32", True, 1e30, "tree", 12),
    ([12, 12], 1000, "f32", False, 1e-30, "tree", 12),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c)[:90])
def test_verify(case):
    nodes, V, dt, with_draft, t, kind, most = case
    gpu_note(f"verify {str(case)[:120]}")
    s = Step(zlib.crc32(str(case).encode()) % 1000, nodes, V, dt, with_draft, t, kind, most, pad=3)
    s.check(s.run())


@pytest.mark.parametrize("V,with_draft,dt", [(40, True, "f32"), (40, False, "f32"), (9001, True, "bf16"), (9001, False, "f16")])
def test_many_walks(V, with_draft, dt):
    """Enough of them to pass every branch, deep paths and long rows of rejected siblings among them."""
    gpu_note(f"verify many {V} {with_draft}")
    rng = np.random.default_rng(5)
    s = Step(V + with_draft, [int(n) for n in rng.integers(1, 25, 150)], V, dt, with_draft, rng.choice([0.0, 0.5, 1.0, 2.0], 150), max_nodes=25)
    count = s.check(s.run())
    assert count.max() >= 4 and (count == 1).any()  # of the inputs: the counts are the walk's by now


def test_chain_without_parents():
    from tinygiant_amd.draft import DraftTree
    gpu_note("verify chain")
    s = Step(8, [6, 1, 4], 500, "f32", True, 1.0, "chain", 6, spread=1.0)
    s.check(s.run(tree=DraftTree(dev(s.cu), s.T, max_nodes=6)))


@pytest.mark.parametrize("with_draft", [True, False])
def test_next_to_a_border(with_draft):
    """u on either side of what decides, by 2^-30 of it: far nearer than sums in 32 bits would tell, and far
    enough for those in 64."""
    gpu_note(f"verify borders {with_draft}")
    for seed in range(6):
        s = Step(100 + seed, [4] * 16, 6007, "f32", with_draft, 0.9, "chain", 4)
        for i in range(16):
            a = s.cu[i]
            side = 1 + 2.0 ** -30 * (1 if i % 2 else -1)
            for j in range(1, 4):
                p = R.chances(s.logits[a + j - 1].double().numpy(), float(s.t[i]))
                q = R.chances(s.draft[a + j - 1].double().numpy(), float(s.t[i])) if with_draft else None
                x = s.tokens[a + j]
                border = p[x] / (q[x] if with_draft else 1.0)
                # tokens that are kept for sure have no border
                s.u[a + j] = border * side if border * side < 1 else 0.3
            # and the token that is drawn at the end, between two others
            path, _ = s.want(i)
            p = R.chances(s.logits[a + path[-1]].double().numpy(), float(s.t[i]))
            if path[-1] < 3:
                if with_draft:
                    p = np.maximum(p - R.chances(s.draft[a + path[-1]].double().numpy(), float(s.t[i])), 0)
                else:
                    p[s.tokens[a + path[-1] + 1]] = 0
            upto = np.cumsum(p) / p.sum()
            k = int(np.searchsorted(upto, s.rng.random()))
            s.u[a] = upto[k] * (1 + 2.0 ** -40 * (1 if i % 3 else -1))
            if not s.u[a] < 1:
                s.u[a] = 0.5
        s.check(s.run())


def test_siblings_that_are_the_same_and_tokens_that_are_none():
    gpu_note("verify same siblings")
    for with_draft in (True, False):
        for seed in range(8):
            s = Step(200 + seed, [20, 20], 11, "f32", with_draft, 1.0, "tree", 20)
            for i in (0, 1):
                rows = np.arange(s.cu[i] + 1, s.cu[i + 1])
                s.tokens[rows[::3]] = s.tokens[rows[0]]
                s.tokens[rows[4::5]] = s.rng.choice([-1, 11, 2 ** 31 - 1, -2 ** 31], len(rows[4::5]))
            s.check(s.run())


def test_everything_rejected():
    """Candidates that are all there is: what is left is nothing, and the token is drawn of all."""
    gpu_note("verify nothing left")
    s = Step(300, [4, 4], 3, "f32", False, 1.0, "tree", 4, ban=0.0)
    s.parents = [[-1, 0, 0, 0]] * 2
    s.tokens[:] = [0, 0, 1, 2] * 2
    s.u[:] = [0.4, 2.0, 2.0, 2.0, 0.9, float("nan"), 5.0, 1e300]  # never kept
    p = [R.chances(s.logits[r].numpy(), 1.0) for r in (0, 4)]
    got = s.run()
    assert got.count.tolist() == [1, 1]
    assert got.tokens[:, 0].tolist() == [int(np.searchsorted(np.cumsum(p[i]), u, side="right")) for i, u in ((0, 0.4), (1, 0.9))]


def test_more_rejections_than_sweeps_have_launches():
    """Siblings that the target never says: 23 sums over the row, and 19 before one that it may."""
    gpu_note("verify many rejections")
    for seed in range(4):
        s = Step(310 + seed, [24, 9, 24], 5000, "f32", True, 1.0, "tree", 24)
        s.parents[0], s.parents[2] = [-1] + [0] * 23, [-1] + [0] * 20 + [1, 20, 20]
        for i, last in ((0, 24), (2, 20)):
            s.logits[s.cu[i], torch.from_numpy(s.tokens[s.cu[i] + 1:s.cu[i] + last]).long()] = -np.inf
        got = s.run()
        s.check(got)
        assert int(got.count[0]) == 1


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "all -inf"])
def test_rows_that_are_no_logits(bad, with_draft):
    """They count where something is decided by them, in the target's rows and the draft's; elsewhere they may hold anything."""
    gpu_note(f"verify bad rows {bad} {with_draft}")
    for t in (1.0, 0.0):
        for seed in range(6):
            s = Step(400 + seed, [6] * 12, 700, "bf16", with_draft, t, "tree", 6)
            for i in range(12):
                row = s.cu[i] + s.rng.integers(6)
                x = s.draft if with_draft and i % 2 else s.logits
                if bad == "all -inf":
                    x[row] = -np.inf
                else:
                    x[row, s.rng.integers(700)] = bad
            s.check(s.run())


def test_masks_and_sizes_of_logits():
    """Masked by the type's lowest value or -inf, logits at the type's ends, equal logits, one token alone."""
    gpu_note("verify masks")
    for dt in DT:
        big = torch.finfo(DT[dt])
        for seed, make in enumerate([lambda x: x.masked_fill(torch.arange(x.shape[1]) % 3 > 0, big.min),
                                     lambda x: torch.where(x > 0, big.max / 2, x.double()).to(x.dtype),
                                     lambda x: torch.zeros_like(x), lambda x: torch.full_like(x, big.min),
                                     lambda x: torch.full_like(x, -np.inf).index_fill(1, torch.tensor([17]), -3.0)]):
            for t in (1.0, 0.0):
                s = Step(500 + seed, [7, 5, 1], 2500, dt, seed % 2 == 0, t, "tree", 8)
                s.logits = make(s.logits)
                if s.draft is not None:
                    s.draft = make(s.draft)
                s.check(s.run())


def test_random_numbers_out_of_range():
    gpu_note("verify bad u")
    s = Step(600, [3, 3, 3, 3, 3], 50, "f32", True, [1.0, 1.0, 1.0, 1.0, 0.0], "chain", 3)
    s.u[s.cu[:-1]] = [1.0, -0.1, float("nan"), 1 - 2.0 ** -53, float("nan")]
    got = s.run()
    count = s.check(got)
    last = got.tokens.cpu().numpy()[np.arange(5), count - 1]
    assert (last[:3] == -1).all() and (last[3:] >= 0).all()


def test_rows_apart_and_odd_places():
    """Views of wider tensors, rows at every alignment of their type."""
    gpu_note("verify strides")
    for dt, with_draft in (("bf16", True), ("f16", False), ("f32", True)):
        s = Step(700, [9, 4], 1237, dt, with_draft, 1.0, "tree", 9, pad=1)
        for width, at in ((1237, 0), (1300, 1), (1239, 2), (1241, 3)):
            wide = torch.full((s.T, width), float("nan"), dtype=DT[dt], device="cuda")
            wide[:, at:at + 1237] = s.logits.cuda()
            draft = None
            if with_draft:
                draft = torch.full((s.T, width + 5), float("nan"), dtype=DT[dt], device="cuda")
                draft[:, 3:1240] = s.draft.cuda()
                draft = draft[:, 3:1240]
            s.check(s.run(logits=wide[:, at:at + 1237], draft=draft))


def test_empty():
    from tinygiant_amd.draft import DraftTree, verify
    gpu_note("verify empty")
    z = torch.zeros(0, 9, device="cuda")
    i, u = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda")
    got = verify(z, i, u, DraftTree(dev(np.zeros(4, np.int32)), 0, max_nodes=5))
    assert got.count.tolist() == [0, 0, 0] and (got.tokens == -1).all() and (got.path == -1).all()
    got = verify(z, i, u, DraftTree(dev(np.zeros(1, np.int32)), 0))
    assert got.tokens.shape == (0, 64) and got.count.numel() == 0


def test_tokens_come_as_the_target_would_draw_them():
    """The first token of a step is distributed as p whatever the draft proposes: 8192 walks over one row, the counts of
    each token within 5 standard deviations."""
    gpu_note("verify distribution")
    from tinygiant_amd.draft import DraftTree, verify
    n, V = 8192, 6
    rng = np.random.default_rng(1)
    parents = [-1, 0, 0, 0]
    p, q = rng.standard_normal((2, V))
    for with_draft in (True, False):
        tokens = rng.choice(V, size=(n, 4), p=R.chances(q, 1.0)) if with_draft else np.tile([0, 3, 1, 5], (n, 1))
        x = torch.from_numpy(np.tile(p, (4 * n, 1)).astype(np.float32)).cuda()
        y = torch.from_numpy(np.tile(q, (4 * n, 1)).astype(np.float32)).cuda() if with_draft else None
        tree = DraftTree(dev(np.arange(0, 4 * n + 1, 4, dtype=np.int32)), 4 * n, dev(np.tile(parents, n).astype(np.int32)), max_nodes=4)
        got = verify(x, dev(tokens.reshape(-1).astype(np.int32)), dev(rng.random(4 * n)), tree, draft=y)
        seen = np.bincount(got.tokens[:, 0].cpu().numpy(), minlength=V)
        want = R.chances(p.astype(np.float32), 1.0)
        assert (np.abs(seen - n * want) <= 5 * np.sqrt(n * want * (1 - want))).all(), (seen, n * want)


def test_graph_streams_and_the_same_call():
    """Captured and replayed on other contents, with eager work between; on a stream of its own; the same bits again."""
    from tinygiant_amd.draft import verify
    gpu_note("verify graph")
    a, b = (Step(seed, [9, 6, 3], 5000, "f32", True, 1.0, "tree", 9) for seed in (800, 801))
    tree = a.tree()
    parent, static = tree.parent, [a.logits.cuda(), dev(a.tokens), dev(a.u), a.draft.cuda()]

    def call():
        tree.build()
        return verify(static[0], static[1], static[2], tree, draft=static[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    a.check(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(6):
        s = (a, b)[k % 2]
        for x, y in zip(static, (s.logits, torch.from_numpy(s.tokens), torch.from_numpy(s.u), s.draft)):
            x.copy_(y)
        parent.copy_(torch.from_numpy(np.concatenate(s.parents).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)
        torch.ones(1000, device="cuda").sum().item()
        assert all(torch.equal(x, y) for x, y in zip(call(), out))
