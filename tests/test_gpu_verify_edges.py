"""Verification of drafted tokens at the edges of what its arguments may hold, on the GPU."""
import numpy as np
import pytest
import torch

from tests.conftest import gpu_note
from tests.test_gpu_attn import dev
from tests.test_gpu_verify import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


def used_memory(byte):
    """What torch gives out next was written before."""
    torch.full((1 << 24,), byte, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("t", [1.0, 0.0])
def test_a_sequence_whose_first_node_is_none(with_draft, t):
    """Nothing of it is part of a tree: no node is kept and no token drawn; the other sequences are walked as ever."""
    gpu_note(f"verify bad roots {with_draft} {t}")
    for byte in (0, 0x3F, 0x7F, 0xFF):
        s = Step(900, [5, 1, 70, 4, 3, 1], 5000, "f32", with_draft, t, "tree", 70)
        for i, bad in ((1, 0), (2, 0), (3, -2), (5, 2 ** 31 - 1)):
            s.parents[i][0] = bad
        used_memory(byte)
        got = s.run()
        s.check(got)
        assert got.count.tolist()[1:4] == [0, 0, 0] and int(got.count[5]) == 0 and int(got.count[0]) >= 1


@pytest.mark.parametrize("gap", [7.2, 7.3])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_a_random_number_of_0_draws_a_token(gap, dt):
    """Values of which a chunk's own largest is exp(-500) of the row's, and others before it that are nothing next to that:
    a number of 0 draws the first token whose exponential is one of 64 bits' normal numbers."""
    gpu_note(f"verify u of 0 {gap}")
    for kids in (0, 1):
        s = Step(910, [1 + kids, 1 + kids], 9000, dt, False, 0.01, "chain", 2, ban=0.0)
        x = torch.full((s.T, 9000), -gap)
        x[:, 2048 + 77] = -5.0
        x[:, 5000] = 0.0
        s.logits = x.to(s.dt)
        s.tokens[:] = 7000                     # not kept: nothing of a chance
        s.u[:] = 0.5
        s.u[s.cu[:-1]] = 0.0
        got = s.run()
        assert got.count.tolist() == [1, 1]
        assert got.tokens[:, 0].tolist() == [2048 + 77] * 2


@pytest.mark.parametrize("V,with_draft,t", [(262145, True, 1.0), (262145, False, 0.7), (262145, True, 0.0), (600001, True, 0.8),
                                            (600001, False, 1.0), (600001, False, 0.0), (1 << 20, True, [0.0, 1.0, 0.5])])
def test_more_chunks_than_lanes(V, with_draft, t):
    """Rows of more than 64 chunks (from 262145 tokens on) and 256 pieces: what decides stands behind them, the largest
    value, kept drafts and the token that is drawn."""
    gpu_note(f"verify {V} {with_draft} {t}")
    s = Step(V % 1000, [4, 3, 1], V, "f32", with_draft, t, "tree", 4, ban=0.0)
    for x in (s.logits, s.draft):
        if x is not None:
            x[:, 262143:] += 3.0 if V > 262145 else 16.0
    if V > 262145:
        at = s.rng.integers(262144, V, s.T)
        s.logits[torch.arange(s.T), torch.from_numpy(at)] = 14.0
        for i, p in enumerate(s.parents):
            for j in range(1, s.nodes[i]):
                if j % 2:
                    s.tokens[s.cu[i] + j] = at[s.cu[i] + p[j]]
    s.u[s.cu[:-1]] = [0.999, 0.97, 0.9999]
    got = s.run()
    count = s.check(got)
    last = got.tokens.cpu().numpy()[np.arange(3), count - 1]
    assert (last >= 262143).all(), last


@pytest.mark.parametrize("with_draft", [True, False])
def test_the_largest_vocabulary_and_the_most_nodes(with_draft):
    """2^20 tokens and trees that may have 1024 nodes: what a walk holds is as large as it gets."""
    gpu_note(f"verify 2^20, 1024 {with_draft}")
    s = Step(930, [3, 2], 1 << 20, "bf16", with_draft, 1.0, "tree", 1024, ban=0.0)
    s.check(s.run())


@pytest.mark.parametrize("with_draft,t", [(True, 1.0), (False, 1.0), (True, 0.0)])
def test_trees_of_fewer_rows_than_counted(with_draft, t):
    """Rows that end before cu does: a tree whose first nodes are there is walked over those, one of which none is there has
    count 0."""
    from tinygiant_amd.draft import DraftTree
    gpu_note(f"verify cut off {with_draft} {t}")
    for T in (0, 1, 9, 13, 14):
        s = Step(920, [9, 5, 4], 700, "f32", with_draft, t, "tree", 9)
        tree = DraftTree(dev(s.cu), T, dev(np.concatenate(s.parents).astype(np.int32)[:T]), max_nodes=9)
        used_memory(0x7F)
        got = s.run(logits=s.logits[:T].cuda(), tokens=dev(s.tokens[:T]), u=dev(s.u[:T]), draft=s.draft[:T].cuda() if with_draft else None, tree=tree)
        s.nodes = [max(0, min(n, T - at)) for n, at in zip(s.nodes, s.cu)]
        s.parents = [p[:n] for p, n in zip(s.parents, s.nodes)]
        whole, s.cu = s.cu, np.concatenate([[0], np.cumsum(s.nodes)]).astype(np.int32)
        assert (s.cu[1:] == np.minimum(whole[1:], T)).all()
        s.check(got)


def test_logits_of_no_rows_have_any_strides():
    from tinygiant_amd.draft import DraftTree, verify
    gpu_note("verify no rows")
    i, u = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda")
    tree = DraftTree(dev(np.zeros(3, np.int32)), 0, max_nodes=5)
    for strides in ((0, 0), (9, 1), (1, 7)):
        x = torch.zeros(0, device="cuda").as_strided((0, 9), strides)
        for draft in (None, x):
            got = verify(x, i, u, tree, draft=draft)
            assert got.count.tolist() == [0, 0] and (got.tokens == -1).all() and (got.path == -1).all()


@pytest.mark.parametrize("with_draft", [True, False])
def test_random_numbers_count_for_nothing_where_a_sequence_is_greedy(with_draft):
    gpu_note(f"verify greedy u {with_draft}")
    for u in (0.0, 1.0, 2.0, -1.0, float("nan"), float("inf")):
        s = Step(940, [12, 30, 1, 5], 40, "f32", with_draft, [0.0, -2.0, float("nan"), 0.0], "tree", 30, spread=1.0)
        for i, p in enumerate(s.parents):       # children that are the largest logits' tokens, so that walks are long
            for j in range(1, len(p)):
                if j % 2:
                    s.tokens[s.cu[i] + j] = int(s.logits[s.cu[i] + p[j]].argmax())
        want = s.run()
        s.u[:] = u
        got = s.run()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(got.count.max()) > 2
        s.check(got)
