"""Verification of drafted tokens at the edges of what its arguments may hold, on the GPU."""
import pytest
import torch

from tests.conftest import gpu_note
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
