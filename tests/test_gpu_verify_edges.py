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
