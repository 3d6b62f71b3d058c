"""Strides that mean nothing: those of tensors without rows, as numpy's empty arrays have them, and of a single column.
Host tensors around the constructors, as in test_attn_calls.py: no call reaches a kernel."""
import pytest
import torch

from tests.test_attn_calls import cache


@pytest.mark.parametrize("shape,strides", [((0, 4, 64), (0, 0, 0)), ((0, 4, 64), (1, 2, 3)), ((0, 256), (0, 0)), ((0, 256), (5, 7))])
def test_no_rows_have_any_strides(shape, strides):
    assert cache()._rows(torch.zeros(0).as_strided(shape, strides), "q", 4, torch.float32, 0) == 256


def test_rows_that_are_there_are_packed():
    kv, x = cache(), torch.zeros(4000)
    assert kv._rows(x.as_strided((2, 4, 64), (700, 64, 1)), "q", 4, torch.float32, 2) == 700
    for n, shape, strides in ((1, (1, 4, 64), (256, 65, 1)), (1, (1, 4, 64), (256, 64, 2)), (1, (1, 256), (256, 2)), (2, (2, 256), (256, 2)),
                              (0, (1, 256), (256, 1)), (0, (0, 4, 63), (0, 0, 0)), (0, (0, 3, 64), (0, 0, 0))):
        with pytest.raises(ValueError, match="packed heads"):
            kv._rows(x.as_strided(shape, strides), "q", 4, torch.float32, n)
