"""matmul_i8 on the GPU where fp32 ends: rows whose scale is subnormal."""
import numpy as np
import pytest
import torch

from oracle import attn as A
from tests.conftest import gpu_note

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


@pytest.mark.parametrize("size", [1e-36, 1e-39, 1e-41, 3e-45])
@pytest.mark.parametrize("M,N,K", [(1, 70, 272), (6, 70, 272), (20, 130, 1040), (130, 70, 272), (300, 300, 4112)])
def test_rows_near_the_least_that_fp32_holds(M, N, K, size):
    """Their codes are those of any row.  The scale a / 127 and the sum times it are fp32 numbers, off by half a subnormal
    step, 2^-150, at the least; channel scales of 1e30 make of that what can be seen: (|sum| + 1) 2^-150 times them,
    and the 5 roundings of 2^-24 that rows of any size have."""
    from tinygiant_amd.linear import matmul_i8
    gpu_note(f"matmul_i8 subnormal {M} {N} {K} {size}")
    rng = np.random.default_rng(M + K)
    x = (rng.standard_normal((M, K)) * size).astype(np.float32)
    w = rng.integers(-128, 128, (N, K)).astype(np.int8)
    ws = (rng.uniform(0.5, 1.5, N) * 1e30).astype(np.float32)
    q, s = A.codes_i8(x)
    acc = q @ w.astype(np.float64).T
    ref = acc * s * ws
    out = matmul_i8(*(torch.from_numpy(t).cuda() for t in (x, w, ws))).cpu().numpy().astype(np.float64)
    tol = (np.abs(acc) + 1) * 2.0 ** -150 * ws + 5 * 2.0 ** -24 * np.abs(ref)
    assert (np.abs(out - ref) <= tol).all(), float((np.abs(out - ref) / tol).max())
