"""int8 matrix product on the GPU: weights int8 with a scale per output
channel, activations quantised per token on the way (tg_matmul_i8_dev).

The projections around PagedKV (q | k | v as one weight, the output
projection added to the residual) and a vocabulary head that stays on the
device; the reference forms them as fp32 or Q4_K matrix-vector products on
host memory (csrc/libtinygiant.c:187, :304).
"""
from __future__ import annotations

import torch

from ._lib import require_lib
from .attn import TYPES, no_gradients, records, run_on
from .moe import RMS_EPS


def _matrix(t, name, device, cols=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in TYPES or (device and t.device != device):
        raise TypeError(f"{name} must be a float32, float16 or bfloat16 tensor on {device or 'a CUDA (HIP) device'}")
    if t.dim() < 1 or (cols is not None and t.shape[-1] != cols):
        raise ValueError(f"{name} of shape {tuple(t.shape)}: rows of {cols} needed")
    if t.dim() != 2:
        if not t.is_contiguous():
            raise ValueError(f"{name} of {t.dim()} dimensions must be contiguous")
        return t.view(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows, its strides are {t.stride()}")
    return t


def _stride(t):
    return max(t.stride(0), t.shape[1]) if t.shape[0] == 1 else t.stride(0)


def matmul_i8(x, w, w_scale, *, norm=None, eps: float = RMS_EPS, residual=None, out=None, out_dtype=None):
    """x [..., K] (float32, float16, bfloat16) times w [N, K] int8 with
    w_scale [N] float32: [..., N] of out_dtype (default: x's type).

    Per row xn = x / rms(x) * norm (norm [K] float32, else xn = x), a =
    max |xn|, codes rint(127 xn / a); the result is the exact int32 product
    times a / 127 and the channel's scale, plus residual (out's type; out may
    be residual itself).  There are no gradients: where torch records them,
    tensors that require one are refused."""
    xm = _matrix(x, "x", None)
    M, K = xm.shape
    dev = xm.device
    if not isinstance(w, torch.Tensor) or w.device != dev or w.dtype != torch.int8 or w.dim() != 2 or not w.is_contiguous():
        raise TypeError(f"w must be a contiguous int8 matrix on {dev}")
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"x has {K} columns, w {w.shape[1]}")
    if max(M, N) > 1 << 30:  # before they become C ints
        raise ValueError(f"{M} rows, {N} channels: at most 2^30 of either")
    if w_scale.dtype != torch.float32 or w_scale.device != dev or w_scale.shape != (N,) or not w_scale.is_contiguous():
        raise TypeError(f"w_scale must be {N} contiguous float32 values on {dev}")
    if norm is not None and (norm.dtype != torch.float32 or norm.device != dev or norm.shape != (K,)
                             or not norm.is_contiguous()):
        raise TypeError(f"norm must be {K} contiguous float32 values on {dev}")
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=out_dtype or x.dtype, device=dev)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"out is {out.dtype}, out_dtype {out_dtype}")
    om = _matrix(out, "out", dev, N)
    rm = None
    if residual is not None:
        rm = _matrix(residual, "residual", dev, N)
        if rm.dtype != om.dtype:
            raise TypeError(f"residual is {rm.dtype}, out {om.dtype}")
    if om.shape[0] != M or (rm is not None and rm.shape[0] != M):
        raise ValueError(f"{M} rows of x, {om.shape[0]} of out" + (f", {rm.shape[0]} of residual" if rm is not None else ""))
    if records(xm, om, rm, norm) or records(w_scale):
        raise no_gradients("matmul_i8")
    if not M:
        return out
    n = require_lib().tg_matmul_i8_workspace(M, N, K)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    run_on(xm, "tg_matmul_i8_dev", xm.data_ptr(), TYPES[xm.dtype], _stride(xm), norm.data_ptr() if norm is not None else None,
           float(eps), w.data_ptr(), w_scale.data_ptr(), rm.data_ptr() if rm is not None else None,
           _stride(rm) if rm is not None else 0, om.data_ptr(), TYPES[om.dtype], _stride(om), M, N, K,
           ws.data_ptr() if n else None, n)
    return out
