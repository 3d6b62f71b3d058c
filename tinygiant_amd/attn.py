"""The attention block's cache on the GPU: a paged Q4_0 KV cache and causal
grouped-query attention over it, for ragged batches.

Device counterpart of the reference's attention step, which runs one token at
a time on host memory (tinygiant/engine.py:199-227):

    q, k: head norm, rotation by position      libtinygiant.c:386-398
    append k, v to the layer's cache           libtinygiant.c:400-403
    softmax(q . k / sqrt(head_dim)) v          libtinygiant.c:405-446

PagedKV holds the pages of every layer; KVBatch says which rows belong to
which sequence and which pages hold its tokens.  The projections before and
after are linear.matmul_i8.  Every step runs in libtinygiant.so's gfx950
kernels; torch is used only to hold device buffers and name the stream.
There are no gradients: where torch records them, calls refuse tensors that
require one.

    kv = PagedKV(n_layers=48, n_pages=4096, page_tokens=64, n_kv_heads=4, head_dim=128)
    batch = KVBatch(cu, kv_len, table)             # int32 CUDA tensors
    q = kv.append(layer, q, k, v, batch, cos, sin, q_norm=qn, k_norm=kn)
    o = kv.attend(layer, q, batch)
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import call, require_lib
from .moe import RMS_EPS

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # TG_T_*


class _Batch(ctypes.Structure):
    """tg_kv_batch of include/tinygiant.h."""
    _fields_ = [("pages", ctypes.c_void_p), ("table", ctypes.c_void_p), ("cu", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p), ("n_pages", ctypes.c_int64), ("page_tokens", ctypes.c_int32),
                ("n_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("table_cols", ctypes.c_int32),
                ("table_stride", ctypes.c_int32), ("n_seqs", ctypes.c_int32), ("n_tokens", ctypes.c_int32)]


def run_on(t, name, *args):
    """call(name, ..., stream) on the current stream of t's device, which is
    made current where it is not (a null stream names none).  The handle by
    itself: a torch.cuda.Stream made of it each time costs 1.8 us."""
    index = t.device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        call(name, *args, stream)
    else:
        with torch.cuda.device(index):
            call(name, *args, stream)


def records(a, b=None, c=None, d=None) -> bool:
    """Would torch record gradients through one of these tensors?"""
    return (a.requires_grad or (b is not None and b.requires_grad) or (c is not None and c.requires_grad)
            or (d is not None and d.requires_grad)) and torch.is_grad_enabled()


def no_gradients(name):
    """The error of a call that would drop them, as torch's out= does."""
    return RuntimeError(f"{name} has no gradients and a tensor requires one: call it under torch.no_grad()")


def _index(t, name, dims):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or t.dim() != dims:
        raise TypeError(f"{name} must be a {dims}-dimensional int32 CUDA (HIP) tensor")


def table_stride(table) -> int:
    """Entries from one sequence's row of a page table to the next's; 0 where
    all of them have the same row (an expanded one).  Of one row there is no
    next, and torch gives its stride any value."""
    n, cols = table.shape
    stride = table.stride(0) if n > 1 else cols
    if 0 < stride < cols:
        raise ValueError(f"rows of table overlap: {cols} entries, {stride} apart")
    return stride


class KVBatch:
    """A ragged batch: rows cu[s]..cu[s+1]-1 are the last tokens of sequence
    s, which has kv_len[s] tokens in the pages table[s].  cu [n_seqs + 1],
    kv_len [n_seqs], table [n_seqs, pages] are int32 CUDA tensors that the
    kernels read at each call, so they may be rewritten in place between
    calls (and graph replays).  table may be a view: columns of a wider one,
    or one row expanded, whose pages the sequences then share (to read: a
    token's place is one sequence's to append to).  Tensors of fewer rows
    than cu counts are its first rows.  max_len: about the longest kv_len;
    it only sets how attention's work is split (default: what the table can
    hold)."""

    def __init__(self, cu, kv_len, table, max_len: int = 0):
        _index(cu, "cu", 1)
        _index(kv_len, "kv_len", 1)
        _index(table, "table", 2)
        n = kv_len.numel()
        if cu.numel() != n + 1 or table.shape[0] != n:
            raise ValueError(f"{n} sequences, {cu.numel()} row bounds, {table.shape[0]} table rows")
        if not cu.is_contiguous() or not kv_len.is_contiguous() or (table.numel() and table.stride(1) != 1):
            raise TypeError("cu, kv_len and the rows of table must be contiguous")
        table_stride(table)
        if not cu.device == kv_len.device == table.device:
            raise ValueError(f"cu on {cu.device}, kv_len on {kv_len.device}, table on {table.device}")
        if max_len < 0:
            raise ValueError(f"max_len {max_len}")
        self.cu, self.kv_len, self.table, self.max_len = cu, kv_len, table, min(int(max_len), 1 << 30)  # no table holds more
        self.n_seqs, self.device = n, cu.device


class PagedKV:
    """The paged Q4_0 KV cache of every layer: pages is a uint8 tensor
    [n_layers, n_pages, n_kv_heads, page_tokens / 16, 18 * head_dim] (tile
    layout: include/tinygiant.h).  pages= wraps an existing one; otherwise
    zeros are allocated."""

    def __init__(self, n_layers: int, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int,
                 device="cuda", pages=None):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim {head_dim} is not 64, 128 or 256")
        if page_tokens % 16 or not 16 <= page_tokens <= 65536:
            raise ValueError(f"page_tokens {page_tokens} is not a multiple of 16 up to 65536")
        if min(n_layers, n_pages, n_kv_heads) < 1:
            raise ValueError(f"n_layers {n_layers}, n_pages {n_pages}, n_kv_heads {n_kv_heads}")
        shape = (n_layers, n_pages, n_kv_heads, page_tokens // 16, 18 * head_dim)
        if pages is None:
            pages = torch.zeros(shape, dtype=torch.uint8, device=device)
        elif (not isinstance(pages, torch.Tensor) or not pages.is_cuda or pages.dtype != torch.uint8
              or tuple(pages.shape) != shape or not pages.is_contiguous()):
            raise TypeError(f"pages must be a contiguous uint8 CUDA (HIP) tensor of shape {shape}")
        self.pages, self.device = pages, pages.device
        self.n_layers, self.n_pages, self.page_tokens = n_layers, n_pages, page_tokens
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.layer_bytes = pages.stride(0)

    def _batch(self, layer: int, batch: KVBatch, n_tokens: int) -> _Batch:
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        if batch.device != self.device:
            raise ValueError(f"batch on {batch.device}, pages on {self.device}")
        t = batch.table
        return _Batch(self.pages.data_ptr() + layer * self.layer_bytes, t.data_ptr(), batch.cu.data_ptr(),
                      batch.kv_len.data_ptr(), self.n_pages, self.page_tokens, self.n_kv_heads, self.head_dim, t.shape[1],
                      table_stride(t), batch.n_seqs, n_tokens)

    def _rows(self, t, name, heads, dtype, n_tokens):
        """A [T, heads, D] (or [T, heads * D]) tensor with packed heads: its row stride."""
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != dtype:
            raise TypeError(f"{name} must be a {dtype} tensor on {self.device}")
        D, shape, stride = self.head_dim, t.shape, t.stride()
        if len(shape) == 3:
            ok = shape[1] == heads and shape[2] == D and stride[2] == 1 and (heads == 1 or stride[1] == D)
        else:
            ok = len(shape) == 2 and shape[1] == heads * D and stride[1] == 1
        if not ok or shape[0] != n_tokens:
            raise ValueError(f"{name} of shape {tuple(shape)}, strides {stride}: "
                             f"[{n_tokens}, {heads}, {D}] with packed heads needed")
        return heads * D if n_tokens == 1 else stride[0]  # of one row the stride is any

    def _heads(self, q):
        D = self.head_dim
        if not isinstance(q, torch.Tensor) or q.dim() not in (2, 3) or (q.shape[-1] != D if q.dim() == 3 else q.shape[1] % D):
            raise ValueError(f"q must be a [T, heads, {D}] tensor")
        return q.shape[1] if q.dim() == 3 else q.shape[1] // D

    def _floats(self, t, name, shape):
        if (not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.float32
                or t.shape != shape or not t.is_contiguous()):
            raise TypeError(f"{name} must be a contiguous float32 tensor of shape {shape} on {self.device}")
        return t.data_ptr()

    def append(self, layer: int, q, k, v, batch: KVBatch, cos=None, sin=None, q_norm=None, k_norm=None,
               eps: float = RMS_EPS, out=None):
        """New rows: q [T, heads, D] (or None), k and v [T, n_kv_heads, D] of
        one type (float32, float16, bfloat16; views of a projection's rows
        do) are normed (q_norm, k_norm [D]) and rotated (cos, sin [max_pos,
        D / 2]); k and v go into the cache, the rotated q into out (default:
        a new tensor; may be q itself), which is returned.  Rows behind the
        last sequence are not written."""
        heads = 0 if q is None else self._heads(q)
        T, dt, D = k.shape[0], k.dtype, self.head_dim
        if dt not in TYPES:
            raise TypeError(f"k of type {dt}: float32, float16 or bfloat16 needed")
        ks = self._rows(k, "k", self.n_kv_heads, dt, T)
        vs = self._rows(v, "v", self.n_kv_heads, dt, T)
        qs = qp = op = os_ = None
        if q is not None:
            qs = self._rows(q, "q", heads, dt, T)
            if out is None:
                out, os_ = q.new_empty((T, heads, D)), heads * D
            else:
                os_ = self._rows(out, "out", heads, dt, T)
            qp, op = q.data_ptr(), out.data_ptr()
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin are given together")
        max_pos = 0 if cos is None else cos.shape[0]
        cp = None if cos is None else self._floats(cos, "cos", (max_pos, D // 2))
        sp = None if sin is None else self._floats(sin, "sin", (max_pos, D // 2))
        qn = None if q_norm is None else self._floats(q_norm, "q_norm", (D,))
        kn = None if k_norm is None else self._floats(k_norm, "k_norm", (D,))
        if records(k, v, q, out) or records(k, q_norm, k_norm, cos) or (sin is not None and records(sin)):
            raise no_gradients("append")
        b = self._batch(layer, batch, T)
        if not T or not batch.n_seqs:
            return out
        run_on(k, "tg_kv_append_q4_dev", ctypes.byref(b), TYPES[dt], qp, qs or 0, k.data_ptr(), ks, v.data_ptr(), vs,
               op, os_ or 0, heads, qn, kn, float(eps), cp, sp, max_pos)
        return out

    def read(self, layer: int, batch: KVBatch, n_tokens: int):
        """What the cache holds for the batch's rows: k, v [n_tokens,
        n_kv_heads, D] float16 (rows behind the last sequence: not written)."""
        if n_tokens < 0:
            raise ValueError(f"n_tokens {n_tokens}")
        k = torch.empty((n_tokens, self.n_kv_heads, self.head_dim), dtype=torch.float16, device=self.device)
        v = torch.empty_like(k)
        b = self._batch(layer, batch, n_tokens)
        if n_tokens and batch.n_seqs:
            run_on(k, "tg_kv_read_q4_dev", ctypes.byref(b), k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, layer: int, q, batch: KVBatch, scale: float | None = None, out=None):
        """softmax(scale q . k) v for q [T, heads, D] float16 or bfloat16
        (scale: above 0, 1 / sqrt(D) by default), each row over the positions up to
        its own; rows at positions below 0 are zero, those behind the last
        sequence not written.  out: default a new tensor; must not overlap q."""
        heads, D = self._heads(q), self.head_dim
        T, dt = q.shape[0], q.dtype
        if dt not in (torch.float16, torch.bfloat16):
            raise TypeError(f"q of type {dt}: float16 or bfloat16 needed")
        qs = self._rows(q, "q", heads, dt, T)
        if out is None:
            out, os_ = q.new_empty((T, heads, D)), heads * D
        else:
            os_ = self._rows(out, "out", heads, dt, T)
        if records(q, out):
            raise no_gradients("attend")
        b = self._batch(layer, batch, T)
        if not T or not batch.n_seqs:
            return out
        ref = ctypes.byref(b)
        n = require_lib().tg_attn_q4_workspace(ref, heads, batch.max_len)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        run_on(q, "tg_attn_q4_dev", ref, TYPES[dt], q.data_ptr(), qs, heads,
               D ** -0.5 if scale is None else float(scale), out.data_ptr(), os_, batch.max_len,
               ws.data_ptr() if n else None, n)
        return out
