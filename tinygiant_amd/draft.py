"""Trees of drafted tokens on the GPU: steps in which one pass of the model
answers several guesses at what follows.

The reference generates one token a pass (tinygiant/engine.py:317-409).  With
drafts, the rows of a sequence in a KVBatch are a tree: node 0 is the last
token that is decided, every other node a guess at what follows its parent.

    tree = DraftTree(batch.cu, n_tokens, parent)        # int32 CUDA tensors; once a step, for all layers
    q = kv.append(layer, q, k, v, batch, cos, sin, tree=tree)   # rotated by depth
    o = kv.attend(layer, q, batch, tree=tree)                   # each node over its own ancestors
    new = verify(logits, tokens, u, tree, draft=draft_logits, temperature=0.7)
    kv.keep(batch, new.path, new.count, kv_len=batch.kv_len)    # the kept nodes' entries, in every layer

Everything runs in libtinygiant.so's gfx950 kernels; torch is used only to
hold device buffers and name the stream.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from ._lib import require_lib
from .attn import TYPES, _index, no_gradients, records, run_on


class _Trees(ctypes.Structure):
    """tg_draft_trees of include/tinygiant.h."""
    _fields_ = [("cu", ctypes.c_void_p), ("parent", ctypes.c_void_p), ("n_seqs", ctypes.c_int32),
                ("n_tokens", ctypes.c_int32), ("max_nodes", ctypes.c_int32)]


class DraftTree:
    """The trees of a batch: cu [n_seqs + 1] is the batch's, node j of
    sequence s its row cu[s] + j, parent [n_tokens] the node (below j) that
    each follows, -1 none; without parent each node follows the one before it.
    max_nodes (1 to 1024): the most nodes of one sequence.

    bits [n_tokens, words] int32 holds the nodes that each row sees (bit i of
    its words: node i; itself and those it follows), depth [n_tokens] int32
    how many it follows.  Rows that are no nodes (a parent that is no node
    before them, nodes from max_nodes on) have no bits and depth -1; what
    attends them is NaN and nothing of them is appended.  cu and parent are
    read by build() and by verify: call build() again, which may be captured
    into a graph, after they were rewritten in place, and do not rewrite them
    between it and verify."""

    def __init__(self, cu, n_tokens: int, parent=None, max_nodes: int = 64):
        _index(cu, "cu", 1)
        if not cu.numel() or not cu.is_contiguous():
            raise ValueError("cu must be contiguous and hold a bound more than there are sequences")
        if not 0 <= n_tokens < 1 << 31:
            raise ValueError(f"n_tokens {n_tokens}")
        if parent is not None:
            _index(parent, "parent", 1)
            if parent.device != cu.device or parent.numel() != n_tokens or not parent.is_contiguous():
                raise ValueError(f"parent of {parent.numel()} entries on {parent.device}: {n_tokens} contiguous ones on {cu.device} needed")
        if not 1 <= max_nodes <= 1024:
            raise ValueError(f"max_nodes {max_nodes} is not 1 to 1024")
        self.cu, self.parent, self.n_tokens, self.max_nodes = cu, parent, int(n_tokens), int(max_nodes)
        self.n_seqs, self.device = cu.numel() - 1, cu.device
        self.words = (self.max_nodes + 31) // 32
        self.bits = torch.empty((self.n_tokens, self.words), dtype=torch.int32, device=self.device)
        self.depth = torch.empty(self.n_tokens, dtype=torch.int32, device=self.device)
        self.links = torch.empty_like(self.depth)  # for verify
        self.build()

    def _trees(self) -> _Trees:
        return _Trees(self.cu.data_ptr(), None if self.parent is None else self.parent.data_ptr(), self.n_seqs,
                      self.n_tokens, self.max_nodes)

    def build(self) -> "DraftTree":
        """bits, depth and links from cu and parent as they now are."""
        if self.n_tokens and self.n_seqs:
            run_on(self.depth, "tg_draft_tree_dev", ctypes.byref(self._trees()), self.bits.data_ptr(), self.depth.data_ptr(),
                   self.links.data_ptr())
        return self


class Verified(NamedTuple):
    """int32 tensors.  path [n_seqs, max_nodes]: the kept nodes of each
    sequence, node 0 first, -1 behind them; count [n_seqs]: how many; tokens
    [n_seqs, max_nodes]: those that the step brings, the kept drafts and then
    the next token (so count of them), -1 behind them."""
    tokens: torch.Tensor
    path: torch.Tensor
    count: torch.Tensor


def _logits(t, name, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in TYPES or t.dim() != 2 or t.shape[1] < 1:
        raise TypeError(f"{name} must be a [rows, vocab] float32, float16 or bfloat16 CUDA (HIP) tensor")
    if like is not None and (t.dtype != like.dtype or t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, the logits {like.dtype} {tuple(like.shape)} on {like.device}")
    if t.shape[0] and t.shape[1] > 1 and t.stride(1) != 1:  # of no rows the strides are any
        raise ValueError(f"{name} must have contiguous rows, its strides are {t.stride()}")
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def verify(logits, tokens, u, tree: DraftTree, draft=None, temperature=1.0) -> Verified:
    """Which drafts stay, and the token that follows them, for every sequence of tree.

    logits [n_tokens, vocab] (float32, float16, bfloat16): the target's after
    each row; tokens [n_tokens] int32: the rows' tokens; u [n_tokens] float64:
    random numbers in [0, 1), one for each draft, that of node 0 for the next token.  draft: the
    logits (of the same type and shape) of the model after each row, of which
    that node's children were drawn, each without regard to the others; without it children
    are candidates that no one drew (a draft head's best ones).  temperature: of both,
    one for all or a float32 [n_seqs] tensor; 0 or below: greedy.

    The children of a node are asked in order.  With p and q the probabilities
    of target and draft, x stays where u q(x) < p(x), and one that does not
    leaves norm(max(p - q, 0)) for the next; without draft x stays where u <
    p(x) and else leaves p without x.  From what is left where none
    stays the next token is drawn, so that tokens are distributed as if they
    had been drawn from the target one by one (numpy's choice in
    tinygiant/engine.py:348-357, at top_p 1).  Decisions are those of 64-bit
    arithmetic.  Rows that hold NaN or +inf, or nothing but -inf: the next
    token is -1 where they decide (Sampler's errors, which a call that does
    not wait cannot raise), as it is where node 0's u is not in [0, 1); a draft
    whose u is not may stay or not.  Drafts outside the vocabulary do not stay.  A sequence without rows, or whose node
    0 is no node (its parent is not -1), has count 0."""
    stride = _logits(logits, "logits")
    dev, (T, V) = logits.device, logits.shape
    if tree.device != dev or tree.n_tokens != T:
        raise ValueError(f"tree of {tree.n_tokens} rows on {tree.device}: {T} on {dev} needed")
    _index(tokens, "tokens", 1)
    if tokens.device != dev or tokens.numel() != T or not tokens.is_contiguous():
        raise ValueError(f"tokens must be {T} contiguous values on {dev}")
    if not isinstance(u, torch.Tensor) or u.dtype != torch.float64 or u.device != dev or u.shape != (T,) or not u.is_contiguous():
        raise TypeError(f"u must be {T} contiguous float64 values on {dev}")
    dstride = 0 if draft is None else _logits(draft, "draft", logits)
    temps, temp = None, 0.0
    if isinstance(temperature, torch.Tensor):
        if (temperature.dtype != torch.float32 or temperature.device != dev or temperature.shape != (tree.n_seqs,)
                or not temperature.is_contiguous()):
            raise TypeError(f"temperature must be a number or {tree.n_seqs} contiguous float32 values on {dev}")
        temps = temperature.data_ptr()
    else:
        temp = float(temperature)
        if not temp < math.inf:
            raise ValueError(f"temperature {temp}")
    if records(logits, draft, u) or (temps and records(temperature)):
        raise no_gradients("verify")
    out = [torch.empty(shape, dtype=torch.int32, device=dev) for shape in ((tree.n_seqs, tree.max_nodes),) * 2 + ((tree.n_seqs,),)]
    if tree.n_seqs:
        t = tree._trees()
        ref = ctypes.byref(t)
        n = require_lib().tg_verify_workspace(ref, V)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        run_on(logits, "tg_verify_dev", ref, tree.links.data_ptr(), TYPES[logits.dtype], logits.data_ptr(), stride,
               None if draft is None else draft.data_ptr(), dstride, V, tokens.data_ptr(), u.data_ptr(), temp, temps,
               out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr() if n else None, n)
    return Verified(*out)
