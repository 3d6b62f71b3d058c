"""Trees of drafted tokens on the GPU: steps in which one pass of the model
answers several guesses at what follows.

The reference generates one token a pass (tinygiant/engine.py:317-409).  With
drafts, the rows of a sequence in a KVBatch are a tree: node 0 is the last
token that is decided, every other node a guess at what follows its parent.

    tree = DraftTree(batch.cu, n_tokens, parent)        # int32 CUDA tensors; once a step, for all layers
    q = kv.append(layer, q, k, v, batch, cos, sin, tree=tree)   # rotated by depth
    o = kv.attend(layer, q, batch, tree=tree)                   # each node over its own ancestors

Everything runs in libtinygiant.so's gfx950 kernels; torch is used only to
hold device buffers and name the stream.
"""
from __future__ import annotations

import ctypes

import torch

from .attn import _index, run_on


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
    attends them is NaN and nothing of them is appended.  The tensors are read
    when build() is called: again after they were rewritten in place, which may be
    captured into a graph."""

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
        self.build()

    def _trees(self) -> _Trees:
        return _Trees(self.cu.data_ptr(), None if self.parent is None else self.parent.data_ptr(), self.n_seqs,
                      self.n_tokens, self.max_nodes)

    def build(self) -> "DraftTree":
        """bits and depth from cu and parent as they now are."""
        if self.n_tokens and self.n_seqs:
            run_on(self.depth, "tg_draft_tree_dev", ctypes.byref(self._trees()), self.bits.data_ptr(), self.depth.data_ptr())
        return self
