"""Draft trees restated in numpy: what a node sees, which drafted tokens a
target's probabilities keep, and the cache afterwards.

TEST INFRASTRUCTURE ONLY: the oracle that tests/ compare libtinygiant's
tg_draft_tree_dev, tg_verify_dev and tg_kv_keep_q4_dev with.  Nothing in the
product imports it.  Everything is computed in float64, step by step as the
operators are defined.
"""
from __future__ import annotations

import numpy as np


def ancestors(parent, max_nodes=1024):
    """For each node the nodes that it sees, itself the last; None for one that is not of the tree."""
    out = []
    for j, p in enumerate(parent):
        up = [] if p == -1 else out[p] if 0 <= p < j else None
        out.append(None if up is None or j >= max_nodes else up + [j])
    return out


def seen(parent, max_nodes=1024):
    """bool [nodes, nodes]; a node that is not of the tree sees nothing."""
    m = np.zeros((len(parent), len(parent)), bool)
    for j, a in enumerate(ancestors(parent, max_nodes)):
        m[j, a or []] = True
    return m


def words(parent, max_nodes):
    """uint32 [nodes, words] and depths."""
    bits = np.zeros((len(parent), (max_nodes + 31) // 32), np.uint32)
    depth = np.full(len(parent), -1, np.int32)
    for j, a in enumerate(ancestors(parent, max_nodes)):
        for x in a or []:
            bits[j, x // 32] |= np.uint32(1 << (x % 32))
        depth[j] = len(a) - 1 if a else -1
    return bits, depth


def chances(logits, t):
    """softmax(logits / t); t 0 (or below): 1 at the first of the largest.  None: no distribution (NaN, +inf, all -inf)."""
    x = np.asarray(logits, np.float64)
    if not (x < np.inf).all() or x.max() == -np.inf:
        return None
    if not t > 0:
        return (np.arange(len(x)) == np.argmax(x)).astype(np.float64)
    w = np.exp((x - x.max()) / t)
    return w / w.sum()


def walk(logits, tokens, u, parent, t, draft=None, max_nodes=1024):
    """One sequence: the kept nodes, and the tokens that follow (drafts that were kept, then the drawn one; -1 where none can
    be drawn).  Each rejected sibling leaves norm(max(r - q, 0)) of what was left, or r without its token where no one
    drew it."""
    V, n = logits.shape[1], min(len(parent), max_nodes)
    if not n or parent[0] != -1:
        return [], []
    at, path, out = 0, [0], []
    while True:
        full = rest = chances(logits[at], t)
        kids = [j for j in range(at + 1, n) if parent[j] == at]
        q = chances(draft[at], t) if draft is not None and t > 0 and kids else None
        if full is None or (draft is not None and t > 0 and kids and q is None):
            return path, out + [-1]
        for j in kids:
            x = int(tokens[j])
            share = rest / rest.sum() if rest.sum() > 0 else rest
            if not 0 <= x < V:
                # no token: never kept.  Drawn from q all the same: what it leaves is formed like any other's
                if q is not None:
                    rest = np.maximum(share - q, 0)
                continue
            if (u[j] * (1.0 if q is None else q[x]) if t > 0 else 0.0) < share[x]:
                at = j
                break
            rest = rest.copy()
            if q is None:
                rest[x] = 0
            else:
                rest = np.maximum(share - q, 0)
        else:
            break
        path.append(at)
        out.append(int(tokens[at]))
    if not rest.sum() > 0:
        rest = full
    if t > 0 and not 0 <= u[0] < 1:
        return path, out + [-1]
    upto = np.cumsum(rest)
    i = int(np.searchsorted(upto, (u[0] if t > 0 else 0.0) * upto[-1], side="right"))
    return path, out + [min(i, int(np.flatnonzero(rest)[-1]))]


def keep(cache, table_row, n, n_nodes, path):
    """The cache (oracle.attn.Cache) of one layer after the sequence of n tokens, n_nodes of them a tree's, kept the nodes
    of path: entries moved halfword by halfword."""
    base, old, size = n - n_nodes, cache.pages.copy(), cache.page_tokens
    for i, p in enumerate(path):
        a = base + i
        to = cache.pages[table_row[a // size], :, a % size // 16].view(np.uint16)
        if i == p:
            continue
        b = base + p if i <= p < n_nodes else a
        frm = old[table_row[b // size], :, b % size // 16].view(np.uint16)
        for k, (x, y) in enumerate(zip(cache._places(a % 16), cache._places(b % 16))):
            if k not in (1, 3):  # those are nibbles, the same for every token
                to[:, x] = frm[:, y] if b != a else (0x7E00 if k >= 4 else to[:, x])
