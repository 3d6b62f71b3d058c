"""Speculative decoding over the paged cache, as cases that can be timed and compared.

op "append"   DraftTree, PagedKV.append(tree=), PagedKV.read: a tree's ancestors and depths, its tokens' rows into the
              cache with each rotated by its depth, and what the cache then holds for them
op "attend"   PagedKV.attend(tree=): attention of a tree's rows, each over the sequence and its own ancestors
op "verify"   verify: which drafted tokens the target's probabilities keep, by given random numbers, and the token that follows
op "keep"     PagedKV.keep: the kept tokens' cache entries to the places behind the sequence, in every layer

Shapes: the 30B shape (48 layers; 32 query and 4 key heads of 128), the 235B shape (64 and 4 heads of 128), the
151936-token vocabulary, and generic ones.  Node j of a sequence is row cu[s] + j; node 0 is the last token that is
decided, the others are drafts, parent[row] < j the node that they follow.  The cache of one layer is uint8
[n_pages][n_kv_heads][page_tokens / 16][18 D]; a 16-token tile holds K codes (8 D bytes), V codes (8 D), K scales (D), V scales (D):
  K code of token r, dimension 32 g + 8 h + 2 n + p: halfword ((h 16 + r) NG + g) 2 + p, bits 4 n..4 n + 3   (NG = D / 32)
  V code of token r, dimension 16 (4 b + n) + c:     halfword (((r / 4) 16 + c) 2 + (r % 4) / 2) NG + 2 b + r % 2, bits 4 n..
  K scale of token r, block g: half r NG + g;        V scale: half ((r / 2) NG + g) 2 + r % 2
and a code stands for scale (code - 8).
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def listed():
    return [
        # one user on the 30B shape, a tree of 16 nodes after 1000 tokens
        dict(name="append_1_user", op="append", seqs=1, nodes=16, shape="tree", ctx=1016, ragged=False, heads=32, kv=4, dim=128,
             page=16, dtype="bf16", norm=True),
        # 37 users on the 235B shape, trees of up to 61 nodes
        dict(name="append_37_users", op="append", seqs=37, nodes=61, shape="tree", ctx=5003, ragged=True, heads=64, kv=4,
             dim=128, page=64, dtype="f16", norm=True),
        # one user on the 30B shape, a tree of 16 nodes, a context of 2005 tokens
        dict(name="attend_1_user", op="attend", seqs=1, nodes=16, shape="tree", ctx=2005, ragged=False, heads=32, kv=4, dim=128,
             page=16, dtype="bf16"),
        # 32 users on the 30B shape, trees of up to 31 nodes, up to 8192 tokens
        dict(name="attend_32_users", op="attend", seqs=32, nodes=31, shape="tree", ctx=8192, ragged=True, heads=32, kv=4,
             dim=128, page=64, dtype="bf16"),
        # a very long document, 235B shape, a chain of four drafts
        dict(name="attend_long", op="attend", seqs=1, nodes=5, shape="chain", ctx=200003, ragged=False, heads=64, kv=4, dim=128,
             page=128, dtype="f16"),
        # eight users with large trees, heads of 64
        dict(name="attend_large_trees", op="attend", seqs=8, nodes=509, shape="tree", ctx=4001, ragged=True, heads=32, kv=8,
             dim=64, page=32, dtype="f16"),
        # one user, a chain of four drafts with the draft model's logits, the 151936-token vocabulary
        dict(name="verify_1_chain", op="verify", seqs=1, nodes=5, shape="chain", ragged=False, vocab=151936, dtype="bf16",
             draft=True, temperature=0.7),
        # 64 users, chains of up to six drafts, half of the users greedy
        dict(name="verify_64_chains", op="verify", seqs=64, nodes=7, shape="chain", ragged=True, vocab=151936, dtype="f32",
             draft=True, temperature=-1.0),
        # 16 users, trees of up to 60 nodes whose candidates are a draft head's best ones, an odd vocabulary
        dict(name="verify_16_trees", op="verify", seqs=16, nodes=60, shape="tree", ragged=True, vocab=50021, dtype="f32",
             draft=False, temperature=1.0),
        # 4 users, trees whose siblings are drawn from the draft model
        dict(name="verify_4_drawn_trees", op="verify", seqs=4, nodes=26, shape="tree", ragged=False, vocab=151936, dtype="f16",
             draft=True, temperature=1.0),
        # one user on the 30B shape: the kept tokens of 16 nodes in 48 layers
        dict(name="keep_1_user", op="keep", seqs=1, nodes=16, shape="tree", ctx=1016, ragged=False, layers=48, kv=4, dim=128, page=16),
        # 64 users on the 30B shape, trees of up to 31 nodes
        dict(name="keep_64_users", op="keep", seqs=64, nodes=31, shape="tree", ctx=250, ragged=True, layers=48, kv=4, dim=128, page=64),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over the range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify", "verify", "keep"])
    case = dict(op=op, shape=rng.choice(["tree", "tree", "chain"]), ragged=rng.random() < 0.7)
    if op == "verify":
        while True:
            seqs, nodes, vocab = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 2, 151936)
            if seqs * nodes * vocab <= 32 * 7 * 151936:
                break
        return dict(case, seqs=seqs, nodes=nodes, vocab=vocab, dtype=rng.choice(list(DT)), draft=rng.random() < 0.5,
                    temperature=rng.choice([-1.0, 0.0, 0.6, 1.0]))
    kv = rng.choice([1, 2, 4, 5, 8])
    case.update(kv=kv, dim=rng.choice([64, 128, 256]), page=rng.choice([16, 32, 64, 128]))
    if op == "keep":
        while True:
            seqs, nodes, layers = _log(rng, 1, 64), _log(rng, 1, 512), rng.choice([1, 5, 48, 94])
            ctx = nodes + _log(rng, 1, 2000)
            if max(seqs * ctx, 8 * seqs * nodes) * layers * kv * case["dim"] <= 32 * 250 * 48 * 4 * 128:
                break
        return dict(case, seqs=seqs, nodes=nodes, ctx=ctx, layers=layers)
    case["heads"] = kv * rng.choice([1, 2, 3, 4, 7, 8, 16])
    while True:
        seqs, nodes = _log(rng, 1, 64), _log(rng, 1, 1024 if op == "append" else 512)
        ctx = nodes + _log(rng, 1, 200000)
        pairs = seqs * nodes * ctx * case["heads"]
        held = seqs * ctx * kv * case["dim"]
        rows = seqs * nodes * case["heads"] * case["dim"]
        if held <= 200003 * 4 * 128 and rows <= 37 * 30 * 64 * 128 and (op == "append" or pairs <= 4 * 509 * 4001 * 32):
            break
    case.update(seqs=seqs, nodes=nodes, ctx=ctx, dtype=rng.choice(["f16", "bf16"] if op == "attend" else list(DT)))
    if op == "append":
        case["norm"] = rng.random() < 0.5
    return case


def _share(case):
    return [1.0 if i == 0 or not case["ragged"] else (0.37 + 0.6180339887 * i) % 1.0 for i in range(case["seqs"])]


def _nodes(case):
    """Each sequence's nodes: the first has the case's, the others a share of them where it is ragged."""
    return [max(1, int(case["nodes"] * f)) for f in _share(case)]


def _lengths(case):
    """Each sequence's tokens, its nodes among them."""
    return [max(n + 1, int(case["ctx"] * f)) for n, f in zip(_nodes(case), _share(case))]


def _parents(case):
    """Parent of every row, by sequence: the tree's shape is the program's, so it goes by the case alone."""
    rng = random.Random(case["nodes"] * 1000003 + case["seqs"])
    if case["shape"] == "chain":
        return [list(range(-1, n - 1)) for n in _nodes(case)]
    return [[-1] + [int(j * rng.random() ** 1.5) for j in range(1, n)] for n in _nodes(case)]


def work(case):
    nodes = _nodes(case)
    rows = sum(nodes)
    if case["op"] == "verify":
        # rows that something follows, of the target and of the draft, and the drawn token's row where it is another
        inner = sum(len(set(p[1:])) for p in _parents(case))
        size = (inner * (2 if case["draft"] else 1) + len(nodes)) * case["vocab"] * DT[case["dtype"]].itemsize
        return {"bytes": size + rows * 20, "flops": 4 * (inner * (2 if case["draft"] else 1) + len(nodes)) * case["vocab"]}
    if case["op"] == "keep":
        kept = sum(len(p) for p in _paths(case, 0))
        return {"bytes": 2 * kept * case["layers"] * case["kv"] * case["dim"] * 9 // 8, "flops": 0}
    e, d, lens = DT[case["dtype"]].itemsize, case["dim"], _lengths(case)
    words = -(-case["nodes"] // 32)
    if case["op"] == "append":
        held = rows * 2 * case["kv"] * d
        # rows in, q out, the cache's bytes written and read once, the values read back, the tree
        return {"bytes": rows * (2 * case["heads"] + 2 * case["kv"]) * d * e + 2 * held * 9 // 16 + held * 2 + rows * d * 4
                + rows * 4 * (words + 2), "flops": 10 * rows * (case["heads"] + 2 * case["kv"]) * d}
    pairs = sum(n * (ln - n) + sum(len(a) for a in _ancestors(p)) for ln, n, p in zip(lens, nodes, _parents(case)))
    return {"bytes": sum(lens) * 2 * case["kv"] * d * 9 // 16 + 2 * rows * case["heads"] * d * e + rows * 4 * words,
            "flops": 4 * pairs * case["heads"] * d}


def _ancestors(parent):
    """The nodes that each node sees, itself among them."""
    seen = []
    for j, p in enumerate(parent):
        seen.append((seen[p] if p >= 0 else []) + [j])
    return seen


def _paths(case, seed):
    """A path from the root of each sequence's tree, as a walk that stops at some node leaves it."""
    rng = random.Random(seed * 7919 + case["nodes"])
    return [_ancestors(p)[rng.randrange(len(p))] for p in _parents(case)]


# ------------------------------------------------------------------ the cache's layout
def _codes(x):
    """fp32 [..., D] -> Q4_0 codes [..., D] and fp16 scales [..., D / 32]."""
    x = x.clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    top = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = top / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    code = (x * inv + 8.5).to(torch.int32).clamp(max=15)
    return code.flatten(-2), d.squeeze(-1).half()


def _pieces(k, ks, v, vs):
    """The halfwords that tokens [..., Hkv, D] put into their tiles: K codes [.., D / 4], V codes, K scales, V scales."""
    D = k.shape[-1]
    four = torch.tensor([1, 16, 256, 4096], device=k.device, dtype=torch.int32)
    kh = (k.unflatten(-1, (D // 32, 4, 4, 2)) * four[:, None]).sum(-2).flatten(-3)       # [g][h][p]
    vh = (v.unflatten(-1, (D // 64, 4, 16)) * four[:, None]).sum(-2).flatten(-2)         # [b][c]
    return torch.cat([kh.to(torch.int16), vh.to(torch.int16), ks.view(torch.int16), vs.view(torch.int16)], -1)


def _places(r, D):
    """Halfword of each of _pieces' values in its tile, for tokens r [...] of their tiles."""
    NG, dev = D // 32, r.device
    r = r.unsqueeze(-1)
    g, h, p = torch.meshgrid(torch.arange(NG, device=dev), torch.arange(4, device=dev), torch.arange(2, device=dev), indexing="ij")
    b, c = torch.meshgrid(torch.arange(D // 64, device=dev), torch.arange(16, device=dev), indexing="ij")
    n = torch.arange(NG, device=dev)
    return torch.cat([((h * 16).flatten() + r) * NG * 2 + (g * 2 + p).flatten(),
                      4 * D + (((r // 4) * 16 + c.flatten()) * 2 + (r % 4) // 2) * NG + 2 * b.flatten() + r % 2,
                      8 * D + r * NG + n,
                      8 * D + D // 2 + ((r // 2) * NG + n) * 2 + r % 2], -1)


def _values(tiles, D):
    """Tiles int16 [..., 9 D] -> fp32 K and V [..., 16, D]."""
    NG, t = D // 32, tiles.to(torch.int32) & 0xFFFF
    shift = torch.tensor([0, 4, 8, 12], device=t.device, dtype=torch.int32)
    k = t[..., :4 * D].unflatten(-1, (4, 16, NG, 1, 2)) >> shift[:, None] & 15            # [h][r][g][n][p]
    k = k.movedim(-5, -3).flatten(-3).float() - 8.0                                      # [r][g][32]
    v = t[..., 4 * D:8 * D].unflatten(-1, (4, 16, 2, NG // 2, 2))                        # [h][c][a][b][p]
    v = v.movedim((-3, -1), (-4, -3)).unsqueeze(-1) >> shift & 15                        # [h][a][p][c][b][n]
    v = v.movedim(-3, -1).flatten(-6, -4).flatten(-3).float() - 8.0                      # [16][D]
    scales = tiles[..., 8 * D:].contiguous().view(torch.float16).float()
    ks = scales[..., :D // 2].unflatten(-1, (16, NG))
    vs = scales[..., D // 2:].unflatten(-1, (8, NG, 2)).transpose(-1, -2).flatten(-3, -2)
    return (k * ks.unsqueeze(-1)).flatten(-2), (v.unflatten(-1, (NG, 32)) * vs.unsqueeze(-1)).flatten(-2)


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _whole(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _trees(case):
    """The batch's rows and the trees over them."""
    nodes, parents = _nodes(case), _parents(case)
    cu = np.concatenate([[0], np.cumsum(nodes)])
    return {"case": case, "cu": _whole(cu), "rows": int(cu[-1]), "nodes": max(nodes),
            "parent": _whole(np.concatenate(parents)) if case["shape"] == "tree" else None}


def _pool(case, seed, s):
    """The sequences' pages, in an order of their own in a pool with a few to spare."""
    lens = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    pool = list(range(sum(need) + 3))
    random.Random(seed).shuffle(pool)
    table = np.zeros((len(lens), max(need)), np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = pool[at:at + n]
        at += n
    s.update(lens=_whole(lens), table=torch.from_numpy(table).to(DEV), n_pages=len(pool), max_len=max(lens))


def _filled(case, n_pages, gen):
    """Pages of one layer whose tokens are normal keys (channels of different size, a few large) and values."""
    D = case["dim"]
    pages = torch.empty(n_pages, case["kv"], case["page"] // 16, 9 * D, dtype=torch.int16, device=DEV)
    size = torch.exp(0.5 * _normal(gen, case["kv"], 1, 1, D))
    places = _places(torch.arange(16, device=DEV), D).flatten()
    step = max(1, (1 << 25) // (case["kv"] * case["page"] * D))
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        shape = (n, case["kv"], case["page"] // 16, 16, D)
        k, ks = _codes(_normal(gen, *shape) * size)
        v, vs = _codes(_normal(gen, *shape))
        pages[p:p + n][..., places] = _pieces(k, ks, v, vs).flatten(-2)
    return pages


def _drafted(case, s, gen, temperature):
    """Logits of a target and of a draft model near it, and tokens that follow from the draft's: drawn from its probabilities, or
    (without those) its best ones, the first child the best.  Some tokens are forbidden (-inf) to both."""
    T, V = s["rows"], case["vocab"]
    row, parents, cu = [], _parents(case), np.concatenate([[0], np.cumsum(_nodes(case))])
    rank = []
    for i, p in enumerate(parents):
        row += [int(cu[i]) + max(q, 0) for q in p]
        rank += [p[:j].count(q) for j, q in enumerate(p)]
    row, rank = torch.tensor(row, device=DEV), torch.tensor(rank, device=DEV) % V
    seq = torch.repeat_interleave(torch.arange(len(parents), device=DEV), torch.tensor(_nodes(case), device=DEV))
    forbidden = torch.rand(V, generator=gen, device=DEV) < 0.02
    forbidden[0] = False
    target, draft = (torch.empty(T, V, dtype=DT[case["dtype"]], device=DEV) for _ in range(2))
    tokens = torch.empty(T, dtype=torch.int64, device=DEV)
    step = max(1, (1 << 25) // V)
    for a in range(0, T, step):
        n = min(step, T - a)
        x = 2.5 * _normal(gen, n, V)
        target[a:a + n] = x.masked_fill(forbidden, -math.inf)
        draft[a:a + n] = (x + 0.7 * _normal(gen, n, V)).masked_fill(forbidden, -math.inf)
    best = min(V, int(rank.max()) + 1)
    for a in range(0, T, step):
        n = min(step, T - a)
        x = draft[row[a:a + n]].float()
        if case["draft"]:
            t = temperature[seq[a:a + n]].clamp(min=0.3).unsqueeze(1)
            noise = torch.rand(n, V, generator=gen, device=DEV).clamp_(min=1e-30).log_().neg_().clamp_(min=1e-30).log_().neg_()
            tokens[a:a + n] = (x / t + noise).argmax(1)
        else:
            tokens[a:a + n] = x.topk(best, 1).indices.gather(1, rank[a:a + n].clamp(max=best - 1).unsqueeze(1)).squeeze(1)
    s.update(logits=target, draft=draft if case["draft"] else None, tokens=tokens.to(torch.int32))


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    s = _trees(case)
    T = s["rows"]
    if case["op"] == "verify":
        t = case["temperature"]
        # below 0: each user's own, every other one greedy
        each = torch.full((case["seqs"],), t, device=DEV) if t >= 0 else torch.arange(case["seqs"], device=DEV).remainder(2) * 0.7
        _drafted(case, s, gen, each)
        s["u"] = torch.rand(s["rows"], generator=gen, device=DEV, dtype=torch.float64)
        s["temperature"] = t if t >= 0 else each
        if own:
            from tinygiant_amd.draft import DraftTree, verify
            s["verify"], s["tree"] = verify, DraftTree(s["cu"], T, s["parent"], max_nodes=s["nodes"])
        return s
    _pool(case, seed, s)
    D = case["dim"]
    if case["op"] == "keep":
        # whatever bytes a cache holds, but scales that are numbers
        pages = torch.randint(0, 256, (case["layers"], s["n_pages"], case["kv"], case["page"] // 16, 18 * D), generator=gen,
                              device=DEV, dtype=torch.uint8)
        pages[..., 16 * D + 1::2] &= 0xBB
        paths = _paths(case, seed)
        path = np.full((len(paths), s["nodes"]), -1, np.int32)
        for i, p in enumerate(paths):
            path[i, :len(p)] = p
        s.update(pages=pages.view(torch.int16), path=_whole(path), count=_whole([len(p) for p in paths]))
        s["kv_len"] = torch.empty_like(s["lens"])
    elif case["op"] == "attend":
        s["pages"] = _filled(case, s["n_pages"], gen)
        s["q"] = (_normal(gen, T, case["heads"], D) * 1.2).to(DT[case["dtype"]])
    else:
        s["pages"] = torch.zeros(s["n_pages"], case["kv"], case["page"] // 16, 9 * D, dtype=torch.int16, device=DEV)
        size = torch.exp(0.5 * _normal(gen, case["kv"], D))
        rows = torch.cat([_normal(gen, T, case["heads"], D), _normal(gen, T, case["kv"], D) * size,
                          _normal(gen, T, case["kv"], D)], 1).to(DT[case["dtype"]])
        # q, k and v of a fused projection: views of its rows
        s["q"], s["k"], s["v"] = rows.split([case["heads"], case["kv"], case["kv"]], 1)
        angle = torch.arange(s["max_len"], device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            1e6, -torch.arange(D // 2, device=DEV, dtype=torch.float64) * 2 / D)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"], s["k_norm"] = ((0.5 + torch.rand(D, generator=gen, device=DEV)) if case["norm"] else None for _ in range(2))
    if own:
        from tinygiant_amd.attn import KVBatch, PagedKV
        from tinygiant_amd.draft import DraftTree
        pages = s["pages"].view(torch.uint8)
        s["kv"] = PagedKV(case.get("layers", 1), s["n_pages"], case["page"], case["kv"], D,
                          pages=pages if case["op"] == "keep" else pages.unsqueeze(0))
        s["batch"] = KVBatch(s["cu"], s["lens"], s["table"], max_len=s["max_len"])
        # a tree of one step serves all of its layers
        s["tree"] = DraftTree(s["cu"], T, s["parent"], max_nodes=s["nodes"])
    return s


# ------------------------------------------------------------------ plain forms
def _rows(s):
    """Sequence, node and parent's node of each row."""
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    node = row - s["cu"][seq]
    return seq, node, node - 1 if s["parent"] is None else s["parent"].long()


def _seen(s):
    """bool [T][nodes]: the nodes that each row sees; the number of steps doubles each time."""
    seq, node, parent = _rows(s)
    row = torch.arange(s["rows"], device=DEV)
    up = torch.where(parent < 0, row, row - node + parent)                              # a root leads to itself
    seen = torch.zeros(s["rows"], s["nodes"], dtype=torch.bool, device=DEV)
    seen[row, node] = True
    for _ in range(s["nodes"].bit_length()):
        seen, up = seen | seen[up], up[up]
    return seen


def _normed(x, w):
    x = x.float()
    if w is None:
        return x
    r = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True).float() + EPS)
    return x * r * w


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    case, D = s["case"], s["case"]["dim"]
    seq, node, _ = _rows(s)
    seen = _seen(s)
    depth = seen.sum(1) - 1
    base = (s["lens"] - (s["cu"][1:] - s["cu"][:-1])).long()[seq]
    cos, sin = s["cos"][base + depth].unsqueeze(1), s["sin"][base + depth].unsqueeze(1)
    q = _rotated(_normed(s["q"], s["q_norm"]), cos, sin).to(s["q"].dtype)
    k, ks = _codes(_rotated(_normed(s["k"], s["k_norm"]), cos, sin))
    v, vs = _codes(s["v"].float())
    pos = base + node
    page = s["table"][seq, pos // case["page"]].long()
    head = torch.arange(case["kv"], device=DEV)
    tile = (page[:, None] * case["kv"] + head) * (case["page"] // 16) + (pos % case["page"] // 16)[:, None]
    tiles = s["pages"].view(-1, 9 * D)
    tiles[tile.unsqueeze(-1), _places(pos % 16, D).unsqueeze(1)] = _pieces(k, ks, v, vs)
    # read back: the tiles' values at the tokens' places
    kk, vv = _values(tiles[tile], D)
    at = (pos % 16).view(-1, 1, 1, 1).expand(-1, case["kv"], 1, D)
    words = -(-s["nodes"] // 32)
    bits = torch.zeros(s["rows"], words * 32, dtype=torch.int64, device=DEV)
    bits[:, :s["nodes"]] = seen
    bits = (bits.view(-1, words, 32) << torch.arange(32, device=DEV)).sum(-1)
    return {"q": q, "k": kk.gather(2, at).squeeze(2).half(), "v": vv.gather(2, at).squeeze(2).half(),
            "bits": torch.where(bits < 1 << 31, bits, bits - (1 << 32)).to(torch.int32), "depth": depth.to(torch.int32)}


def _plain_attend(s):
    case, D = s["case"], s["case"]["dim"]
    B, H, L = case["seqs"], case["kv"], s["table"].shape[1] * case["page"]
    G, N = case["heads"] // H, s["nodes"]
    k, v = _values(s["pages"][s["table"].long()].transpose(1, 2), D)                     # [B][H][pages][tiles][16][D]
    k, v = k.reshape(B * H, L, D), v.reshape(B * H, L, D)
    seq, node, _ = _rows(s)
    q = torch.zeros(B, N, H, G, D, device=DEV)
    q[seq, node] = s["q"].float().view(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B * H, G * N, D)
    base = (s["lens"] - (s["cu"][1:] - s["cu"][:-1])).long()
    tok = torch.arange(L, device=DEV) - base[:, None]                                    # token's node [B][L], below 0 before the tree
    seen = torch.zeros(B, N, N, dtype=torch.bool, device=DEV)
    seen[seq, node] = _seen(s)
    hidden = ~(seen.gather(2, tok.clamp(0, N - 1).unsqueeze(1).expand(B, N, L)) & (tok < N).unsqueeze(1) | (tok < 0).unsqueeze(1))
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, G, N, L)
    score.masked_fill_(hidden.view(B, 1, 1, N, L), -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = score.sum(-1).unsqueeze(-1)
    out = torch.matmul(score.view(B * H, G * N, L), v).view(B, H, G, N, D) / total
    return out.permute(0, 3, 1, 2, 4)[seq, node].reshape(-1, case["heads"], D).to(s["q"].dtype)


def _plain_verify(s):
    B, N, V = s["case"]["seqs"], s["nodes"], s["case"]["vocab"]
    first, n = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    _, _, parent = _rows(s)
    t = torch.as_tensor(s["temperature"], dtype=torch.float32, device=DEV).double().expand(B).unsqueeze(1)

    def chances(x):  # in 64 bits: what a random number next to a border decides is compared
        x = x.double()
        best = torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
        return torch.where(t > 0, torch.softmax(x / torch.where(t > 0, t, torch.ones_like(t)), 1), best)

    seq = torch.arange(B, device=DEV)
    at = torch.zeros(B, dtype=torch.int64, device=DEV)                                   # the node that the walk stands at
    count = torch.ones_like(at)
    path, tokens = (torch.full((B, N), -1, dtype=torch.int64, device=DEV) for _ in range(2))
    path[:, 0] = 0
    whole = p = chances(s["logits"][first])
    drawn = (t > 0).double()                                                             # a greedy walk asks nothing of the draft's
    q = None if s["draft"] is None else chances(s["draft"][first]) * drawn
    left, taken = torch.ones(B, device=DEV, dtype=torch.float64), torch.zeros(B, device=DEV, dtype=torch.float64)
    # nodes follow their parents, so one sweep over them in order is the walk
    for j in range(1, N):
        row = torch.minimum(first + j, first + n - 1)
        asked = (j < n) & (parent[row] == at)
        x = s["tokens"][row].long().unsqueeze(1)
        px, u = p.gather(1, x).squeeze(1), s["u"][row]
        if q is None:
            yes = asked & (u * left < px) & (px > 0)
            no = (asked & ~yes).unsqueeze(1)
            left = torch.where(asked & ~yes, left - px, left)
            p = torch.where(no, p.scatter(1, x, 0.0), p)
        else:
            qx = q.gather(1, x).squeeze(1)
            yes = asked & (u * left * qx < px - taken * qx)
            taken = torch.where(asked & ~yes, taken + left, taken)
            left = torch.where(asked & ~yes, (p - taken.unsqueeze(1) * q).clamp_(min=0).sum(1), left)
            q = torch.where(yes.unsqueeze(1), chances(s["draft"][row]) * drawn, q)
        tokens[seq, count - 1] = torch.where(yes, x.squeeze(1), tokens[seq, count - 1])
        path[seq, count.clamp(max=N - 1)] = torch.where(yes, torch.full_like(at, j), path[seq, count.clamp(max=N - 1)])
        count, at = count + yes, torch.where(yes, torch.full_like(at, j), at)
        left, taken = torch.where(yes, torch.ones_like(left), left), torch.where(yes, torch.zeros_like(taken), taken)
        new = chances(s["logits"][row])
        whole, p = torch.where(yes.unsqueeze(1), new, whole), torch.where(yes.unsqueeze(1), new, p)
    rest = p if q is None else (p - taken.unsqueeze(1) * q).clamp_(min=0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, whole)
    upto = rest.cumsum(1)
    tokens[seq, count - 1] = torch.searchsorted(upto, s["u"][first].unsqueeze(1) * upto[:, -1:], right=True).squeeze(1).clamp(max=V - 1)
    return {"tokens": tokens.to(torch.int32), "path": path.to(torch.int32), "count": count.to(torch.int32)}


def _plain_keep(s):
    case, D = s["case"], s["case"]["dim"]
    B, P = s["path"].shape
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    base = s["lens"].long() - n
    i = torch.arange(P, device=DEV).expand(B, P)
    to = torch.minimum(i, n.unsqueeze(1) - 1)                                            # behind a tree's end: its last node
    frm = torch.where(i < s["count"].unsqueeze(1), s["path"].long(), to)                 # what is not kept stays
    tiles = s["pages"].view(case["layers"], -1, 9 * D)
    head, seq = torch.arange(case["kv"], device=DEV), torch.arange(B, device=DEV).unsqueeze(1)

    def places(node):
        pos = base.unsqueeze(1) + node
        page = s["table"][seq, pos // case["page"]].long()
        tile = (page.unsqueeze(-1) * case["kv"] + head) * (case["page"] // 16) + (pos % case["page"] // 16).unsqueeze(-1)
        return tile.unsqueeze(-1), _places(pos % 16, D).unsqueeze(2)

    a, b = places(frm)
    moved = tiles[:, a, b]
    a, b = places(to)
    tiles[:, a, b] = moved
    s["kv_len"].copy_(base + s["count"])
    return {"pages": s["pages"], "kv_len": s["kv_len"]}


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "verify":
            r = s["verify"](s["logits"], s["tokens"], s["u"], s["tree"], draft=s["draft"], temperature=s["temperature"])
            return {"tokens": r.tokens, "path": r.path, "count": r.count}
        if op == "attend":
            return s["kv"].attend(0, s["q"], s["batch"], tree=s["tree"])
        if op == "keep":
            s["kv"].keep(s["batch"], s["path"], s["count"], kv_len=s["kv_len"])
            return {"pages": s["pages"], "kv_len": s["kv_len"]}
        s["tree"].build()
        q = s["kv"].append(0, s["q"], s["k"], s["v"], s["batch"], s["cos"], s["sin"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=EPS, tree=s["tree"])
        k, v = s["kv"].read(0, s["batch"], s["rows"])
        return {"q": q, "k": k, "v": v, "bits": s["tree"].bits, "depth": s["tree"].depth}
    return {"verify": _plain_verify, "attend": _plain_attend, "keep": _plain_keep, "append": _plain_append}[op](s)


# ------------------------------------------------------------------ the definition in 64 bits
def _held(s, page_ids, n):
    """K and V [n][Hkv][D] of the first n tokens on these pages, value by value from the layout."""
    case, D = s["case"], s["case"]["dim"]
    NG, t, dim = D // 32, torch.arange(n, device=DEV), torch.arange(D, device=DEV)
    r = (t % 16)[:, None]
    flat = s["pages"].reshape(-1)
    base = (page_ids.long()[t // case["page"]][:, None] * case["kv"] + torch.arange(case["kv"], device=DEV)) * (case["page"] // 16)
    base = ((base + (t % case["page"] // 16)[:, None]) * 9 * D).unsqueeze(-1)            # [n][Hkv][1]
    g, e = dim // 32, dim % 32
    j, c = dim // 16, dim % 16
    kat, kn = ((e // 8 * 16 + r) * NG + g) * 2 + e % 2, e % 8 // 2
    vat, vn = 4 * D + ((r // 4 * 16 + c) * 2 + r % 4 // 2) * NG + 2 * (j // 4) + r % 2, j % 4
    ksat, vsat = 8 * D + r * NG + g, 8 * D + D // 2 + (r // 2 * NG + g) * 2 + r % 2
    got = []
    for at, nib, sat in ((kat, kn, ksat), (vat, vn, vsat)):
        code = torch.bitwise_and(torch.bitwise_right_shift(flat[base + at.unsqueeze(1)].to(torch.int32), 4 * nib), 15)
        got.append((code - 8).double() * flat[base + sat.unsqueeze(1)].view(torch.float16).double())
    return got


def _q40(x):
    """fp64 [..., D] -> the fp64 values that Q4_0 blocks of 32 hold for it."""
    x = x.clamp(-65504, 65504).reshape(*x.shape[:-1], -1, 32)
    size = x.abs()
    first = (size == size.amax(-1, keepdim=True)).to(torch.int8).argmax(-1, keepdim=True)
    d = torch.take_along_dim(x, first, -1) / -8
    code = torch.where(d == 0, torch.full_like(x, 8.0), torch.floor(x / d + 8.5).clamp(0, 15))
    return ((code - 8) * d.half().double()).flatten(-2)


def _exact_walk(s, i, start, parent):
    """One sequence's kept nodes and tokens."""
    t = float(torch.as_tensor(s["temperature"], dtype=torch.float32).reshape(-1).expand(s["case"]["seqs"])[i])
    tokens, u = s["tokens"].tolist(), s["u"].tolist()

    def chance(x):
        x = x.double()
        if t <= 0:
            return (torch.arange(len(x), device=DEV) == int((x == x.max()).nonzero()[0])).double()
        w = torch.exp((x - x.max()) / t)
        return w / w.sum()

    at, path, got = 0, [0], []
    while True:
        full = rest = chance(s["logits"][start + at])
        q = chance(s["draft"][start + at]) if s["draft"] is not None and t > 0 else None
        step = None
        for j in range(at + 1, len(parent)):
            if parent[j] != at:
                continue
            x = tokens[start + j]
            share = rest / rest.sum() if float(rest.sum()) > 0 else rest
            if u[start + j] * (1.0 if q is None else float(q[x])) < float(share[x]):
                step = j
                break
            if q is None:
                rest = rest.clone()
                rest[x] = 0
            else:
                rest = torch.relu(share - q)
        if step is None:
            break
        at = step
        path.append(at)
        got.append(tokens[start + at])
    rest = rest if float(rest.sum()) > 0 else full
    upto = torch.cumsum(rest, 0)
    got.append(int((upto > u[start] * upto[-1]).nonzero()[0]))
    return path, got


def exact(case, seed):
    s = prepare(case, seed)
    parents, start = _parents(case), 0
    if case["op"] == "verify":
        out = {k: torch.full((case["seqs"], s["nodes"]), -1, dtype=torch.int32) for k in ("tokens", "path")}
        out["count"] = torch.zeros(case["seqs"], dtype=torch.int32)
        for i, parent in enumerate(parents):
            path, got = _exact_walk(s, i, start, parent)
            out["path"][i, :len(path)], out["tokens"][i, :len(got)], out["count"][i] = _whole(path).cpu(), _whole(got).cpu(), len(path)
            start += len(parent)
        return out
    lens, D = _lengths(case), case["dim"]
    if case["op"] == "keep":
        half = s["pages"].view(case["layers"], s["n_pages"], case["kv"], case["page"] // 16, 9 * D)
        old, table, place = half.clone(), s["table"].tolist(), _places(torch.arange(16, device=DEV), D)
        for i, (path, n, parent) in enumerate(zip(_paths(case, seed), lens, parents)):
            base = n - len(parent)
            for to, frm in enumerate(path):
                if to != frm:
                    a, b = base + to, base + frm
                    pa, pb = table[i][a // case["page"]], table[i][b // case["page"]]
                    half[:, pa, :, a % case["page"] // 16, place[a % 16]] = old[:, pb, :, b % case["page"] // 16, place[b % 16]]
        return {"pages": s["pages"], "kv_len": _whole([n - len(p) + len(k) for n, p, k in zip(lens, parents, _paths(case, seed))])}
    if case["op"] == "append":
        def turned(x, w, cos, sin):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
            a, b = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

        out = {"q": [], "k": [], "v": []}
        bits = np.zeros((s["rows"], -(-s["nodes"] // 32)), np.uint32)
        depths = []
        for n, parent in zip(lens, parents):
            seen = _ancestors(parent)
            rows, at = slice(start, start + len(parent)), torch.tensor([n - len(parent) + len(a) - 1 for a in seen], device=DEV)
            cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
            out["q"].append(turned(s["q"][rows], s["q_norm"], cos, sin))
            out["k"].append(_q40(turned(s["k"][rows], s["k_norm"], cos, sin)))
            out["v"].append(_q40(s["v"][rows].double()))
            for j, a in enumerate(seen):
                for x in a:
                    bits[start + j, x // 32] |= np.uint32(1 << (x % 32))
                depths.append(len(a) - 1)
            start += len(parent)
        out = {name: torch.cat(v) for name, v in out.items()}
        return dict(out, bits=torch.from_numpy(bits.view(np.int32)), depth=torch.tensor(depths, dtype=torch.int32))
    out = torch.empty(s["rows"], case["heads"], D, dtype=torch.float64, device=DEV)
    G = case["heads"] // case["kv"]
    for i, (n, parent) in enumerate(zip(lens, parents)):
        new = len(parent)
        k, v = _held(s, s["table"][i], n)
        hide = torch.zeros(new, n, dtype=torch.bool)
        hide[:, n - new:] = True
        for j, a in enumerate(_ancestors(parent)):
            hide[j, [n - new + x for x in a]] = False
        hide = hide.to(DEV)
        for head in range(case["heads"]):
            p = torch.mm(s["q"][start:start + new, head].double(), k[:, head // G].t()) / math.sqrt(D)
            p.masked_fill_(hide, -math.inf)
            out[start:start + new, head] = torch.mm(torch.softmax(p, 1), v[:, head // G])
        start += new
    return out
