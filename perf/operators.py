"""An attention block's operators on the device, as cases that can be timed and compared.

op "append"   PagedKV.append, then PagedKV.read of the same tokens: head norm and rotation of new q and k rows, k and v
              into the paged Q4_0 cache, and what the cache then holds for them
op "attend"   PagedKV.attend: causal grouped-query attention of a ragged batch over that cache
op "product"  matmul_i8: int8 product with a scale per token (quantised on the way, after an RMS norm where one is
              given) and per channel, added to a residual where one is given

Shapes: the 30B shape (embedding 2048; 32 query and 4 key heads of 128), the 235B shape (4096; 64 and 4 heads of 128), the
151936-token vocabulary, and generic ones.  The cache of one layer is uint8 [n_pages][n_kv_heads][page_tokens / 16][18 D];
a 16-token tile holds K codes (8 D bytes), V codes (8 D), K scales (D), V scales (D):
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
        # one user decoding on the 30B shape: one token's rows into a cache of 1000 tokens
        dict(name="append_1_token", op="append", seqs=1, new=1, ctx=1000, ragged=False, heads=32, kv=4, dim=128, page=16,
             dtype="bf16", norm=True),
        # batched decode on the 235B shape, 61 sequences of different lengths
        dict(name="append_61_tokens", op="append", seqs=61, new=1, ctx=5003, ragged=True, heads=64, kv=4, dim=128, page=64,
             dtype="f16", norm=True),
        # prompt processing: three prompts of different lengths, fp32 rows, a model without head norms
        dict(name="append_prompts_f32", op="append", seqs=3, new=3001, ctx=3001, ragged=True, heads=32, kv=8, dim=64,
             page=32, dtype="f32", norm=False),
        # one user decoding on the 30B shape, a context of 2005 tokens
        dict(name="attend_1_token", op="attend", seqs=1, new=1, ctx=2005, ragged=False, heads=32, kv=4, dim=128, page=16,
             dtype="bf16"),
        # batched decode on the 30B shape, 64 sequences of up to 8192 tokens
        dict(name="attend_64_tokens", op="attend", seqs=64, new=1, ctx=8192, ragged=True, heads=32, kv=4, dim=128, page=64,
             dtype="bf16"),
        # two users with very long documents, 235B shape: few rows, a long axis
        dict(name="attend_long", op="attend", seqs=2, new=1, ctx=200003, ragged=True, heads=64, kv=4, dim=128, page=128,
             dtype="f16"),
        # prompt processing on the 30B shape: three prompts, the longest of 4096 tokens
        dict(name="attend_prompts", op="attend", seqs=3, new=4096, ctx=4096, ragged=True, heads=32, kv=4, dim=128, page=64,
             dtype="bf16"),
        # a chunk of 500 tokens of two long prompts, heads of 64
        dict(name="attend_chunk", op="attend", seqs=2, new=500, ctx=16001, ragged=False, heads=32, kv=8, dim=64, page=32,
             dtype="f16"),
        # q, k and v projections of one token on the 30B shape, with the norm before them
        dict(name="product_1_token", op="product", m=1, n=5120, k=2048, x="f32", out="bf16", norm=True, add=False),
        # the vocabulary head for seven sequences
        dict(name="product_vocab_7", op="product", m=7, n=151936, k=2048, x="f32", out="f32", norm=True, add=False),
        # the output projection of a prompt of odd length on the 30B shape, added to the residual
        dict(name="product_out_1999", op="product", m=1999, n=2048, k=4096, x="bf16", out="f32", norm=False, add=True),
        # q, k and v projections of a large prefill on the 235B shape
        dict(name="product_8192", op="product", m=8192, n=9216, k=4096, x="f32", out="bf16", norm=True, add=False),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over the range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "product"])
    if op == "product":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 16, 151936), 16 * _log(rng, 4, 1024)
            if m * n * k <= 8192 * 9216 * 4096 and m * n <= 8192 * 9216:
                break
        return dict(op=op, m=m, n=n, k=k, x=rng.choice(list(DT)), out=rng.choice(list(DT)), norm=rng.random() < 0.5,
                    add=rng.random() < 0.3)
    kv = rng.choice([1, 2, 4, 5, 8])
    case = dict(op=op, kv=kv, heads=kv * rng.choice([1, 2, 3, 4, 7, 8, 16]), dim=rng.choice([64, 128, 256]),
                page=rng.choice([16, 32, 64, 128]), ragged=rng.random() < 0.7)
    kind = rng.choice(["decode", "few", "prompt", "chunk"])
    while True:
        seqs = _log(rng, 1, 64)
        ctx = _log(rng, 1, 200000)
        new = 1 if kind == "decode" else min(ctx, rng.randint(2, 8)) if kind == "few" else ctx if kind == "prompt" else min(ctx, _log(rng, 16, 2048))
        pairs = seqs * new * ctx * case["heads"] * case["dim"]
        held = seqs * ctx * kv * case["dim"]
        rows = seqs * new * case["heads"] * case["dim"]
        if pairs <= 3 * 4096 * 4096 * 32 * 128 and held <= 64 * 8192 * 4 * 128 and rows <= 3 * 4096 * 32 * 128:
            break
    case.update(seqs=seqs, new=new, ctx=ctx, dtype=rng.choice(["f16", "bf16"] if op == "attend" else list(DT)))
    if op == "append":
        case["norm"] = rng.random() < 0.5
    return case


def _lengths(case):
    """Each sequence's length and its new tokens: the first has the case's, the others a share of it where it is ragged."""
    share = [1.0 if i == 0 or not case["ragged"] else (0.37 + 0.6180339887 * i) % 1.0 for i in range(case["seqs"])]
    lens = [max(1, int(case["ctx"] * f)) for f in share]
    news = [max(1, min(n, int(case["new"] * f))) for n, f in zip(lens, share)]
    return lens, news


def work(case):
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        size = m * k * DT[case["x"]].itemsize + n * k + 4 * n + m * n * DT[case["out"]].itemsize * (2 if case["add"] else 1)
        return {"bytes": size + (4 * k if case["norm"] else 0), "flops": 2 * m * n * k}
    lens, news = _lengths(case)
    e, d, rows = DT[case["dtype"]].itemsize, case["dim"], sum(news)
    if case["op"] == "append":
        held = rows * 2 * case["kv"] * d
        # rows in, q out, the cache's bytes written and read once, the values read back
        return {"bytes": rows * (2 * case["heads"] + 2 * case["kv"]) * d * e + 2 * held * 9 // 16 + held * 2 + rows * d * 4,
                "flops": 10 * rows * (case["heads"] + 2 * case["kv"]) * d}
    pairs = sum(n * ln - n * (n - 1) // 2 for ln, n in zip(lens, news))
    return {"bytes": sum(lens) * 2 * case["kv"] * d * 9 // 16 + 2 * rows * case["heads"] * d * e,
            "flops": 4 * pairs * case["heads"] * d}


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
def _seeded(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _batch(case, seed):
    """Lengths, and the sequences' pages in an order of their own in a pool with a few to spare."""
    lens, news = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    pool = list(range(sum(need) + 3))
    random.Random(seed).shuffle(pool)
    table = np.zeros((len(lens), max(need)), np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = pool[at:at + n]
        at += n
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cu = np.concatenate([[0], np.cumsum(news)])
    return {"case": case, "lens": whole(lens), "cu": whole(cu), "table": torch.from_numpy(table).to(DEV),
            "n_pages": len(pool), "rows": int(cu[-1]), "max_new": max(news), "max_len": max(lens)}


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


def prepare(case, seed):
    gen = _seeded(seed)
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        w = torch.randint(-127, 128, (n, k), generator=gen, device=DEV, dtype=torch.int8)
        s = {"case": case, "w": w, "scale": (0.5 + torch.rand(n, generator=gen, device=DEV)) * (0.02 / 73.0),
             "x": (_normal(gen, m, k) * (0.2 + 2.0 * torch.rand(m, 1, generator=gen, device=DEV))).to(DT[case["x"]]),
             "norm": 0.5 + torch.rand(k, generator=gen, device=DEV) if case["norm"] else None,
             "add": _normal(gen, m, n).to(DT[case["out"]]) if case["add"] else None}
        return s
    s = _batch(case, seed)
    D, T = case["dim"], s["rows"]
    if case["op"] == "attend":
        s["pages"] = _filled(case, s["n_pages"], gen)
        s["q"] = (_normal(gen, T, case["heads"], D) * 1.2).to(DT[case["dtype"]])
    else:
        s["pages"] = torch.zeros(s["n_pages"], case["kv"], case["page"] // 16, 9 * D, dtype=torch.int16, device=DEV)
        size = torch.exp(0.5 * _normal(gen, case["kv"], D))
        rows = torch.cat([_normal(gen, T, case["heads"], D), _normal(gen, T, case["kv"], D) * size,
                          _normal(gen, T, case["kv"], D)], 1).to(DT[case["dtype"]])
        # q, k and v of a fused projection: views of its rows
        s["q"], s["k"], s["v"] = rows.split([case["heads"], case["kv"], case["kv"]], 1)
        angle = torch.arange(case["ctx"], device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            1e6, -torch.arange(D // 2, device=DEV, dtype=torch.float64) * 2 / D)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"], s["k_norm"] = ((0.5 + torch.rand(D, generator=gen, device=DEV)) if case["norm"] else None for _ in range(2))
    if own:
        from tinygiant_amd.attn import KVBatch, PagedKV
        s["kv"] = PagedKV(1, s["n_pages"], case["page"], case["kv"], D, pages=s["pages"].view(torch.uint8).unsqueeze(0))
        s["batch"] = KVBatch(s["cu"], s["lens"], s["table"], max_len=s["max_len"])
    return s


# ------------------------------------------------------------------ plain forms
def _tokens(s):
    """Sequence and position of each row."""
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    return seq, s["lens"][seq].long() - s["cu"][seq + 1] + row


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
    seq, pos = _tokens(s)
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    q = _rotated(_normed(s["q"], s["q_norm"]), cos, sin).to(s["q"].dtype)
    k, ks = _codes(_rotated(_normed(s["k"], s["k_norm"]), cos, sin))
    v, vs = _codes(s["v"].float())
    page = s["table"][seq, pos // case["page"]].long()
    head = torch.arange(case["kv"], device=DEV)
    tile = (page[:, None] * case["kv"] + head) * (case["page"] // 16) + (pos % case["page"] // 16)[:, None]
    tiles = s["pages"].view(-1, 9 * D)
    tiles[tile.unsqueeze(-1), _places(pos % 16, D).unsqueeze(1)] = _pieces(k, ks, v, vs)
    # read back: the tiles' values at the tokens' places
    kk, vv = _values(tiles[tile], D)
    at = (pos % 16).view(-1, 1, 1, 1).expand(-1, case["kv"], 1, D)
    return {"q": q, "k": kk.gather(2, at).squeeze(2).half(), "v": vv.gather(2, at).squeeze(2).half()}


def _plain_attend(s):
    case, D = s["case"], s["case"]["dim"]
    B, H, L = case["seqs"], case["kv"], s["table"].shape[1] * case["page"]
    G, N = case["heads"] // H, s["max_new"]
    k, v = _values(s["pages"][s["table"].long()].transpose(1, 2), D)                     # [B][H][pages][tiles][16][D]
    k, v = k.reshape(B * H, L, D), v.reshape(B * H, L, D)
    seq, pos = _tokens(s)
    at = torch.arange(s["rows"], device=DEV) - s["cu"][seq]
    q = torch.zeros(B, N, H, G, D, device=DEV)
    q[seq, at] = s["q"].float().view(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B * H, G * N, D)
    own_pos = torch.full((B, N), -1, device=DEV)
    own_pos[seq, at] = pos
    hidden = torch.arange(L, device=DEV) > own_pos.unsqueeze(-1)                         # [B][N][L]
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, G, N, L)
    score.masked_fill_(hidden.view(B, 1, 1, N, L), -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = score.sum(-1).unsqueeze(-1)
    out = torch.matmul(score.view(B * H, G * N, L), v).view(B, H, G, N, D) / total
    return out.permute(0, 3, 1, 2, 4)[seq, at].reshape(-1, case["heads"], D).to(s["q"].dtype)


def _plain_product(s):
    # codes next to a border decide by 64 bits: half the largest value of a row lies on one
    x = s["x"].double()
    if s["norm"] is not None:
        x = x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)) * s["norm"].double()
    top = x.abs().amax(-1, keepdim=True)
    code = torch.where(top == 0, torch.zeros_like(x), torch.round(x * 127.0 / top))
    out = torch.matmul(code.float(), s["w"].float().t()) * (top / 127.0).float() * s["scale"]
    if s["add"] is not None:
        out = out + s["add"].float()
    return out.to(DT[s["case"]["out"]])


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "product":
            from tinygiant_amd.linear import matmul_i8
            return matmul_i8(s["x"], s["w"], s["scale"], norm=s["norm"], eps=EPS, residual=s["add"],
                             out_dtype=DT[s["case"]["out"]])
        if op == "attend":
            return s["kv"].attend(0, s["q"], s["batch"])
        q = s["kv"].append(0, s["q"], s["k"], s["v"], s["batch"], s["cos"], s["sin"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=EPS)
        k, v = s["kv"].read(0, s["batch"], s["rows"])
        return {"q": q, "k": k, "v": v}
    return _plain_product(s) if op == "product" else _plain_attend(s) if op == "attend" else _plain_append(s)


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


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        x = s["x"].double()
        if s["norm"] is not None:
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["k"] + EPS) * s["norm"].double()
        a = x.abs().amax(1, keepdim=True)
        code = torch.round(127 * x / a).nan_to_num()
        out = torch.mm(code, s["w"].double().t()) * (a / 127) * s["scale"].double()
        return out if s["add"] is None else out + s["add"].double()
    lens, news = _lengths(case)
    D, start = case["dim"], 0
    if case["op"] == "append":
        def turned(x, w, cos, sin):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
            a, b = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

        out = {"q": [], "k": [], "v": []}
        for n, new in zip(lens, news):
            rows, at = slice(start, start + new), slice(n - new, n)
            cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
            out["q"].append(turned(s["q"][rows], s["q_norm"], cos, sin))
            out["k"].append(_q40(turned(s["k"][rows], s["k_norm"], cos, sin)))
            out["v"].append(_q40(s["v"][rows].double()))
            start += new
        return {name: torch.cat(v) for name, v in out.items()}
    out = torch.empty(s["rows"], case["heads"], D, dtype=torch.float64, device=DEV)
    G = case["heads"] // case["kv"]
    for i, (n, new) in enumerate(zip(lens, news)):
        k, v = _held(s, s["table"][i], n)
        hide = torch.ones(new, n, dtype=torch.bool, device=DEV).triu(n - new + 1)
        for head in range(case["heads"]):
            p = torch.mm(s["q"][start:start + new, head].double(), k[:, head // G].t()) / math.sqrt(D)
            p.masked_fill_(hide, -math.inf)
            out[start:start + new, head] = torch.mm(torch.softmax(p, 1), v[:, head // G])
        start += new
    return out
