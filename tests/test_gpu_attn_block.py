"""The attention block's operators run together, as an engine runs them:
norm + q | k | v product, append, attend, output product added to x, and the
MoE block behind it; over decode steps, streams and graph replays."""
import numpy as np
import pytest
import torch

from oracle import attn as A
from tests.conftest import gpu_note

pytestmark = pytest.mark.gpu

H, HEADS, KV, D, PAGE = 256, 4, 2, 64, 16


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


class Block:
    def __init__(self, seed, n_pages=40):
        from tinygiant_amd.attn import PagedKV
        rng = np.random.default_rng(seed)
        n = (HEADS + 2 * KV) * D
        i8 = lambda *s: rng.integers(-127, 128, s).astype(np.int8)
        f = lambda *s: rng.uniform(0.5, 1.5, s).astype(np.float32)
        self.h = dict(wqkv=i8(n, H), sqkv=f(n) / 1200, wo=i8(H, HEADS * D), so=f(H) / 1200, norm=f(H), qn=f(D), kn=f(D))
        ang = np.arange(512)[:, None] * 1e4 ** (-np.arange(D // 2) / (D // 2))
        self.h["cos"], self.h["sin"] = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        self.d = {k: torch.from_numpy(v).cuda() for k, v in self.h.items()}
        self.kv = PagedKV(1, n_pages, PAGE, KV, D)

    def step(self, x, batch):
        """x <- x + attention block of x, on the device."""
        from tinygiant_amd.linear import matmul_i8
        d = self.d
        qkv = matmul_i8(x, d["wqkv"], d["sqkv"], norm=d["norm"], out_dtype=torch.float16).view(-1, HEADS + 2 * KV, D)
        q, k, v = qkv.split([HEADS, KV, KV], 1)
        q = self.kv.append(0, q, k, v, batch, d["cos"], d["sin"], q_norm=d["qn"], k_norm=d["kn"])
        o = self.kv.attend(0, q, batch)
        return matmul_i8(o.view(-1, HEADS * D), d["wo"], d["so"], residual=x, out=x)

    def plain(self, x, past, new_of):
        """The same in float64 on the host for one sequence: past holds its
        k, v values so far; x [n, H]."""
        h = self.h
        qkv = A.matmul_i8(x, h["wqkv"], h["sqkv"], h["norm"]).astype(np.float16).astype(np.float32).reshape(len(x), -1, D)
        q, k, v = np.split(qkv, [HEADS, HEADS + KV], 1)
        n0 = past[0].shape[1]
        c, s = (h[n][n0:n0 + len(x)][:, None] for n in ("cos", "sin"))
        q = A.rotate(A.norm_rows(q, h["qn"], 1e-6), c, s).astype(np.float16).astype(np.float64)
        k = A.rotate(A.norm_rows(k, h["kn"], 1e-6), c, s)
        for i, y in enumerate((k, v)):
            code, d = A.q4_0(y)
            y = (code.astype(float) - 8) * np.repeat(d.astype(float), 32, axis=-1)
            past[i] = np.concatenate([past[i], y.transpose(1, 0, 2)], 1)
        o, _, _ = A.attend(q, past[0], past[1], len(x), D ** -0.5)
        return A.matmul_i8(o.reshape(len(x), -1), h["wo"], h["so"], residual=x)


def tables(n_seqs, cols, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).permutation(n_seqs * cols).astype(np.int32).reshape(n_seqs, cols)).cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_prompts_then_decode_steps():
    """Three prompts of different lengths, then steps of one token each: the
    whole run against float64.  Tolerance: a rounding that falls the other
    way moves one Q4_0 or int8 code, 1/16 of a block's range of one key or
    1/127 of a row's; the outputs stay within 1 % of their size."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("block: prompts and decode")
    b, rng = Block(1), np.random.default_rng(2)
    lens = [37, 1, 90]
    past = [[np.zeros((KV, 0, D)), np.zeros((KV, 0, D))] for _ in lens]
    table = tables(3, 8)
    news = list(lens)
    for step in range(4):
        T = sum(news)
        x = rng.standard_normal((T, H)).astype(np.float32)
        cu = np.concatenate([[0], np.cumsum(news)])
        got = b.step(torch.from_numpy(x).cuda(), KVBatch(ints(*cu), ints(*lens), table, max_len=max(lens))).cpu().numpy()
        for i in range(3):
            rows = slice(cu[i], cu[i + 1])
            ref = b.plain(x[rows], past[i], news[i])
            rel = np.linalg.norm(got[rows] - ref) / np.linalg.norm(ref - x[rows])
            assert rel < 1e-2, (step, i, rel)
        news = [1, 1, 1] if step != 1 else [2, 1, 5]
        lens = [n + m for n, m in zip(lens, news)]


def test_with_the_moe_block():
    """Attention block and MoE block of one layer alternate on the same fp32 x."""
    from tinygiant_amd.arena import HBMExpertArena
    from tinygiant_amd.attn import KVBatch
    from tinygiant_amd.moe import MoEBlock
    gpu_note("block: with the MoE block")
    b = Block(3)
    with HBMExpertArena(1, 32, H, 64, 8) as a:
        a.synth_layer(0, seed=5, sigma=0.05)
        moe = MoEBlock(a)
        x = torch.randn(2, H, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        batch = KVBatch(ints(0, 1, 2), ints(1, 1), tables(2, 2))
        y = b.step(x.clone(), batch)
        z = y + moe.forward(0, y)
        w = moe.step(b.step(x.clone(), batch))
        torch.cuda.synchronize()
        assert torch.equal(z, w) and torch.isfinite(w).all() and not torch.equal(w, x)


def test_two_streams_at_once():
    """Two blocks' steps on two streams, interleaved, give what each gives alone."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("block: two streams")
    blocks = [Block(5), Block(6)]
    streams = [torch.cuda.Stream() for _ in blocks]
    batch = KVBatch(ints(0, 60, 61), ints(60, 30), tables(2, 4))
    xs = [torch.randn(61, H, device="cuda") for _ in blocks]
    alone = [b.step(x.clone(), batch) for b, x in zip(blocks, xs)]
    torch.cuda.synchronize()
    ys = [[] for _ in blocks]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                ys[i].append(blocks[i].step(xs[i].clone(), batch))
    torch.cuda.synchronize()
    for want, got in zip(alone, ys):
        for g in got:
            assert torch.equal(want, g)


def test_graph_replays_follow_the_buffers():
    """A captured step replayed while lengths, rows and the table change in
    place, eager work of the same kind and synchronisations between."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("block: graph")
    b, ref = Block(7), Block(7)
    cu, ln, table = ints(0, 1, 2, 3), ints(20, 1, 3), tables(3, 6)
    for blk in (b, ref):
        blk.kv.pages.random_(0, 256, generator=torch.Generator("cuda").manual_seed(3))
        blk.kv.pages[..., 16 * D:].view(torch.float16).normal_(0, 0.2, generator=torch.Generator("cuda").manual_seed(4))
    batch = KVBatch(cu, ln, table, max_len=96)
    x = torch.zeros(3, H, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.step(x.clone(), batch)
    torch.cuda.synchronize()
    b.kv.pages.copy_(ref.kv.pages)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.step(x, batch)
    b.kv.pages.copy_(ref.kv.pages)
    for i in range(4):
        new = torch.randn(3, H, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        x.copy_(new)
        ln.copy_(ints(21 + 7 * i, 2 + i, 90 - i))
        if i == 2:
            table.copy_(tables(3, 6, seed=9))
        g.replay()
        want = ref.step(new.clone(), batch)
        torch.cuda.synchronize()
        assert torch.equal(x, want), i
        assert torch.equal(b.kv.pages, ref.kv.pages), i


def test_results_do_not_change_from_run_to_run():
    from tinygiant_amd.attn import KVBatch
    gpu_note("block: repeat")
    b = Block(8)
    batch = KVBatch(ints(0, 60, 61), ints(60, 30), tables(2, 4))
    x = torch.randn(61, H, device="cuda")
    first = b.step(x.clone(), batch)
    for _ in range(5):
        assert torch.equal(first, b.step(x.clone(), batch))
