"""Calls of the attention block that its documentation allows, each of which
once went wrong: views of page tables, blocks that are not finite next to
others, rows that are not all there, scores beyond ordinary sizes.  Bounds are
those of test_gpu_attn.py."""
import numpy as np
import pytest
import torch

from oracle import attn as A
from tests.conftest import gpu_note
from tests.test_gpu_attn import DT, Setup, check_attend, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 40, 100]])
@pytest.mark.parametrize("view", ["expanded", "columns", "every other row"])
def test_views_of_page_tables(view, news):
    """One row expanded to all sequences (a prefix that they share), columns and rows of a wider table."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"table views {view} {news}")
    lens = [70, 90, 110]
    s = Setup(51, 128, 2, 16, lens, news)
    if view == "expanded":
        s.table[:] = s.table[2]
        table = dev(s.table[2]).expand(3, -1)
    elif view == "columns":
        table = torch.full((3, s.table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")[:, 2:-3]
    else:
        table = torch.full((5, s.table.shape[1]), -9, dtype=torch.int32, device="cuda")[::2]
    if view != "expanded":
        table.copy_(dev(s.table))
    batch = KVBatch(s.batch.cu, s.batch.kv_len, table, max_len=110)
    q, qn = s.rows(8, "bf16")
    check_attend(s, q, qn, s.kv.attend(0, q, batch))
    k, v = s.kv.read(0, batch, s.T)
    for i, (n, new) in enumerate(zip(lens, news)):
        kr, vr = s.cache.rows(s.table[i], n)
        for got, ref in ((k, kr), (v, vr)):
            assert np.array_equal(got[s.cu[i]:s.cu[i + 1]].cpu().numpy(), ref[:, n - new:].transpose(1, 0, 2).astype(np.float16))


def test_overlapping_rows_of_a_page_table_are_refused():
    from tinygiant_amd.attn import KVBatch
    s = Setup(52, 64, 1, 16, [40, 40], [1, 1])
    with pytest.raises(ValueError, match="overlap"):
        KVBatch(s.batch.cu, s.batch.kv_len, torch.as_strided(s.batch.table, (2, 3), (1, 1)))


# ---------------------------------------------------------------- blocks that are not finite
def value_scales(s, i, t):
    """The value scales of token t of sequence i as bits [n_kv, D / 32], to be written in place."""
    tiles = s.cache.pages[s.table[i, t // s.page], :, t % s.page // 16].view(np.uint16)
    at = s.cache._places(t % 16)[5]
    return tiles, at


def set_scales(s, i, t, f):
    """Token t's value scales multiplied by f, or set to it where it is not finite."""
    tiles, at = value_scales(s, i, t)
    old = tiles[:, at].view(np.float16)
    tiles[:, at] = (old * np.float16(f) if np.isfinite(f) else np.full_like(old, f)).view(np.uint16)


class Prefix:
    """Sequence 0 of s without its tokens from n on, and its first rows."""

    def __init__(self, s, n, new):
        self.lens, self.news, self.cu, self.table, self.cache, self.D = [n], [new], [0, new], s.table, s.cache, s.D


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what", ["page", "nan pair", "inf pair", "nan other tile"])
@pytest.mark.parametrize("factor", [16, 256, 2048])
@pytest.mark.parametrize("G,after,dt", [(2, 4, "f16"), (1, 16, "bf16"), (5, 1, "f16")])
def test_a_block_that_is_not_finite_stays_in_the_rows_that_see_it(D, what, factor, G, after, dt):
    """Rows before it are as exact as ever, also where the largest value scales so far stand next to it: in the other
    tile of its 32 tokens, or in the other half of its pair."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend not finite {D} {what} {factor} {G} {after}")
    bad = {"page": 144, "nan pair": 137, "inf pair": 137, "nan other tile": 148}[what]  # the token that is not finite
    large = {"page": [128, 129], "nan pair": [136], "inf pair": [136], "nan other tile": [132]}[what]
    before = 3 if bad == 137 else 6  # rows that do not see it; the last one does see the large scales
    s = Setup(60 + D, D, 2, 16, [bad + after], [before + after])
    for t in large:
        set_scales(s, 0, t, factor)
    table = s.table.copy()
    if what == "page":
        table[0, bad // 16] = -1
    else:
        set_scales(s, 0, bad, np.inf if what == "inf pair" else np.nan)
    s.kv.pages.copy_(dev(s.all))
    q, qn = s.rows(2 * G, dt)
    for hint in (1, 0):  # the tile whole, and split
        out = s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=hint))
        check_attend(Prefix(s, bad, before), None, qn[:before], out[:before])
        assert torch.isnan(out[before:]).all()


@pytest.mark.parametrize("what", ["page", "nan", "inf"])
@pytest.mark.parametrize("D,G,dt,new", [(64, 4, "f16", 400), (64, 2, "bf16", 400), (128, 4, "f16", 400), (128, 1, "bf16", 700), (256, 2, "bf16", 400)])
def test_many_rows_before_a_block_that_is_not_finite(D, G, dt, new, what):
    """The same where rows are many; the row before the first that sees it shares its column tile."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend many rows not finite {D} {G} {dt} {what}")
    n, bad = 4000, 3850 if what != "page" else 3856
    s = Setup(160 + D, D, 1, 16, [n], [new])
    set_scales(s, 0, bad - 1, 256)
    table = s.table.copy()
    if what == "page":
        table[0, bad // 16] = len(s.cache.pages)
    else:
        set_scales(s, 0, bad, {"nan": np.nan, "inf": np.inf}[what])
    s.kv.pages.copy_(dev(s.all))
    q, qn = s.rows(G, dt)
    before = bad - (n - new)
    for hint in (1, 0):
        out = s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=hint))
        check_attend(Prefix(s, bad, before), None, qn[:before], out[:before])
        assert torch.isnan(out[before:]).all()


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 90, 1]])
def test_rows_beside_bad_pages_are_as_exact_as_ever(news):
    """A page outside the pool in one of three sequences: the rows that do not see it, and the other sequences."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend beside bad pages {news}")
    s = Setup(14, 128, 2, 16, [100, 100, 100], news)
    q, qn = s.rows(8, "f16")
    q[0, 3] = float("nan")
    for page in (len(s.cache.pages), -1):
        table = s.table.copy()
        table[1, 3] = page  # tokens 48..63 of sequence 1
        out = s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=100))
        assert torch.isnan(out[0, 3]).all() and torch.isfinite(out[0, :3]).all() and torch.isfinite(out[0, 4:]).all()
        qn[0, 3] = 0  # a query of zeros weighs all values alike: key head 0's mean takes the place of the NaN row
        out[0, 3] = dev(s.cache.rows(s.table[0], 100)[1].mean(axis=1)[0], torch.float16)
        check_attend(s, q, qn, out, bad=(1,))
        before = max(0, 48 - (100 - news[1]))
        if before:
            at = s.cu[1]
            p = Prefix(s, 48, before)
            p.table = s.table[1:]
            check_attend(p, None, qn[at:at + before], out[at:at + before])


# ---------------------------------------------------------------- fewer rows than the batch counts
@pytest.mark.parametrize("T", [1, 7, 30, 44])
def test_rows_that_are_not_there(T):
    """Row tensors that end before cu[n_seqs] does: the rows they hold are those rows, at their own positions."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"fewer rows than the batch {T}")
    lens, news = [60, 45, 9], [5, 40, 4]
    s = Setup(71, 64, 2, 16, lens, news)
    pos = np.concatenate([np.arange(n - new, n) for n, new in zip(lens, news)])[:T]
    seq = np.repeat(np.arange(3), news)[:T]
    k, v = s.kv.read(0, s.batch, T)
    for got, at in ((k, 0), (v, 1)):
        ref = np.stack([s.cache.rows(s.table[i], p + 1)[at][:, p] for i, p in zip(seq, pos)])
        assert np.array_equal(got.cpu().numpy(), ref.astype(np.float16))
    (q, qh), (k, kh), (v, vh) = s.rows(4, "f32"), s.rows(2, "f32"), s.rows(2, "f32")
    ang = s.rng.uniform(0, 9, (60, 32))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    out = s.kv.append(0, q[:T], k[:T], v[:T], s.batch, dev(cos), dev(sin))
    rq, rk = (A.rotate(x[:T], cos[pos][:, None], sin[pos][:, None]) for x in (qh, kh))
    assert torch.equal(out, dev(rq))
    for t, (i, p) in enumerate(zip(seq, pos)):
        for h in range(2):
            s.cache.put(s.table[i, p // 16], h, p % 16, rk[t, h], vh[t, h])
    assert np.array_equal(s.kv.pages.cpu().numpy()[0], s.cache.pages)


@pytest.mark.parametrize("news,T,G,dt", [([3, 40, 2], 20, 2, "f16"), ([300, 700], 900, 1, "bf16"), ([300, 700], 200, 4, "f16"),
                                         ([1] * 9 + [600], 300, 2, "bf16")])
def test_attention_of_rows_that_are_not_there(news, T, G, dt):
    gpu_note(f"attend fewer rows {news} {T}")
    lens = [n + 50 for n in news]
    s = Setup(72, 64, 1, 16, lens, news)
    q, qn = s.rows(G, dt)
    out = s.kv.attend(0, q[:T], s.batch)
    assert len(out) == T
    for i, (n, new) in enumerate(zip(lens, news)):
        there = min(max(T - int(s.cu[i]), 0), new)
        if there:
            p = Prefix(s, n - new + there, there)
            p.table = s.table[i:]
            at = s.cu[i]
            check_attend(p, None, qn[at:at + there], out[at:at + there])


# ---------------------------------------------------------------- scores of any size
def check_weights(s, qn, out, ref_of):
    """out against sums of values whose weights are known: off by the weights' and values' roundings alone."""
    half, u = torch.finfo(out.dtype).eps / 2, 2.0 ** -11
    got = out.double().cpu().numpy()
    v, step = s.cache.rows(s.table[0], s.lens[0])[1], s.cache.rows(s.table[0], s.lens[0], steps=True)[1]
    G = got.shape[1] // s.n_kv
    for i in range(s.news[0]):
        w = ref_of(i)  # [tokens]
        for h in range(got.shape[1]):
            ref, size, vstep = w @ v[h // G], w @ np.abs(v[h // G]), w @ np.abs(step[h // G])
            tol = size * (2.0 ** -16 + 2 * u) + 2.0 ** -10 * vstep + half * np.abs(ref) * (1 + 1e-3) + 2.0 ** -24
            assert (np.abs(got[i, h] - ref) <= tol).all(), (i, h, got[i, h][:4], ref[:4])


# of the query (times the key) and of the keys, and the scale; in the last three the one or the other of their factors passes fp32's range on the way
LARGE = [(1.0, 1.0, 0.1), (1.0, 1.0, 1e3), (1.0, 1.0, 3e5), (1.0, 1.0, 1e6), (1.0, 1.0, 1e7), (1.0, 1.0, 1e8), (1.0, 1.0, 1e12),
         (1.0, 1.0, 1e30), (1e20, 1.0, 0.1), (1e34, 1.0, 0.1), (1e40, 1e-3, 0.1), (1e-36, 1.0, 3e38), (1e40, 1e-3, 1e-3)]


@pytest.mark.parametrize("D,G,news", [(128, 4, 1), (128, 4, 3), (64, 2, 300), (256, 2, 2), (128, 2, 200), (256, 1, 200)])
@pytest.mark.parametrize("size,small,scale", LARGE)
def test_a_key_that_outweighs_all_others(D, G, news, size, small, scale):
    """Queries along one token's key: its value is the result, however large the scores are."""
    gpu_note(f"attend large scores {D} {G} {news} {size} {small} {scale}")
    s = Setup(81, D, 1, 16, [600], [news])
    winner = 200
    s.cache.pages[..., 16 * D:17 * D].view(np.float16)[...] *= np.float16(small)
    s.cache.pages[s.table[0, winner // 16], :, 0].view(np.uint16)[:, s.cache._places(winner % 16)[4]] = np.float16(small).view(np.uint16)
    s.kv.pages.copy_(dev(s.all))
    k = s.cache.rows(s.table[0], 600)[0][0]  # the other keys' steps are 0.15 of the winner's
    q = dev(np.broadcast_to(k[winner] * size, (news, G, D)).astype(np.float32), torch.bfloat16)
    score = q[0, 0].double().cpu().numpy() @ k.T * scale
    assert score.argmax() == winner and np.sort(score)[-2] < 0.5 * score.max() < 1e38
    if score.max() < 100:
        return check_attend(s, q, q.float().cpu().numpy(), s.kv.attend(0, q, s.batch, scale=scale), scale=scale)
    one = np.zeros(600)
    one[winner] = 1
    for b in (s.batch, type(s.batch)(s.batch.cu, s.batch.kv_len, s.batch.table, max_len=1)):
        check_weights(s, None, s.kv.attend(0, q, b, scale=scale), lambda i: one)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D,G,news", [(128, 4, 1), (64, 2, 3), (256, 2, 2), (128, 2, 200)])
@pytest.mark.parametrize("scale", [0.1, 3e5, 1e7, 1e9, 1e12, 1e30])
def test_equal_scores_of_any_size(D, G, news, scale, sign):
    """The same key in every place: all values weigh alike, whatever the score and however the values' sizes differ."""
    gpu_note(f"attend equal scores {D} {G} {news} {scale} {sign}")
    s = Setup(82, D, 1, 16, [500], [news])
    pages, rng = s.cache.pages.view(np.uint16), np.random.default_rng(5)
    code, step = rng.integers(0, 16, D), np.float16(rng.uniform(0.1, 0.2, D // 32))
    for r in range(16):
        ka, kn, _, _, ks, _ = s.cache._places(r)
        half = np.zeros(pages.shape[-1], np.int64)
        np.add.at(half, ka, code << (4 * kn))
        pages[..., ka] = half[ka].astype(np.uint16)
        pages[..., ks] = step.view(np.uint16)
    for t in range(0, 500):
        set_scales(s, 0, t, [1.0, 30.0, 0.01, 900.0][t // 32 % 4])  # each of a block's waves its own size
    s.kv.pages.copy_(dev(s.all))
    k = s.cache.rows(s.table[0], 500)[0][0]
    assert (k == k[0]).all()
    q = dev(np.broadcast_to(k[0] * sign, (news, G, D)).astype(np.float32), torch.bfloat16)
    def weights(i):
        n = 500 - news + i + 1
        return np.where(np.arange(500) < n, 1 / n, 0)
    for b in (s.batch, type(s.batch)(s.batch.cu, s.batch.kv_len, s.batch.table, max_len=1)):
        check_weights(s, None, s.kv.attend(0, q, b, scale=scale), weights)


# ---------------------------------------------------------------- gradients
def test_parameters_without_gradients():
    """Tensors that require gradients are operands as any where torch does not record them, and refused where it does."""
    from tinygiant_amd.linear import matmul_i8
    gpu_note("parameters")
    s = Setup(91, 64, 2, 16, [30], [3])
    q, qn = s.rows(4, "f16")
    k, v = s.rows(2, "f16")[0], s.rows(2, "f16")[0]
    norm = torch.ones(64, device="cuda")
    w, ws, x = torch.ones(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"), torch.ones(3, 64, device="cuda")
    plain = s.kv.append(0, q, k, v, s.batch, q_norm=norm), s.kv.attend(0, q, s.batch), matmul_i8(x, w, ws, norm=norm)
    p, xp, qp = torch.nn.Parameter(norm), torch.nn.Parameter(x), q.clone().requires_grad_()
    for call in (lambda: s.kv.append(0, q, k, v, s.batch, q_norm=p), lambda: s.kv.attend(0, qp, s.batch),
                 lambda: matmul_i8(xp, w, ws), lambda: matmul_i8(x, w, ws, norm=p)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            got = s.kv.append(0, qp, k, v, s.batch, q_norm=p), s.kv.attend(0, qp, s.batch), matmul_i8(xp, w, ws, norm=p)
        assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(plain, got))


# ---------------------------------------------------------------- one row, hints
def test_one_row_of_a_tensor_of_odd_width():
    """Aligned rows whose stride is no multiple of what a kernel loads at a time: with one of them it is not used."""
    gpu_note("one row")
    s = Setup(95, 64, 1, 16, [20], [1])
    buf = torch.zeros(1, 64 * 4 + 3, device="cuda", dtype=torch.float16)
    x, xn = s.rows(4, "f16")
    buf[:, :256] = x.view(1, 256)
    q, k, v = buf[:, :128], buf[:, 128:192], buf[:, 192:256]
    out = torch.full((1, 131), 3.0, device="cuda", dtype=torch.float16)
    got = s.kv.append(0, q, k, v, s.batch, out=out[:, :128])
    assert torch.equal(got, q) and (out[:, 128:] == 3).all()
    s.cache.put(s.table[0, 1], 0, 3, xn[0, 2], xn[0, 3])
    assert np.array_equal(s.kv.pages.cpu().numpy()[0], s.cache.pages)
    s.kv.attend(0, q, s.batch, out=out[:, :128])
    check_attend(s, q, xn[:, :2], out[:, :128].view(1, 2, 64))
    assert (out[:, 128:] == 3).all()


@pytest.mark.parametrize("hint", [(1 << 31) - 1, 1 << 31, (1 << 32) + 1, 10 ** 15])
def test_hints_beyond_32_bits(hint):
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend hint {hint}")
    s = Setup(96, 128, 1, 16, [300, 20], [1, 2])
    q, qn = s.rows(4, "bf16")
    whole = s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, s.batch.table))  # 0: what the table holds
    assert torch.equal(s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, s.batch.table, max_len=hint)), whole)
    check_attend(s, q, qn, whole)


@pytest.mark.parametrize("D,G,lens,news,dt", [(128, 8, [2005], [1], "bf16"), (64, 4, [3000, 70], [300, 70], "f16"),
                                              (256, 2, [2500, 700, 3], [200, 1, 3], "bf16"), (128, 4, [900] * 70, [1] * 70, "f16")])
def test_the_same_call_gives_the_same_bits(D, G, lens, news, dt):
    """Splits are joined in an order of their own: no result depends on which block was first."""
    gpu_note(f"attend twice {D} {G} {dt}")
    s = Setup(97, D, 2, 16, lens, news)
    q, _ = s.rows(2 * G, dt)
    first = s.kv.attend(0, q, s.batch)
    for _ in range(5):
        assert torch.equal(s.kv.attend(0, q, s.batch), first)
