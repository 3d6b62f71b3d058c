"""The paged Q4_0 cache and the attention over it on the GPU, against
oracle/attn.py.

The cache's bytes and the rotated q are compared exactly: both sides round
each step alike.  Attention's tolerance counts the kernels' roundings, u = 2^-11 being half a
step of fp16 (weights and values are fp16 operands of the matrix
instructions; keys and queries too where rows are many):
  scores   off by at most 2 u S (S: the largest scale * sum |q_i k_i| of the
           row), 2^-18 (S + 1) of fp32 sums and exponents, and, where the codes are
           operands themselves, 2^-11 of the largest query value times one step of
           each block: the instruction aligns 32 products to the largest one,
           a subnormal operand (code 2^-18) counting as 2^-14, and cuts 2^-24 below
           it, so 32 * 2^-38 * 16 / 2^-18 steps are lost (16 lies between the two
           kinds of codes).  A weight is off by the factor e^(2 delta).
  weights  u as a half; values u as a half; and again 2 * 32 * 2^-38 / 2^-22 = 2^-10 of one
           step of each value block where the codes are operands (the codes' sum
           and its offset's).
These move the output by at most that times sum p |v| (p times one step); the
result is then rounded by half a step of its type."""
import zlib

import numpy as np
import pytest
import torch

from oracle import attn as A
from tests.conftest import gpu_note

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True, scope="module")
def _lib(tglib):
    yield


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Setup:
    """A random cache of n_kv heads and a batch over shuffled pages: lens and
    news per sequence, `pad` rows behind the last sequence."""

    def __init__(self, seed, D, n_kv, page, lens, news, pad=0, spare=2, layers=1, layer=0):
        from tinygiant_amd.attn import KVBatch, PagedKV
        self.rng = rng = np.random.default_rng(seed)
        self.D, self.n_kv, self.page, self.lens, self.news, self.layer = D, n_kv, page, lens, news, layer
        need = [-(-n // page) for n in lens]
        pool = rng.permutation(sum(need) + spare)
        cols = max(need + [1])
        table = np.full((len(lens), cols), -7, np.int32)  # what no sequence uses is no page
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = pool[at:at + n]
            at += n
        self.table, self.cu = table, np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.T = int(self.cu[-1]) + pad
        raw = rng.integers(0, 256, (layers, len(pool), n_kv, page // 16, 18 * D), dtype=np.uint8)
        scales = (0.15 * rng.standard_normal((layers, len(pool), n_kv, page // 16, D))).astype(np.float16)
        raw[..., 16 * D:] = scales.view(np.uint8)
        self.cache = A.Cache(len(pool), page, n_kv, D, raw[layer])
        self.all = raw
        self.kv = PagedKV(layers, len(pool), page, n_kv, D, pages=dev(raw))
        self.batch = KVBatch(dev(self.cu), dev(np.array(lens, np.int32)), dev(table), max_len=max(lens))

    def rows(self, heads, dtype, scale=1.0):
        x = dev((scale * self.rng.standard_normal((self.T, heads, self.D))).astype(np.float32), DT[dtype])
        return x, x.float().cpu().numpy()


def check_attend(s, q, qn, out, scale=None, bad=()):
    """out against the oracle, sequence by sequence; rows of `bad` sequences are left to the caller."""
    got = out.float().cpu().numpy().astype(np.float64)
    half = torch.finfo(out.dtype).eps / 2
    u = 2.0 ** -11
    for i, (n, new) in enumerate(zip(s.lens, s.news)):
        if i in bad or not new:
            continue
        k, v = s.cache.rows(s.table[i], n)
        rows = slice(s.cu[i], s.cu[i + 1])
        ref, size, top, vstep, kstep = A.attend(qn[rows], k, v, new, s.D ** -0.5 if scale is None else scale,
                                                steps=s.cache.rows(s.table[i], n, steps=True))
        delta = 2 * u * top + 2.0 ** -18 * (top + 1) + 2.0 ** -11 * kstep
        tol = size * (np.expm1(2 * delta) + 2 * u) + 2.0 ** -10 * vstep + half * np.abs(ref) * (1 + 1e-3) + 2.0 ** -24
        off = np.abs(got[rows] - ref)
        at = np.unravel_index((off / tol).argmax(), off.shape)
        assert off[at] <= tol[at], (i, n, new, at, got[rows][at], ref[at], size[at], top[at[0], at[1]], float(off[at] / tol[at]))
        # and on the whole far inside it where scores are ordinary (up to S = 64 their fp32 sums are off by at most
        # 2^-18 S = u / 2): independent roundings, not a bias
        if ref.size > 2000 and top.max() <= 64:
            err, norm = np.linalg.norm(got[rows] - ref), np.linalg.norm(ref)
            assert err <= (2 * half + 8 * u) * norm, (i, err, norm)


# (D, n_kv, group, page, lens, news, type)
ATTEND = [
    (128, 4, 8, 16, [1], [1], "bf16"),                            # one token that sees itself
    (128, 4, 8, 16, [15, 16, 17, 31, 32, 33, 47, 48, 49], [1] * 9, "f16"),  # around tile and step ends
    (128, 4, 16, 64, [700, 1, 64, 65, 0, 333], [1, 1, 1, 1, 1, 1], "bf16"),  # a sequence of no token: zero
    (64, 2, 1, 32, [129, 40], [1, 1], "f16"),                      # one query head per key head
    (256, 1, 5, 16, [257, 130, 3], [1, 1, 1], "f16"),
    (256, 2, 16, 48, [500], [1], "bf16"),
    (64, 8, 4, 16, [100, 5, 999], [3, 5, 1], "bf16"),              # a few rows each
    (128, 1, 24, 128, [300, 77], [2, 1], "f16"),                   # more heads than a tile has columns
    (128, 2, 3, 16, [50, 9, 0, 20], [7, 0, 0, 20], "f16"),         # sequences without rows between others
    (128, 4, 8, 64, [190], [190], "bf16"),                         # a prompt
    (128, 2, 8, 16, [300, 17, 128], [300, 17, 100], "f16"),        # prompts and a chunk
    (64, 2, 4, 32, [1000], [257], "f16"),                          # a chunk of a longer prompt
    (64, 1, 1, 16, [400], [400], "bf16"),
    (256, 1, 2, 64, [333, 64], [200, 64], "bf16"),
    (128, 2, 1, 16, [10, 4], [30, 20], "f16"),                     # more rows than tokens: the first see nothing
    (128, 1, 7, 16, [1], [300], "bf16"),
    (64, 8, 2, 16, [5 + i % 37 for i in range(80)] + [3000, 1700], [1] * 82, "f16"),  # more tiles than shares, two long ones
    (64, 1, 3, 32, [900 + 13 * i for i in range(10)], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10], "bf16"),
    (128, 2, 8, 16, [3000, 40], [64, 40], "bf16"),                                    # many columns, split over the tokens
    (256, 2, 4, 32, [2000, 700, 3], [90, 1, 3], "f16"),
    (64, 4, 4, 64, [5000], [33], "bf16"),
    (256, 2, 4, 32, [2500, 700, 3], [200, 90, 3], "bf16"),                            # heads of 256: two waves to a column
    (256, 1, 7, 16, [310, 77], [310, 77], "bf16"),
    (128, 2, 8, 32, [900, 700, 33, 0, 1500, 64, 5, 6, 7, 8], [600, 1, 33, 0, 1, 2, 1, 1, 1, 1], "bf16"),  # chunks and single tokens: two launches
    (64, 1, 4, 16, [2600, 1, 40, 3000] + [20 + i for i in range(70)], [2600, 1, 7, 900] + [1] * 70, "f16"),
    (256, 1, 4, 16, [600, 500, 7] + [31] * 7, [500, 3, 1] + [1] * 7, "bf16"),
    (256, 2, 4, 32, [2500, 700, 3], [250, 90, 3], "f16"),
    (256, 1, 7, 16, [310, 77, 20], [310, 77, 20], "f16"),
    (256, 1, 16, 48, [33], [33], "f16"),
    (128, 1, 16, 48, [777, 1300], [100, 300], "f16"),
    (64, 1, 16, 16, [8 + i % 30 for i in range(64)] + [3000, 2500], [8] * 66, "bf16"),     # wide column tiles of more sequences than lanes
    (128, 1, 16, 32, [40 + i for i in range(70)] + [4000], [16] * 71, "f16"),
    (128, 1, 4, 16, [i % 5 * 100 for i in range(130)], [1] * 130, "f16"),             # more sequences than lanes, some empty
    (64, 1, 8, 16, [0], [40], "f16"),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend(case):
    D, n_kv, G, page, lens, news, dt = case
    gpu_note(f"attend {case}")
    s = Setup(zlib.crc32(str(case).encode()) % 1000, D, n_kv, page, lens, news)
    q, qn = s.rows(n_kv * G, dt)
    check_attend(s, q, qn, s.kv.attend(0, q, s.batch))


@pytest.mark.parametrize("n,news", [(70001, 1), (33000, 3), (20000, 100)])
def test_attend_long(n, news):
    gpu_note(f"attend long {n} {news}")
    s = Setup(n, 128, 1, 64, [n, 5], [news, 1])
    q, qn = s.rows(16, "f16")
    check_attend(s, q, qn, s.kv.attend(0, q, s.batch))


@pytest.mark.parametrize("D", [64, 128])
def test_many_fp16_columns_are_as_exact_as_few(D):
    """Keys and values are taken whole on either way and each weight is rounded to fp16 once.  With values of mean 0 that
    are independent of the weights, |out|^2 is sum p^2 |v|^2 on the mean and the weights' roundings e move out by sum e^2 p^2
    |v|^2: as much, relatively, as rounding out to fp16 does (weights and results both spread over their
    binades), so together sqrt(2) = 1.41 of the latter, 1.5 with room for how they spread.  Rounded keys
    and values would add 0.8 and 0.6 squared: 1.8 and more."""
    gpu_note(f"attend fp16 many and few {D}")
    s = Setup(40 + D, D, 1, 32, [900], [300])
    q, qn = s.rows(2, "f16")
    many = s.kv.attend(0, q, s.batch)  # 600 columns ...
    one = [s.kv.attend(0, q[i:i + 1], type(s.batch)(dev(np.array([0, 1], np.int32)), dev(np.array([600 + i + 1], np.int32)),
                                                    s.batch.table)) for i in range(300)]  # ... and 2
    many, few = many.double().cpu().numpy(), torch.cat(one).double().cpu().numpy()
    k, v = s.cache.rows(s.table[0], 900)
    ref = A.attend(qn, k, v, 300, D ** -0.5)[0]
    rounding = np.linalg.norm(ref.astype(np.float16).astype(np.float64) - ref)
    off = [np.linalg.norm(x - ref) / rounding for x in (many, few)]
    assert max(off) <= 1.5, off


@pytest.mark.parametrize("hint", [1, 16, 100, 10 ** 9])
def test_attend_any_hint(hint):
    """max_len is a hint: too small or too large changes nothing but the split."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend hint {hint}")
    s = Setup(11, 128, 2, 16, [1500, 3, 400], [1, 1, 2])
    q, qn = s.rows(16, "bf16")
    b = KVBatch(s.batch.cu, s.batch.kv_len, s.batch.table, max_len=hint)
    check_attend(s, q, qn, s.kv.attend(0, q, b))


def test_attend_scores_far_apart():
    """A first token that outweighs the rest by far, scores beyond what
    exponents hold, and values of very different size."""
    gpu_note("attend far scores")
    s = Setup(12, 128, 1, 16, [600, 600], [1, 50])
    sc = s.cache.pages[..., 16 * 128:].view(np.float16)
    for p, f in ((s.table[0, 0], 8.0), (s.table[0, 5], 1e-5), (s.table[0, 7], 0.0), (s.table[1, 1], 30.0)):
        sc[p] *= np.float16(f)
    s.kv.pages.copy_(dev(s.all))
    for scale, size in ((128 ** -0.5, 1.0), (4.0, 1.0), (128 ** -0.5, 300.0), (1e-4, 1e-3)):
        q, qn = s.rows(8, "f16", size)
        check_attend(s, q, qn, s.kv.attend(0, q, s.batch, scale=scale), scale=scale)


def test_attend_q_of_any_size():
    """bf16 queries beyond fp16's range, and tiny ones."""
    gpu_note("attend q sizes")
    s = Setup(13, 128, 2, 16, [80, 200], [1, 40])
    for size in (1e6, 1e-8, 1e-30):
        q, qn = s.rows(4, "bf16", size)
        check_attend(s, q, qn, s.kv.attend(0, q, s.batch, scale=0.1 / size), scale=0.1 / size)
    q, qn = s.rows(4, "bf16", 0.0)
    check_attend(s, q, qn, s.kv.attend(0, q, s.batch))


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 90, 1]])
def test_attend_nan_and_bad_pages_stay_in_their_rows(news):
    """A page outside the pool, and positions beyond the table, make NaN of
    the rows that see them; a NaN query of its own head; nothing else."""
    from tinygiant_amd.attn import KVBatch
    gpu_note(f"attend bad pages {news}")
    s = Setup(14, 128, 2, 16, [100, 100, 100], news)
    table = s.table.copy()
    table[1, 3] = len(s.cache.pages)            # tokens 48..63 of sequence 1
    b = KVBatch(s.batch.cu, s.batch.kv_len, dev(table), max_len=100)
    q, qn = s.rows(8, "f16")
    q[0, 3] = float("nan")
    out = s.kv.attend(0, q, b)
    got = out.float().cpu().numpy()
    assert np.isnan(got[0, 3]).all()
    got[0, 3], qn[0, 3] = 0, 0
    first = 100 - news[1]                        # position of sequence 1's first row
    sees = np.arange(first, 100) >= 48
    one = got[s.cu[1]:s.cu[2]]
    assert np.isnan(one[sees]).all() and np.isfinite(one[~sees]).all()
    for i in (0, 2):
        assert np.isfinite(got[s.cu[i]:s.cu[i + 1]]).all()
    table[1, 3] = -1
    assert np.isnan(s.kv.attend(0, q, KVBatch(s.batch.cu, s.batch.kv_len, dev(table))).float().cpu().numpy()[s.cu[1]:s.cu[2]][sees]).all()
    # a length beyond the table
    lens = dev(np.array([100, 16 * s.table.shape[1] + 1, 100], np.int32))
    got = s.kv.attend(0, q, KVBatch(s.batch.cu, lens, s.batch.table)).float().cpu().numpy()
    assert np.isnan(got[s.cu[2] - 1]).all() and np.isfinite(got[s.cu[2]:]).all()


def test_attend_strides_padding_layers_and_out():
    """Rows of a wider tensor, rows behind the last sequence left as they
    were, a layer of several, an out of the caller's with its own stride."""
    gpu_note("attend strides")
    for news in ([1, 1], [30, 2], [100, 60]):
        s = Setup(15, 128, 2, 32, [120, 61], news, pad=3, layers=3, layer=1)
        wide = torch.randn(s.T, 8 + 5, 128, device="cuda").to(torch.bfloat16)
        q = wide[:, 2:10]
        out = torch.full((s.T, 11, 128), 7.0, device="cuda", dtype=torch.bfloat16)
        s.kv.attend(1, q, s.batch, out=out[:, 1:9])
        check_attend(s, q, q.float().cpu().numpy(), out[:, 1:9])
        assert (out[:, 0] == 7).all() and (out[:, 9:] == 7).all() and (out[s.cu[-1]:] == 7).all()


def test_sequences_share_pages():
    """A prefix in common."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("attend shared pages")
    s = Setup(16, 64, 2, 16, [90, 70], [1, 20])
    s.table[1, :3] = s.table[0, :3]
    s.batch = KVBatch(s.batch.cu, s.batch.kv_len, dev(s.table), max_len=90)
    q, qn = s.rows(4, "f16")
    check_attend(s, q, qn, s.kv.attend(0, q, s.batch))


def test_offsets_beyond_32_bits():
    """Pages more than 4 GiB into the pool: appended to, read and attended."""
    from tinygiant_amd.attn import KVBatch, PagedKV
    n_pages, D = 2_000_000, 128
    gpu_note("pages beyond 4 GiB")
    kv = PagedKV(1, n_pages, 16, 1, D)
    table = np.array([[n_pages - 1, 3, n_pages - 2]], np.int32)
    cu, ln = dev(np.array([0, 40], np.int32)), dev(np.array([40], np.int32))
    b = KVBatch(cu, ln, dev(table))
    rng = np.random.default_rng(3)
    x = rng.standard_normal((40, 10, D)).astype(np.float32)
    t = dev(x)
    kv.append(0, None, t[:, 8:9], t[:, 9:], b)
    k, v = kv.read(0, b, 40)
    q16 = t[:, :8].half()
    for news in (40, 1):
        b2 = KVBatch(dev(np.array([0, news], np.int32)), ln, b.table)
        out = kv.attend(0, q16[40 - news:], b2).float().cpu().numpy()
        kk, vv = (z.cpu().numpy().astype(np.float64).transpose(1, 0, 2) for z in (k, v))
        ref, _, _ = A.attend(q16[40 - news:].float().cpu().numpy(), kk, vv, news, D ** -0.5)
        assert np.abs(out - ref).max() < 0.01
    code, d = A.q4_0(x[:, 8])
    want = ((code.astype(float) - 8) * np.repeat(d.astype(float), 32, axis=1)).astype(np.float16)
    assert np.array_equal(k[:, 0].cpu().numpy(), want)
    del kv
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- append and read
APPEND = [
    (128, 4, 8, 16, [1000], [1], "bf16", True, True),
    (128, 2, 16, 64, [64, 65, 1, 300], [1, 1, 1, 1], "f16", True, True),
    (64, 8, 4, 32, [40, 33], [40, 17], "f32", False, True),
    (64, 1, 1, 16, [19], [19], "bf16", True, False),
    (256, 1, 3, 16, [50, 7], [33, 7], "f16", True, True),
    (256, 3, 2, 48, [100], [20], "f32", True, True),
    (128, 1, 1, 16, [70] * 70, [1] * 70, "bf16", True, True),   # more sequences than lanes
    (128, 5, 7, 128, [200, 0, 130], [200, 0, 3], "f32", True, True),
]


def plain_append(s, q, k, v, cos, sin, qn, kn, eps=1e-6):
    """The rotated q [T, heads, D] float32, and k, v as the cache is given them."""
    pos = np.concatenate([np.arange(n - new, n) for n, new in zip(s.lens, s.news)] + [np.zeros(0)]).astype(int)
    q, k = A.norm_rows(q[:len(pos)], qn, eps), A.norm_rows(k[:len(pos)], kn, eps)
    if cos is not None:
        q, k = (A.rotate(x, cos[pos][:, None], sin[pos][:, None]) for x in (q, k))
    return q, k, v[:len(pos)]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("fused", [False, True])
def test_append_and_read(case, fused):
    D, n_kv, G, page, lens, news, dt, norm, rope = case
    gpu_note(f"append {case} {fused}")
    s = Setup(zlib.crc32(str(case).encode()) % 1000, D, n_kv, page, lens, news, pad=2, layers=2, layer=1)
    heads = n_kv * G
    if fused:  # views of one projection's rows
        x, xn = s.rows(heads + 2 * n_kv, dt)
        q, k, v = x.split([heads, n_kv, n_kv], 1)
        qh, kh, vh = np.split(xn, [heads, heads + n_kv], 1)
    else:
        (q, qh), (k, kh), (v, vh) = s.rows(heads, dt), s.rows(n_kv, dt), s.rows(n_kv, dt, 3.0)
    ang = s.rng.uniform(0, 1e3, (max(lens), D // 2))
    cos, sin = (np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)) if rope else (None, None)
    qn, kn = (s.rng.uniform(0.5, 1.5, (2, D)).astype(np.float32)) if norm else (None, None)
    d = lambda a: None if a is None else dev(a)
    before = s.kv.pages.clone()
    out = torch.full((s.T, heads, D), 5.0, dtype=DT[dt], device="cuda")
    s.kv.append(1, q, k, v, s.batch, d(cos), d(sin), q_norm=d(qn), k_norm=d(kn), out=out)
    rq, rk, rv = plain_append(s, qh, kh, vh, cos, sin, qn, kn)
    n = len(rq)
    assert torch.equal(out[:n], dev(rq).to(DT[dt])), "rotated q"
    assert (out[n:] == 5).all(), "padding rows"
    t = 0
    for i, (ln, new) in enumerate(zip(lens, news)):
        for p in range(ln - new, ln):
            for h in range(n_kv):
                s.cache.put(s.table[i, p // page], h, p % page, rk[t, h], rv[t, h])
            t += 1
    got = s.kv.pages.cpu().numpy()
    assert np.array_equal(got[1], s.cache.pages), f"{(got[1] != s.cache.pages).sum()} bytes differ"
    assert torch.equal(s.kv.pages[0], before[0]), "another layer"
    kk, vv = s.kv.read(1, s.batch, n)
    for x, y in ((kk, rk), (vv, rv)):
        code, sc = A.q4_0(y)
        assert np.array_equal(x.cpu().numpy(), ((code.astype(np.float32) - 8) * np.repeat(sc.astype(np.float32), 32, axis=-1)).astype(np.float16))
    # q in place
    s.kv.append(1, q, k, v, s.batch, d(cos), d(sin), q_norm=d(qn), k_norm=d(kn), out=q)
    assert torch.equal(q[:n], out[:n])


def test_append_values_at_the_edges():
    """Zeros, ties, infinities, NaN, subnormals and values beyond fp16, byte for byte; k and v alone."""
    gpu_note("append edges")
    s = Setup(21, 64, 1, 16, [20], [20])
    x = s.rng.standard_normal((20, 64)).astype(np.float32)
    x[0] = 0
    x[1, :32], x[1, 32:] = np.tile([1, -1], 16), np.tile([-2, 2], 16)
    x[2, 5], x[3, 40], x[4, 9], x[5, 33] = np.inf, -np.inf, np.nan, 1e30
    x[6], x[7], x[8, :32] = 1e-41 * np.arange(64), 3e-6, 65504
    x[9] = np.where(np.arange(64) % 2, 8, 7.5)
    k = dev(x[:, None])
    v = dev(x[::-1, None])
    assert s.kv.append(0, None, k, v, s.batch) is None
    for t in range(20):
        s.cache.put(s.table[0, t // 16], 0, t % 16, x[t], x[19 - t])
    got = s.kv.pages.cpu().numpy()[0]
    ref = s.cache.pages
    sc = slice(16 * 64, None)  # a NaN has many bit patterns
    a, b = got[..., sc].view(np.float16), ref[..., sc].view(np.float16)
    assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])
    kk, vv = s.kv.read(0, s.batch, 20)
    assert torch.isnan(kk[4, 0, :32]).all() and torch.isfinite(kk[4, 0, 32:]).all()
    kr, vr = s.cache.rows(s.table[0], 20)
    for z, r in ((kk, kr), (vv, vr)):
        assert np.array_equal(z[:, 0].cpu().numpy(), r[0].astype(np.float16), equal_nan=True)


def test_append_refused_positions():
    """Tokens outside the table, the pool or the rotation table: not
    written, their q rows NaN; the others as ever."""
    from tinygiant_amd.attn import KVBatch
    gpu_note("append refused positions")
    s = Setup(22, 128, 2, 16, [40, 40, 3, 40], [6, 6, 6, 6])
    table = s.table.copy()
    table[0, 2] = -1                   # tokens 32.. of sequence 0: rows 0..5 (34..39)
    lens = np.array([40, 16 * table.shape[1] + 2, 3, 40], np.int32)  # two rows past the table; three below 0
    b = KVBatch(s.batch.cu, dev(lens), dev(table))
    (q, qh), (k, kh), (v, vh) = s.rows(4, "f32"), s.rows(2, "f32"), s.rows(2, "f32")
    ang = s.rng.uniform(0, 9, (38, 64))   # positions 38 and 39 of sequence 3 have no row, nor sequence 1's
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    before = s.kv.pages.clone()
    out = s.kv.append(0, q, k, v, b, dev(cos), dev(sin))
    nan = torch.isnan(out).all(-1).all(-1).cpu().numpy()
    want = np.array([1] * 6 + [1] * 6 + [1, 1, 1, 0, 0, 0] + [0, 0, 0, 0, 1, 1], bool)
    assert np.array_equal(nan, want) and np.isfinite(out[torch.from_numpy(~want).cuda()].cpu().numpy()).all()
    rk = A.rotate(kh[[15, 16, 17, 18, 19, 20, 21]], cos[[0, 1, 2, 34, 35, 36, 37]][:, None], sin[[0, 1, 2, 34, 35, 36, 37]][:, None])
    for j, (row, seq, p) in enumerate([(15, 2, 0), (16, 2, 1), (17, 2, 2), (18, 3, 34), (19, 3, 35), (20, 3, 36), (21, 3, 37)]):
        for h in range(2):
            s.cache.put(table[seq, p // 16], h, p % 16, rk[j, h], vh[row, h])
    assert np.array_equal(s.kv.pages.cpu().numpy()[0], s.cache.pages)
    assert not torch.equal(before, s.kv.pages)
    kk, _ = s.kv.read(0, b, 24)
    assert torch.isnan(kk[:6]).all() and torch.isnan(kk[10:15]).all() and torch.isfinite(kk[6:10]).all()


def test_empty_batches():
    from tinygiant_amd.attn import KVBatch
    s = Setup(31, 64, 2, 16, [20], [4])
    none = KVBatch(dev(np.zeros(1, np.int32)), dev(np.zeros(0, np.int32)), dev(np.zeros((0, 3), np.int32)))
    z = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16)
    before = s.kv.pages.clone()
    for b, x in ((none, z), (s.batch, z), (none, torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16))):
        assert s.kv.append(0, x, x, x, b).shape == x.shape
        assert s.kv.attend(0, x, b).shape == x.shape
        assert s.kv.read(0, b, len(x))[0].shape == x.shape
    assert torch.equal(before, s.kv.pages)
