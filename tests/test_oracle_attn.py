"""The attention block's oracle (oracle/attn.py) against the C oracle and
against itself restated another way.  No GPU."""
import numpy as np
import pytest

from oracle import attn as A


def test_q4_0_is_the_framework_s(O):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    x[3] = 0
    x[4, :32] = np.tile([1.0, -1.0], 16)  # ties of magnitude: the first decides
    x[5, 7] = -1e3
    code, d = A.q4_0(x)
    blocks = O.quantize_q4_0(x.reshape(-1)).reshape(-1, 18)
    assert np.array_equal(blocks[:, :2].copy().view(np.float16).reshape(50, 2), d)
    nib = np.concatenate([blocks[:, 2:] & 15, blocks[:, 2:] >> 4], axis=1).reshape(50, 64)
    assert np.array_equal(nib, code)


def test_q4_0_saturates_and_keeps_nan():
    x = np.zeros((4, 32), np.float32)
    x[0, 3], x[1, 3], x[2, 3], x[3, :] = np.inf, -1e30, np.nan, 1e-42
    code, d = A.q4_0(x)
    assert d[0, 0] == -8188 and code[0, 3] == 0 and (code[0, :3] == 8).all()
    assert d[1, 0] == 8188 and code[1, 3] == 0
    assert np.isnan(d[2, 0])
    assert d[3, 0] == 0


def test_rotation_is_the_reference_s(O):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 64)).astype(np.float32)
    ang = rng.uniform(0, 100, (5, 32))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    ref = x.copy()
    O.lib().tgo_rope(ref.ctypes.data, 3, 64, cos.ctypes.data, sin.ctypes.data, 4)
    # the reference fuses the second half's product and sum: one rounding less
    assert np.abs(A.rotate(x, cos[4], sin[4]) - ref).max() <= 2.0 ** -23 * np.abs(x).max()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_cache_round_trip_and_layout(D):
    rng = np.random.default_rng(D)
    c = A.Cache(3, 32, 2, D)
    k, v = rng.standard_normal((2, 2, 40, D)).astype(np.float32)
    table = [2, 0]
    for t in range(40):
        for h in range(2):
            c.put(table[t // 32], h, t % 32, k[h, t], v[h, t])
    kk, vv = c.rows(table, 40)
    for x, y in ((k, kk), (v, vv)):
        code, d = A.q4_0(x)
        assert np.array_equal(y, (code.astype(float) - 8) * np.repeat(d.astype(float), 32, axis=-1))
    k1, v1 = c.get(0, 1, 3)
    assert np.array_equal(k1, kk[1, 35]) and np.array_equal(v1, vv[1, 35])
    # every place of a tile is one value's: 16 tokens fill its 18 D bytes
    seen = np.zeros((9 * D, 4), int)
    for r in range(16):
        ka, kn, va, vn, ks, vs = c._places(r)
        np.add.at(seen, (ka, kn), 1)
        np.add.at(seen, (va, vn), 1)
        np.add.at(seen, (np.concatenate([ks, vs])[:, None], np.arange(4)), 1)
    assert (seen == 1).all()


def test_attend_against_the_c_oracle(O):
    """One token through tgo_attention_decode's softmax part: identity
    projections, unit norms and no rotation leave q, k and v as they are."""
    rng = np.random.default_rng(5)
    n, D = 9, 64
    k, v = rng.standard_normal((2, 1, n, D)).astype(np.float32)
    x = rng.standard_normal(D).astype(np.float32)
    x /= np.sqrt((x.astype(np.float64) ** 2).mean()).astype(np.float32)  # its norm leaves it (to 1e-6)
    kc, vc = np.zeros((2, 1, n + 1, D), np.float32)
    kc[:, :n], vc[:, :n] = k, v
    eye, one = np.eye(D, dtype=np.float32), np.ones(D, np.float32)
    cos, sin = np.ones((n + 1, D // 2), np.float32), np.zeros((n + 1, D // 2), np.float32)
    out = np.zeros(D, np.float32)
    p = lambda a: a.ctypes.data
    O.lib().tgo_attention_decode(p(eye), p(eye), p(eye), p(eye), p(one), p(one), p(kc), p(vc), n, n + 1, p(cos), p(sin),
                                 p(x), p(out), D, 1, 1, D, n)
    ref, _, _ = A.attend(x.reshape(1, 1, D), kc.astype(float), vc.astype(float), 1, D ** -0.5)
    assert np.abs(ref[0, 0] - out).max() < 1e-5


def test_attend_rows_that_see_nothing():
    q = np.ones((4, 2, 64), np.float32)
    k = v = np.ones((1, 2, 64))
    out, size, _ = A.attend(q, k, v, 4, 1.0)
    assert (out[:2] == 0).all() and np.allclose(out[2:], 1) and (size[:2] == 0).all()
    out, _, _ = A.attend(q, k[:, :0], v[:, :0], 4, 1.0)
    assert (out == 0).all()


def test_matmul_i8_codes():
    x = np.array([[1.0, 0.5, -0.5, 0.25], [0, 0, 0, 0]], np.float32)
    q, s = A.codes_i8(x)
    assert q[0].tolist() == [127, 64, -64, 32] and (q[1] == 0).all() and s[1] == 0  # 63.5 goes to even
    w = np.eye(4, dtype=np.int8)
    assert np.allclose(A.matmul_i8(x, w, np.ones(4))[0], np.array([127, 64, -64, 32]) / 127)
