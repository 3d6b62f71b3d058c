"""The attention block restated in numpy: the paged Q4_0 cache, causal
grouped-query attention over it, and the int8 product.

TEST INFRASTRUCTURE ONLY: the checker that tests/ compare libtinygiant's
tg_kv_*_q4_dev, tg_attn_q4_dev and tg_matmul_i8_dev with.  Nothing in the
product imports it.  The cache's arithmetic (norm, rotation, quantisation) is
restated in the types the operator is defined in, so its bytes are compared
exactly; attention and the product are computed in float64.
"""
from __future__ import annotations

import numpy as np

f32 = np.float32


def norm_rows(x, w, eps):
    """x / rms(x) * w over the last axis: the mean square in float64 rounded
    to float32, everything else in float32."""
    x = np.asarray(x, f32)
    if w is None:
        return x
    ms = np.mean(x.astype(np.float64) ** 2, axis=-1, keepdims=True).astype(f32)
    return x * (f32(1) / np.sqrt(ms + f32(eps))) * np.asarray(w, f32)


def rotate(x, cos, sin):
    """Pairs (i, i + half) of the last axis turned by their table row
    (csrc/libtinygiant.c:344-361, each product and sum rounded)."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], axis=-1)


def q4_0(x):
    """Q4_0 of float32 [..., D]: codes uint8 [..., D], scales float16 [..., D / 32]."""
    x = np.asarray(x, f32)
    x = np.where(np.isnan(x), x, np.clip(x, f32(-65504), f32(65504)))
    b = x.reshape(*x.shape[:-1], -1, 32)
    nan = np.isnan(b).any(axis=-1, keepdims=True)
    first = np.argmax(np.nan_to_num(np.abs(b), nan=-1.0), axis=-1)[..., None]  # first of the largest
    d = np.take_along_axis(b, first, axis=-1) / f32(-8)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(d != 0, f32(1) / d, f32(0)).astype(f32)
        code = np.clip(np.nan_to_num(np.trunc(b * inv + f32(8.5)), nan=15.0), 0, 15)
    d = np.where(nan, f32(np.nan), d)
    return code.astype(np.uint8).reshape(x.shape), d[..., 0].astype(np.float16)


class Cache:
    """One layer's pages as bytes [n_pages, n_kv, page_tokens / 16, 18 D]."""

    def __init__(self, n_pages, page_tokens, n_kv, D, pages=None):
        self.page_tokens, self.n_kv, self.D = page_tokens, n_kv, D
        self.pages = np.zeros((n_pages, n_kv, page_tokens // 16, 18 * D), np.uint8) if pages is None else pages

    def _places(self, r):
        """Halfword and nibble of each dim's K and V code, and the halfword of each block's scales, for token r."""
        D, NG = self.D, self.D // 32
        d = np.arange(D)
        g, e = d // 32, d % 32
        j, c = d // 16, d % 16
        k = (((e // 8) * 16 + r) * NG + g) * 2 + e % 2
        v = 4 * D + (((r // 4) * 16 + c) * 2 + (r % 4) // 2) * NG + 2 * (j // 4) + r % 2
        n = np.arange(NG)
        return k, (e % 8) // 2, v, j % 4, 8 * D + r * NG + n, 8 * D + D // 2 + ((r // 2) * NG + n) * 2 + r % 2

    def put(self, page, head, p, k, v):
        """Float32 k, v [D] of the token at place p of a page."""
        tile = self.pages[page, head, p // 16].view(np.uint16)
        ka, kn, va, vn, ks, vs = self._places(p % 16)
        for x, at, nib, sat in ((k, ka, kn, ks), (v, va, vn, vs)):
            code, d = q4_0(x)
            for i, a in enumerate(at):
                tile[a] = (int(tile[a]) & ~(15 << (4 * int(nib[i])))) | (int(code[i]) << (4 * int(nib[i])))
            tile[sat] = d.view(np.uint16)

    def get(self, page, head, p):
        """Float64 k, v [D] that the cache holds."""
        tile = self.pages[page, head, p // 16].view(np.uint16)
        ka, kn, va, vn, ks, vs = self._places(p % 16)
        out = []
        for at, nib, sat in ((ka, kn, ks), (va, vn, vs)):
            code = (tile[at].astype(np.int64) >> (4 * nib)) & 15
            out.append((code - 8) * np.repeat(tile[sat].view(np.float16).astype(np.float64), 32))
        return out

    def rows(self, table_row, n, steps=False):
        """K and V [n_kv, n, D] float64 of a sequence's first n tokens;
        steps: the scales of their blocks instead, spread over the dims."""
        t = np.arange(n)
        page = np.asarray(table_row)[t // self.page_tokens]
        tile = self.pages[page, :, t % self.page_tokens // 16].view(np.uint16)  # [n, n_kv, 9 D]
        places = [self._places(r) for r in range(16)]
        out = []
        for code_at, nib, scale_at in ((0, 1, 4), (2, 3, 5)):
            at = np.stack([pl[code_at] for pl in places])[t % 16][:, None]
            sat = np.stack([pl[scale_at] for pl in places])[t % 16][:, None]
            d = np.repeat(np.take_along_axis(tile, sat, axis=2).view(np.float16).astype(np.float64), 32, axis=2)
            code = (np.take_along_axis(tile, at, axis=2).astype(np.int64) >> (4 * places[0][nib])) & 15
            out.append(np.moveaxis(d if steps else (code - 8) * d, 1, 0))
        return out


def attend(q, k, v, n_new, scale, steps=None, seen=None):
    """q [n_new, heads, D], the last rows of a sequence with k, v [n_kv, n,
    D]: row i sees positions 0 .. n - n_new + i, and of the last n_new of them
    (seen [n_new, n_new], for draft trees) those that seen[i] says.  Returns in float64 out
    [n_new, heads, D], sum p |v| of the same shape, and the largest scale *
    sum |q_i k_i| that each row sees [n_new, heads, 1] (for error bounds).
    steps (the scales of k's and v's blocks): two more for bounds, sum p
    |step of v| and the largest scale * max |q| * sum of |steps of k|'s
    blocks that a row sees."""
    n_kv, n, D = k.shape
    heads = q.shape[1]
    G = heads // n_kv
    out, size, vstep = np.zeros((3, n_new, heads, D))
    top, kstep = np.zeros((2, n_new, heads, 1))
    hide = np.arange(n)[None, :] > np.arange(n - n_new, n)[:, None]
    if seen is not None:
        hide[:, max(0, n - n_new):] |= ~seen[:, max(0, n_new - n):]
    blind = hide.all(axis=1) if n else np.ones(n_new, bool)
    for h in range(heads if n else 0):
        x = q[:, h].astype(np.float64)
        s = np.where(hide, -np.inf, scale * (x @ k[h // G].T))
        s[blind] = 0
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        w[blind] = 0
        out[:, h], size[:, h] = w @ v[h // G], w @ np.abs(v[h // G])
        a = np.where(hide, 0, scale * (np.abs(x) @ np.abs(k[h // G]).T))
        top[:, h, 0] = a.max(axis=1)
        if steps:
            vstep[:, h] = w @ np.abs(steps[1][h // G])
            a = np.where(hide, 0, np.abs(steps[0][h // G][:, ::32]).sum(axis=1)[None, :])
            kstep[:, h, 0] = scale * np.abs(x).max(axis=1) * a.max(axis=1)
    return (out, size, top, vstep, kstep) if steps else (out, size, top)


def codes_i8(x, norm=None, eps=1e-6):
    """Per-row int8 codes and scales (float64) of x [M, K]."""
    x = np.asarray(x, np.float64)
    if norm is not None:
        x = x * (1.0 / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps)) * np.asarray(norm, np.float64)
    a = np.abs(x).max(axis=1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(a > 0, np.rint(127.0 * x / a), 0.0)
    return q, a / 127.0


def matmul_i8(x, w, w_scale, norm=None, eps=1e-6, residual=None):
    q, s = codes_i8(x, norm, eps)
    out = (q @ w.astype(np.float64).T) * s * np.asarray(w_scale, np.float64)
    return out if residual is None else out + np.asarray(residual, np.float64)
