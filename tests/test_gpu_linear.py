"""matmul_i8 on the GPU against oracle/attn.py.

The codes and the int32 sums are exact.  Left are roundings of fp32: the sum
as a float, the row's scale, the two scale products (2^-24 each) and the
residual's addition (2^-24 of the result), then half a step of out's type."""
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


def problem(seed, M, N, K, xt, norm, res, ot):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((M, K)) * rng.uniform(0.1, 3, (M, 1))).astype(np.float32)).to(DT[xt])
    w = torch.from_numpy(rng.integers(-128, 128, (N, K)).astype(np.int8))
    ws = torch.from_numpy(rng.uniform(0.5, 1.5, N).astype(np.float32) / 1000)
    nw = torch.from_numpy(rng.uniform(0.5, 1.5, K).astype(np.float32)) if norm else None
    r = torch.from_numpy(rng.standard_normal((M, N)).astype(np.float32)).to(DT[ot]) if res else None
    return x, w, ws, nw, r


def check(out, x, w, ws, nw, r, eps=1e-6):
    n = lambda t: None if t is None else t.float().cpu().numpy()
    ref = A.matmul_i8(n(x), w.cpu().numpy(), n(ws), n(nw), eps)
    full = ref if r is None else ref + n(r)
    # where a norm is given its fp64 steps may round the other way: a code on a border differs (never seen; not allowed for)
    tol = 5 * 2.0 ** -24 * (np.abs(ref) + np.abs(full)) + torch.finfo(out.dtype).eps / 2 * np.abs(full) * (1 + 1e-3) + 2.0 ** -25
    off = np.abs(out.float().cpu().numpy().astype(np.float64) - full)
    assert (off <= tol).all(), (float((off / tol).max()), np.unravel_index((off / tol).argmax(), off.shape), int((off > tol).sum()))


SHAPES = [(1, 1, 16), (1, 5120, 2048), (2, 48, 64), (3, 200, 80), (7, 1000, 2048), (8, 256, 4096), (9, 130, 1040), (16, 512, 2048),
          (17, 333, 512), (31, 64, 96), (32, 96, 1008), (33, 2048, 1024), (64, 640, 768), (65, 129, 160), (100, 255, 2064), (128, 128, 128),
          (200, 1111, 336), (257, 300, 2048), (511, 515, 272), (600, 1024, 4096),
          (1, 64, 8208), (4, 4096, 8192), (3, 40, 16384), (5, 33000, 64), (20, 33010, 208), (50, 32768, 128), (70, 16, 16384), (4096, 4100, 144),
          (222, 130, 2576), (300, 515, 4112), (129, 1922, 2704), (66, 1, 5008), (2000, 4098, 160)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("xt,ot,norm,res", [("f32", "f32", True, False), ("bf16", "f32", False, True), ("f16", "bf16", True, True),
                                            ("f32", "f16", False, False)])
def test_matmul(M, N, K, xt, ot, norm, res):
    from tinygiant_amd.linear import matmul_i8
    gpu_note(f"matmul_i8 {M} {N} {K} {xt} {ot} {norm} {res}")
    x, w, ws, nw, r = problem(M * 7 + N, M, N, K, xt, norm, res, ot)
    c = lambda t: None if t is None else t.cuda()
    out = matmul_i8(c(x), c(w), c(ws), norm=c(nw), residual=c(r), out_dtype=DT[ot])
    check(out, x, w, ws, nw, r)


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_matmul_largest_sums(M):
    """Every code +-127 against +-127 and -128 over the longest row: the sum fills 31 bits."""
    from tinygiant_amd.linear import matmul_i8
    gpu_note(f"matmul_i8 largest sums {M}")
    K = 131072
    x = torch.ones(M, K) * (1 - 2 * (torch.arange(M) % 2))[:, None]
    w = torch.full((20, K), -128, dtype=torch.int8)
    w[1::2] = 127
    ws = torch.ones(20)
    out = matmul_i8(x.cuda(), w.cuda(), ws.cuda())
    check(out, x, w, ws, None, None)


@pytest.mark.parametrize("M", [1, 6, 20, 130])
def test_matmul_rows_at_the_edges(M):
    """Zero rows, rows with NaN or inf (NaN, and only they), tiny and huge rows, halves of the largest value."""
    from tinygiant_amd.linear import matmul_i8
    gpu_note(f"matmul_i8 edges {M}")
    N, K = 70, 272
    for kind in range(6):
        for norm in (False, True):
            x, w, ws, nw, _ = problem(kind, M, N, K, "f32", norm, False, "f32")
            row = M // 2
            if kind == 0:
                x[row] = 0
            elif kind == 1:
                x[row, K - 1] = float("nan")
            elif kind == 2:
                x[row, 3] = float("-inf")
            elif kind == 3:
                x[row] *= 1e-41 if not norm else 1e-30
            elif kind == 4:
                x[row] *= 1e30 if not norm else 1e18
            else:
                x[row] = torch.where(torch.arange(K) % 3 == 0, 1.0, 0.5) * 3
            out = matmul_i8(x.cuda(), w.cuda(), ws.cuda(), norm=None if nw is None else nw.cuda()).cpu()
            if kind in (1, 2):
                assert torch.isnan(out[row]).all()
                keep = torch.arange(M) != row
                out, x = out[keep], x[keep]
            if len(x) and not (kind == 3 and not norm):
                check(out, x, w, ws, nw, None)
            elif len(x):
                assert torch.isfinite(out).all() and (out[row].abs() < 1e-35).all()


def test_matmul_strides_shapes_and_aliases():
    from tinygiant_amd.linear import matmul_i8
    gpu_note("matmul_i8 strides")
    for M in (1, 4, 50, 200):
        x, w, ws, nw, r = problem(M, M, 96, 128, "bf16", True, True, "f32")
        wide = torch.zeros(M, 300, dtype=torch.bfloat16, device="cuda")
        xs = wide[:, 3:131]
        xs.copy_(x)
        acc = torch.full((M, 101), 9.0, device="cuda")
        acc[:, 1:97] = r.cuda()
        o = matmul_i8(xs, w.cuda(), ws.cuda(), norm=nw.cuda(), residual=acc[:, 1:97], out=acc[:, 1:97])
        check(o, x, w, ws, nw, r)
        assert (acc[:, 0] == 9).all() and (acc[:, 97:] == 9).all()
    x, w, ws, nw, _ = problem(5, 24, 40, 64, "f16", False, False, "f16")
    out = matmul_i8(x.cuda().view(2, 3, 4, 64), w.cuda(), ws.cuda())
    assert out.shape == (2, 3, 4, 40) and out.dtype == torch.float16
    check(out.view(24, 40), x, w, ws, None, None)
    assert matmul_i8(x.cuda()[:0], w.cuda(), ws.cuda()).shape == (0, 40)


def test_matmul_split_columns_in_place():
    """Few tiles, many columns (split): strided rows, the residual in out's place, the bytes around it untouched, twice the same."""
    from tinygiant_amd.linear import matmul_i8
    gpu_note("matmul_i8 split columns in place")
    x, w, ws, nw, r = problem(3, 150, 90, 4112, "f16", True, True, "bf16")
    for width, at in ((101, 3), (128, 16)):
        outs = []
        for _ in range(2):
            acc = torch.full((150, width), 9.0, dtype=torch.bfloat16, device="cuda")
            acc[:, at:at + 90] = r.cuda()
            o = matmul_i8(x.cuda(), w.cuda(), ws.cuda(), norm=nw.cuda(), residual=acc[:, at:at + 90], out=acc[:, at:at + 90])
            check(o, x, w, ws, nw, r)
            assert (acc[:, :at] == 9).all() and (acc[:, at + 90:] == 9).all()
            outs.append(o.clone())
        assert torch.equal(*outs)


def test_matmul_refuses_on_device():
    from tinygiant_amd.linear import matmul_i8
    x, w, ws = torch.zeros(4, 64, device="cuda"), torch.zeros(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: matmul_i8(x[:, ::2], w[:, :32].contiguous(), ws), lambda: matmul_i8(x, w[:, :32], ws),
                lambda: matmul_i8(x, w, ws[:7]), lambda: matmul_i8(x, w, ws.half()), lambda: matmul_i8(x.int(), w, ws),
                lambda: matmul_i8(x, w, ws, norm=torch.ones(64)), lambda: matmul_i8(x, w, ws, residual=torch.zeros(4, 8, device="cuda").half()),
                lambda: matmul_i8(x, w, ws, out=torch.zeros(3, 8, device="cuda")),
                lambda: matmul_i8(x, w, ws, out=torch.zeros(4, 8, device="cuda"), out_dtype=torch.float16)):
        with pytest.raises((TypeError, ValueError)):
            bad()
