"""Quantisation to 4 bits and back against the definition in 64 bits: equal bit for bit."""
import numpy as np
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S

pytestmark = pytest.mark.gpu
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _host(t):
    return t.double().cpu().numpy()


def _same_dense(X, fmt):
    q = S.Fp4Matrix.quantize(X, fmt)
    codes, s, p = F.quantize_dense(_host(X), fmt)
    K = X.shape[1]
    got = F.unpack(q.codes.cpu().numpy())
    assert np.array_equal(q.group_scales().cpu().numpy(), s)
    assert np.array_equal(got[:, :K] & 7, codes & 7)
    assert np.array_equal((got[:, :K] > 8), codes > 8)  # the sign of a zero is free
    assert not got[:, K:].any()
    if fmt == "nvfp4":
        assert np.array_equal(q.row_scale.double().cpu().numpy(), p)
    else:
        assert q.row_scale is None
    return q, F.dense_values(codes, s, p, fmt)


def _same_values(t, want):
    """t holds `want` (64 bits) rounded once to its type."""
    want = torch.from_numpy(want).to(t.dtype).cpu()
    assert torch.equal(torch.nan_to_num(t.cpu().float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("N,K", [(1, 16), (1, 32), (5, 48), (33, 64), (129, 80), (3, 1040), (2, 4112), (300, 256), (1, 28672), (2, 8192), (3, 16384), (2, 36880), (2, 65536)])
def test_quantize(fmt, dt, N, K):
    g = torch.Generator("cuda").manual_seed(N + K)
    X = (torch.randn((N, K), generator=g, device="cuda") * torch.exp(torch.randn((N, 1), generator=g, device="cuda"))).to(DTYPES[dt])
    q, want = _same_dense(X, fmt)
    for out in DTYPES.values():
        _same_values(q.dequantize(out), want)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_quantize_ties(fmt, dt):
    """Quotients on the borders between codes and between scales, and their neighbours."""
    rng = np.random.default_rng(1)
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 1.5, 2, 3, 4, 6, 5.5, 6.25])
    rows = []
    for s in [1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875]:
        x = border * s
        x[14] = 6 * s  # the group's largest: its scale is s
        rows.append(x)
    mids = (F.E4M3[1:] + F.E4M3[:-1]) / 2
    X = np.tile(np.array(rows), (40, 2)) * rng.choice([-1.0, 1.0], (320, 32))
    X[:126, 0] = 6 * mids * np.where(mids > 1, 1 / 64, 1)  # scales next to a tie
    X = torch.from_numpy(X).cuda().to(DTYPES[dt])
    if dt == "f32":
        i = X.view(torch.int32)
        X = torch.cat([X, (i + 1).view(torch.float32), (i - 1).view(torch.float32)])
    _same_dense(X, fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_quantize_extremes(fmt, dt):
    """Rows of zeros, of the type's smallest and largest values, NaN and infinities, which spoil their group only."""
    t = DTYPES[dt]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    X = torch.randn((12, 160), device="cuda").to(t)
    X[0] = 0
    X[1] = big
    X[2] = tiny
    X[3] = 0
    X[3, 7] = torch.finfo(t).smallest_normal * torch.finfo(t).eps  # the smallest subnormal
    X[4, ::3] = big
    X[5, 20] = float("nan")
    X[6, 33] = float("inf")
    X[7] = float("-inf")
    X[8, 150:] = float("nan")
    X[9] = -0.0
    X[10, 1:] = 0
    X[11] *= tiny
    q, want = _same_dense(X, fmt)
    assert np.isnan(want[5, 16:32]).all() and np.isfinite(want[5, 32:]).all()
    _same_values(q.dequantize(torch.float32), want)


def test_quantize_rows_far_apart_and_out():
    """Strided rows, and storage that is used again."""
    X = torch.randn((40, 512), device="cuda", dtype=torch.float16)
    part = X[::2, 64:64 + 208]
    q, want = _same_dense(part, "nvfp4")
    again = S.Fp4Matrix.quantize(part.contiguous() * 2, "nvfp4", out=q)
    assert again is q
    wide = torch.full((20, 256), 7.0, device="cuda", dtype=torch.float32)
    q.dequantize(out=wide[:, 16:224])
    _same_values(wide[:, 16:224], 2 * want)
    assert bool((wide[:, :16] == 7).all()) and bool((wide[:, 224:] == 7).all())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_from_codes(fmt):
    """Arrays of a checkpoint, with any row scales; two roundings of fp32 on the way back."""
    rng = np.random.default_rng(2)
    N, K = 131, 112
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    s = rng.integers(40, 120, (N, -(-K // F.GROUP[fmt]))).astype(np.uint8)
    p = (rng.random(N) + 0.5).astype(np.float32) if fmt == "nvfp4" else None
    q = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), K, fmt, p)
    assert np.array_equal(q.group_scales().cpu().numpy(), s)
    want = F.dense_values(codes, s, p, fmt)
    got = _host(q.dequantize(torch.float32))
    assert np.max(np.abs(got - want) / np.maximum(np.abs(want), 1e-300)) <= 2 * 2.0 ** -24 * (1 + 1e-6)
    if fmt == "nvfp4":
        one = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s).view(torch.float8_e4m3fn), K, fmt, 0.25)
        _same_values(one.dequantize(torch.float32), F.dense_values(codes, s, np.full(N, 0.25), fmt))


def _matrix(rng, counts, Kb, scale=0.1):
    rowptr, colidx = F.random_blocks(rng, counts, Kb)
    vals = (rng.standard_normal((rowptr[-1], 16, 16)) * scale).astype(np.float16)
    return rowptr, colidx, vals, S.SparseMatrix.from_bcsr(len(counts) * 16, Kb * 16, rowptr, colidx, vals.reshape(-1))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("counts,Kb", [([1], 1), ([0, 3, 0, 0, 9], 9), ([7, 16, 1, 33, 0, 2], 37), ([200, 5, 190], 201)])
def test_quantize_blocks(fmt, counts, Kb):
    rng = np.random.default_rng(len(counts) + Kb)
    rowptr, colidx, vals, A = _matrix(rng, counts, Kb)
    if len(vals) > 20:
        vals[5] = 0
        vals[6, 3, 4], vals[7, 2, 1], vals[8, 15, 15] = np.inf, np.nan, 6e4
        A = S.SparseMatrix.from_bcsr(A.M, A.K, rowptr, colidx, vals.reshape(-1))
    A4 = S.Fp4SparseMatrix.quantize(A, fmt, check=True)
    codes, s, p = F.quantize_blocks(vals, rowptr, colidx, fmt)
    got = F.unpack(A4.codes.cpu().numpy())
    assert np.array_equal(A4.scales.cpu().numpy(), s)
    assert np.array_equal(got & 7, codes & 7) and np.array_equal(got > 8, codes > 8)
    if fmt == "nvfp4":
        assert np.array_equal(A4.row_scale.double().cpu().numpy(), p)
    back = A4.dequantize(check=True)
    assert (back.M, back.K, back.nnzb) == (A.M, A.K, A.nnzb)
    _same_values(back.bcsrVal.view(-1, 16, 16), F.block_values(codes, s, p, rowptr, fmt))


def test_pairs_across_block_rows_do_not_share():
    """The last block of a block-row and the first of the next one may be neighbours in the arrays and in their columns."""
    rowptr, colidx = np.array([0, 1, 2], np.int32), np.array([0, 16], np.int32)
    vals = np.ones((2, 16, 16), np.float16)
    vals[1] *= 100
    A = S.SparseMatrix.from_bcsr(32, 32, rowptr, colidx, vals.reshape(-1))
    s = S.Fp4SparseMatrix.quantize(A, "mxfp4").scales.cpu().numpy()
    assert (s[0] == 127 - 2).all() and (s[1] == 127 + 6 - 2).all()


def test_bad_row_pointers_are_reported():
    rowptr, colidx = np.array([0, 2, 1, 3], np.int32), np.array([0, 16, 0], np.int32)
    vals = np.ones((3, 16, 16), np.float16)
    A = S.SparseMatrix.from_bcsr(48, 32, rowptr, colidx, vals.reshape(-1))
    with pytest.raises(S.SmatError) as e:
        S.Fp4SparseMatrix.quantize(A, "nvfp4", check=True)
    assert e.value.code == -6
    A4 = S.Fp4SparseMatrix.quantize(S.SparseMatrix.from_bcsr(48, 32, np.array([0, 1, 2, 3], np.int32), colidx, vals.reshape(-1)), check=True)
    A4.bcsrRowPtr = A.bcsrRowPtr
    with pytest.raises(S.SmatError) as e:
        A4.dequantize(check=True)
    assert e.value.code == -6
