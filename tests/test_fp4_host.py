"""Refusals and host-side layouts of the 4-bit entry points; none needs a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S
from smat_b200 import fp4

P = 1 << 20  # an aligned address that no refused call touches
BAD, RANGE = -1, -6


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("N,K", [(1, 16), (5, 48), (128, 64), (130, 80), (257, 400)])
def test_scale_tiles(fmt, N, K):
    rng = np.random.default_rng(N)
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    s = rng.integers(0, 120, (N, -(-K // F.GROUP[fmt]))).astype(np.uint8)
    q = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), K, fmt, device="cpu")
    L = fp4._lib()
    L.smat_fp4_codes_bytes.argtypes = L.smat_fp4_scales_bytes.argtypes = [C.c_size_t, C.c_size_t]
    L.smat_fp4_codes_bytes.restype = L.smat_fp4_scales_bytes.restype = C.c_size_t
    assert q.codes.numel() == L.smat_fp4_codes_bytes(N, K) and q.scales.numel() == L.smat_fp4_scales_bytes(N, K)
    assert np.array_equal(q.group_scales().numpy(), s)
    assert np.array_equal(F.unpack(q.codes.numpy())[:, :K], codes) and not F.unpack(q.codes.numpy())[:, K:].any()
    flat, quads = q.scales.numpy(), -(-K // 64)
    for r, k in [(0, 0), (N - 1, K - 16), (N // 2, K // 2 // 16 * 16)]:  # the byte where the header says it is
        j = k // 16 % 4 if fmt == "nvfp4" else k // 32 % 2
        assert flat[(r // 128 * quads + k // 64) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + j] == s[r, k // F.GROUP[fmt]]


def test_sign_of_e4m3_scales_is_dropped():
    s = torch.tensor([[0x85]], dtype=torch.uint8)
    q = S.Fp4Matrix.from_codes(torch.zeros((1, 8), dtype=torch.uint8), s, 16, device="cpu")
    assert int(q.group_scales()) == 5


def test_python_refusals():
    ok = torch.zeros((2, 32), dtype=torch.float16)
    codes, sc = torch.zeros((2, 16), dtype=torch.uint8), torch.zeros((2, 2), dtype=torch.uint8)
    for call in (
        lambda: S.Fp4Matrix.quantize(ok),                                # not on a GPU
        lambda: S.Fp4Matrix.quantize(ok, "fp8"),
        lambda: S.Fp4Matrix.quantize(ok.double()),
        lambda: S.Fp4Matrix.quantize(ok[0]),
        lambda: S.Fp4Matrix.quantize(ok.T),
        lambda: S.Fp4Matrix(2, 24, device="cpu"),
        lambda: S.Fp4Matrix.from_codes(codes, sc, 32, "nvfp4", torch.ones(3), device="cpu"),
        lambda: S.Fp4Matrix.from_codes(codes, sc[:, :1], 32, device="cpu"),
        lambda: S.Fp4Matrix.from_codes(codes.short(), sc, 32, device="cpu"),
        lambda: S.Fp4Matrix.from_codes(codes, sc[:, :1], 32, "mxfp4", 2.0, device="cpu"),
        lambda: S.Fp4Matrix.from_codes(codes, sc, 32, device="cpu").dequantize(),
        lambda: S.Fp4SparseMatrix.from_codes(32, 32, [0, 1], [0], torch.zeros((1, 16, 8), dtype=torch.uint8), torch.zeros((1, 16), dtype=torch.uint8), device="cpu"),
        lambda: S.Fp4SparseMatrix.from_codes(16, 32, [0, 1], [0], torch.zeros((1, 128), dtype=torch.uint8), torch.zeros((1, 16), dtype=torch.uint8), device="cpu"),
    ):
        with pytest.raises(S.SmatError) as e:
            call()
        assert e.value.code == BAD


def test_c_refusals_of_quantize():
    L = fp4._lib()
    call = L.smat_fp4_quantize
    good = dict(X=P, dtype=0, N=4, K=64, ldx=64, fmt=0, codes=P, scales=P, row=P)

    def rc(**kw):
        a = {**good, **kw}
        return call(a["X"], a["dtype"], a["N"], a["K"], a["ldx"], a["fmt"], a["codes"], a["scales"], a["row"], None)
    for kw, code in [(dict(K=24, ldx=24), BAD), (dict(dtype=3), BAD), (dict(fmt=2), BAD), (dict(fmt=-1), BAD), (dict(X=None), BAD), (dict(codes=None), BAD),
                     (dict(scales=None), BAD), (dict(row=None), BAD), (dict(X=P + 8), BAD), (dict(codes=P + 4), BAD), (dict(scales=P + 1), BAD),
                     (dict(ldx=48), BAD), (dict(ldx=68), BAD), (dict(dtype=2, ldx=66), BAD), (dict(N=1 << 31), RANGE), (dict(K=1 << 30, ldx=1 << 30), RANGE)]:
        assert rc(**kw) == code, kw
    assert L.smat_fp4_dequantize(P, P, None, 0, 4, 64, P, 5, 64, None) == BAD
    assert L.smat_fp4_dequantize(P, P, None, 0, 4, 64, P, 0, 32, None) == BAD


def test_c_refusals_of_blocks_and_plans():
    L = fp4._lib()
    q, d = L.smat_fp4_quantize_blocks, L.smat_fp4_dequantize_blocks
    assert q(P, 0, P, P, 24, 1, 0, P, P, P, None) == BAD
    assert q(P, 0, None, P, 32, 1, 0, P, P, P, None) == BAD
    assert q(P, 0, P, None, 32, 1, 0, P, P, P, None) == BAD
    assert q(P, 0, P, P, 32, 1, 0, P, P, None, None) == BAD
    assert q(P + 2, 0, P, P, 32, 1, 0, P, P, P, None) == BAD
    assert q(P, 0, P, P, 32, 1 << 27, 0, P, P, P, None) == RANGE
    assert d(P, P, None, 3, P, 32, 1, P, 0, None) == BAD
    assert d(P, P, None, 0, P, 32, 1, None, 0, None) == BAD
    h = C.c_void_p()
    good = [P, P, None, 0, P, P, 64, 64, 3, 0, 4, 1]

    def rc(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return L.smat_fp4_plan_create(C.byref(h), *a, None)
    for kw, code in [(dict(a0=None), BAD), (dict(a1=None), BAD), (dict(a0=P + 8), BAD), (dict(a3=2), BAD), (dict(a4=None), BAD), (dict(a5=None), BAD),
                     (dict(a6=40), BAD), (dict(a7=40), BAD), (dict(a9=3, a10=2), BAD), (dict(a10=5), BAD), (dict(a8=1 << 27), RANGE), (dict(a7=1 << 31), RANGE), (dict(a7=1 << 26), RANGE)]:
        assert rc(**kw) == code and not h.value, kw
    assert L.smat_fp4_plan_create(None, *good, None) == BAD
    assert L.smat_fp4_plan_spmm(None, P, 0, P, 8, None) == BAD
    assert L.smat_fp4_plan_spmm(None, P, 2, P, 8, None) == BAD
    assert L.smat_fp4_plan_spmm_fp4(None, P, P, None, 0, P, 0, 8, None) == BAD
    assert L.smat_fp4_plan_set_values(None, None) == BAD
    assert L.smat_fp4_plan_destroy(None) == 0
