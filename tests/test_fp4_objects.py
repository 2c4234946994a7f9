"""Objects for matrices in 4 bits on the host: copies, what from_codes takes, and arrays that do not fit."""
import copy
import ctypes as C
import io
import pickle

import numpy as np
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S


def _matrix(N=5, K=80, fmt="nvfp4"):
    rng = np.random.default_rng(N + K)
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    s = rng.integers(1, 120, (N, -(-K // F.GROUP[fmt]))).astype(np.uint8)
    row = rng.random(N).astype(np.float32) if fmt == "nvfp4" else None
    return S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), K, fmt, row, device="cpu")


def _saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)), _saved])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_copies_have_their_own_memory(how, fmt):
    """What a copy hands to the kernels are its own arrays, and they are the ones that it shows."""
    q = _matrix(fmt=fmt)
    want = [t.clone() for t in (q.codes, q.scales)] + [None if q.row_scale is None else q.row_scale.clone()]
    c = how(q)
    q.codes.zero_()
    q.scales.zero_()
    for t, w, at in zip((c.codes, c.scales, c.row_scale), want, c._at):
        assert (t is None and w is None and at is None) or (torch.equal(t, w) and t.data_ptr() == at)
    c.codes.fill_(7)
    assert c._at[0] == c.codes.data_ptr() and int(q.codes.max()) == 0
    if fmt == "nvfp4":
        c.row_scale = None
        assert c._at[2] is None and c.row_scale is None and q._at[2] is not None and how(c).row_scale is None


def test_sizes_next_to_the_index_range():
    """Refused before anything is looked up: columns are counted in 32 bits, in tiles of up to 256 with offsets into them."""
    L = S.fp4._lib()
    P = 1 << 20  # an aligned address that no refused call touches
    for N in (1 << 31, (1 << 31) - 1, (1 << 31) - 512):
        assert L.smat_fp4_plan_spmm(None, P, 0, P, N, None) == -6
        assert L.smat_fp4_plan_spmm_fp4(None, P, P, None, 0, P, 0, N, None) == -6
    assert L.smat_fp4_plan_spmm(None, P, 0, P, (1 << 31) - 513, None) == -1  # no plan
    h = C.c_void_p()
    for M in (1 << 34, (1 << 35) - 16):
        assert L.smat_fp4_plan_create(C.byref(h), P, P, None, 0, P, P, M, 64, 3, 0, M // 16, 1, None) == -6 and not h.value


def _sparse(fmt="nvfp4"):
    rowptr, colidx = np.array([0, 2, 3], np.int32), np.array([0, 32, 16], np.int32)
    return S.Fp4SparseMatrix.from_codes(32, 48, rowptr, colidx, torch.zeros((3, 16, 8), dtype=torch.uint8), torch.zeros((3, 16), dtype=torch.uint8),
                                        fmt, np.ones(32, np.float32) if fmt == "nvfp4" else None, device="cpu")


@pytest.mark.parametrize("use", [S.Fp4Plan, lambda A: A.dequantize()])
def test_arrays_that_do_not_fit(use):
    """Arrays put in the place of a matrix's own are looked over before their addresses go to a kernel."""
    for name, value in (("row_scale", torch.ones(32, dtype=torch.float64)), ("row_scale", torch.ones(1).expand(32)), ("row_scale", torch.ones(16)),
                        ("row_scale", np.ones(32, np.float32)),
                        ("codes", torch.zeros((2, 16, 8), dtype=torch.uint8)), ("codes", torch.zeros((3, 16, 16), dtype=torch.uint8)[:, :, ::2]),
                        ("scales", torch.zeros((3, 16), dtype=torch.int32)), ("scales", torch.zeros((16, 3), dtype=torch.uint8).T),
                        ("bcsrRowPtr", torch.zeros(2, dtype=torch.int32)), ("bcsrRowPtr", torch.zeros(3, dtype=torch.int64)),
                        ("bcsrColIdx", torch.zeros(2, dtype=torch.int32)), ("bcsrColIdx", torch.zeros(3, dtype=torch.int32, device="meta"))):
        A = _sparse()
        setattr(A, name, value)
        with pytest.raises(S.SmatError, match=name) as e:
            use(A)
        assert e.value.code == -1
    A = _sparse("mxfp4")
    A.row_scale = torch.ones(32)
    with pytest.raises(S.SmatError, match="row_scale"):
        use(A)
    with pytest.raises(S.SmatError, match="current CUDA device"):  # the arrays of from_codes are fine
        use(_sparse())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_from_codes_takes_arrays_and_tensors(fmt):
    """numpy arrays, lists and tensors alike; what has no two dimensions is refused like any other wrong shape."""
    q = _matrix(fmt=fmt)
    codes, scales = q.codes[:, :40].numpy().copy(), q.group_scales().numpy().copy()
    row = None if q.row_scale is None else q.row_scale.numpy().copy()
    for convert in (lambda a: a, torch.from_numpy, lambda a: torch.from_numpy(a).t().contiguous().t()):
        p = S.Fp4Matrix.from_codes(convert(codes), convert(scales), 80, fmt, row, device="cpu")
        assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
        assert p.row_scale is None if row is None else torch.equal(p.row_scale, q.row_scale)
    for bad in (codes.reshape(-1), codes[0], np.uint8(3), codes[None]):
        with pytest.raises(S.SmatError, match="codes") as e:
            S.Fp4Matrix.from_codes(bad, scales, 80, fmt, row, device="cpu")
        assert e.value.code == -1
    for N, K in ((-1, 32), (2, -16)):
        with pytest.raises(S.SmatError):
            S.Fp4Matrix(N, K, device="cpu")


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, pickle.dumps])
def test_plans_are_not_copied(how):
    """Two objects with one handle would free it twice."""
    plan = S.Fp4Plan.__new__(S.Fp4Plan)
    plan._h = None
    with pytest.raises(TypeError, match="plan"):
        how(plan)
