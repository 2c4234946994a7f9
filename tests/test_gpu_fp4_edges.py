"""Matrices in 4 bits where ranges, structures and host state end: scales next to both ends, inconsistent arrays, plans made on
several threads, errors that must not outlive their call."""
import threading

import numpy as np
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S
from test_gpu_fp4_spmm import HALF, LEAST, Case, _close

pytestmark = pytest.mark.gpu


def _case(fmt, counts, Kb, scales, seed=3):
    """A Case whose scale bytes are `scales` [rows of all block-rows], the same for all blocks of a row."""
    c = Case(seed, counts, Kb, fmt, row_scale=False)
    brow = np.repeat(np.arange(len(counts)), counts)
    c.scales = np.asarray(scales, np.uint8).reshape(-1, 16)[brow]
    c.A = S.Fp4SparseMatrix.from_codes(c.M, c.K, c.rowptr, c.colidx, F.pack(c.codes), c.scales, fmt)
    c.vals = F.block_values(c.codes, c.scales, None, c.rowptr, fmt)
    return c


@pytest.mark.parametrize("N", [40, 150])
def test_refreshed_tiles(N):
    """set_values brings changed codes and scales to the tiles too, of one CTA and of pairs."""
    c = Case(8, [30] * 40, 48, "nvfp4")
    B, b = c.acts4(N)
    plan = S.Fp4Plan(c.A)
    C = torch.empty((c.M, N), dtype=torch.bfloat16, device="cuda")
    plan.spmm(B, C, check=True)
    _close(C, *F.multiply(c.vals, c.rowptr, c.colidx, b), c.longest)
    c.A.codes.copy_(c.A.codes.flip(0))
    c.A.scales.copy_(c.A.scales.roll(5, 0))
    plan.set_values()
    plan.spmm(B, C, check=True)
    vals = F.block_values(F.unpack(c.A.codes.cpu().numpy()), c.A.scales.cpu().numpy(), c.p, c.rowptr, "nvfp4")
    _close(C, *F.multiply(vals, c.rowptr, c.colidx, b), c.longest)
    D = torch.empty_like(C)
    S.Fp4Plan(c.A).spmm(B, D)
    assert torch.equal(C, D)


@pytest.mark.parametrize("N", [5, 40, 150])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("swap", [False, True])
def test_e8m0_from_end_to_end(N, tiles, swap):
    """mxfp4 scales over their whole range on one side, all of the reverse size on the other: the products are of ordinary size and
    so are all sums, in every kernel.  swap: the rows of A get one scale, the tokens theirs."""
    rng = np.random.default_rng(N)
    Kb = 24
    byte = np.concatenate([[0, 1, 2, 3, 4, 5, 249, 250, 251, 252, 253, 254], rng.integers(6, 249, 20)])
    rows, tokens = byte, np.resize(byte, N)
    for other in (1, 60, 127, 190, 254):
        a, t = (rows, np.full(N, other)) if not swap else (np.full(32, other), tokens)
        c = _case("mxfp4", [20, 24], Kb, a)
        codes = rng.integers(0, 16, (N, c.K)).astype(np.uint8)
        s = np.repeat(t.astype(np.uint8)[:, None], Kb // 2, 1)
        B = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), c.K, "mxfp4")
        ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, F.dense_values(codes, s, None, "mxfp4"))
        C = torch.full((c.M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
        S.Fp4Plan(c.A, tiles=tiles).spmm(B, C, check=True)
        got = C.double().cpu().numpy()
        fine = (mag < 2.0 ** 127) & (mag > 2.0 ** -100)  # sums that fp32 holds with all their digits
        tol = (c.longest + 32) * 2.0 ** -22 * mag + HALF[C.dtype] * np.abs(ref) * (1 + 1e-3) + LEAST[C.dtype]
        assert np.all(np.abs(got - ref)[fine] <= tol[fine]), (other, np.argwhere(fine & ~(np.abs(got - ref) <= tol))[:5].tolist())


@pytest.mark.parametrize("N", [1, 5, 40, 100])
def test_e8m0_of_weights_with_bf16(N):
    """The same with activations in bf16."""
    rng = np.random.default_rng(N)
    byte = np.concatenate([[0, 1, 2, 3, 4, 5, 249, 250, 251, 252, 253, 254], rng.integers(6, 249, 20)])
    c = _case("mxfp4", [20, 24], 24, byte)
    for size in (-120, -60, 0, 60, 120):
        x = torch.from_numpy(rng.standard_normal((N, c.K)) * 2.0 ** size).bfloat16().cuda()
        ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, x.double().cpu().numpy())
        C = torch.full((c.M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
        S.Fp4Plan(c.A).spmm(x, C, check=True)
        got = C.double().cpu().numpy()
        fine = (mag < 2.0 ** 127) & (mag > 2.0 ** -100)
        tol = (c.longest + 32) * 2.0 ** -22 * mag + HALF[C.dtype] * np.abs(ref) * (1 + 1e-3) + LEAST[C.dtype]
        assert np.all(np.abs(got - ref)[fine] <= tol[fine]), size


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_row_scales_of_any_size(dtype):
    """Values on the way back are code * scale, which is exact, times the row scale, rounded to fp32 and from there to their type:
    nothing between overflows, loses digits or turns a zero into NaN."""
    rng = np.random.default_rng(4)
    N, K = 24, 64
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    s = rng.integers(1, 127, (N, K // 16)).astype(np.uint8)
    s[:, 0] = 126  # 448
    p = (rng.random(N) + 0.5).astype(np.float32)
    p[:4] = [3e38, 1e37, 2e-38, 1e-39]
    q = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), K, "nvfp4", p)
    exact = F.dense_values(codes, s, p, "nvfp4")
    with np.errstate(over="ignore"):
        want = torch.from_numpy(exact.astype(np.float32)).to(dtype)  # numpy rounds once to fp32, torch once to the type
    assert torch.equal(q.dequantize(dtype).cpu(), want)
    rowptr, colidx = np.array([0, 2], np.int32), np.array([0, 32], np.int32)
    bc, bs = codes[:16].reshape(16, 4, 16)[:, :2].transpose(1, 0, 2), s[:16, :2].T
    A = S.Fp4SparseMatrix.from_codes(16, 48, rowptr, colidx, F.pack(np.ascontiguousarray(bc)), np.ascontiguousarray(bs), "nvfp4", p[:16])
    with np.errstate(over="ignore"):
        want = torch.from_numpy(F.block_values(bc, bs, p[:16], rowptr, "nvfp4").astype(np.float32)).half()
    assert torch.equal(A.dequantize(check=True).bcsrVal.cpu().view(2, 16, 16), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_first_e4m3_scales(dtype):
    """Groups whose scale is among the first e4m3 numbers, beside a large value in the row: their quotients reach 9, and lie on and next
    to the borders between codes."""
    eighths = np.arange(0, 73) / 8  # multiples of 1/8 up to 9: all borders and what is next to them in 11 bits
    rows = []
    for byte in range(1, 9):
        s = F.E4M3[byte]
        for gmax in (s * 6 * (1 - 2.0 ** -5), s * 6, s * 6 * (1 + 2.0 ** -5), (s + 2.0 ** -10) * 6 * (1 - 2.0 ** -7)):
            x = np.minimum(np.resize(eighths * s, 16 * 5), gmax).reshape(5, 16)
            x[:, 0] = gmax
            rows.append(np.concatenate([[2688.0], np.zeros(15), x.reshape(-1)]))
    X = torch.from_numpy(np.array(rows)).to(dtype).cuda()
    q = S.Fp4Matrix.quantize(X)
    codes, s, p = F.quantize_dense(X.double().cpu().numpy(), "nvfp4")
    assert (p == 1).all() and s[:, 1:].min() <= 1 and s[:, 1:].max() <= 9
    assert np.array_equal(q.group_scales().cpu().numpy(), s)
    got = F.unpack(q.codes.cpu().numpy())[:, :X.shape[1]]
    assert np.array_equal(got & 7, codes & 7)
    d = X.double().cpu().numpy()[:, 16:].reshape(len(rows), 5, 16) / np.maximum(F.E4M3[s[:, 1:]], 2.0 ** -12)[..., None]
    assert d.max() > 8.5


@pytest.mark.parametrize("N,tiles", [(3, True), (5, False), (40, True), (40, False), (150, True)])
def test_pairs_with_different_scales_are_reported(N, tiles):
    """mxfp4: blocks of a pair share their scales; a block-row where they do not counts as empty, in every kernel."""
    c = Case(21, [16, 16, 16], 16, "mxfp4")
    x, (B, b) = c.acts(N, torch.float16), c.acts4(N)
    ref4, mag4 = F.multiply(c.vals, c.rowptr, c.colidx, b)
    ref16, mag16 = F.multiply(c.vals, c.rowptr, c.colidx, x.double().cpu().numpy())
    good = c.A.scales.clone()
    C = torch.empty((c.M, N), dtype=torch.float16, device="cuda")
    plan = S.Fp4Plan(c.A, tiles=tiles)
    for made_anew in (True, False):
        c.A.scales.copy_(good)
        c.A.scales[16 + 7, 3] ^= 1
        if made_anew:
            plan = S.Fp4Plan(c.A, tiles=tiles)
        else:
            plan.set_values()
        with pytest.raises(S.SmatError) as e:
            plan.spmm(x, C, check=True)
        assert e.value.code == -6
        for right, ref, mag in ((x, ref16, mag16), (B, ref4, mag4)):
            C.fill_(float("nan"))
            plan.spmm(right, C, check=True)  # reported once
            assert bool((C[16:32] == 0).all())
            for lo in (0, 32):
                _close(C[lo:lo + 16], ref[lo:lo + 16], mag[lo:lo + 16], 16)
        c.A.scales.copy_(good)
        plan.set_values()
        for right, ref, mag in ((x, ref16, mag16), (B, ref4, mag4)):
            plan.spmm(right, C, check=True)
            _close(C, ref, mag, 16)


def test_pairs_that_are_not_stored_together():
    """One block of a pair alone, and neighbours of different pairs or block-rows, may have any scales."""
    rowptr, colidx = np.array([0, 3, 5], np.int32), np.array([16, 32, 80, 64, 112], np.int32)
    rng = np.random.default_rng(2)
    codes, scales = rng.integers(0, 16, (5, 16, 16)).astype(np.uint8), np.repeat(np.arange(120, 125, dtype=np.uint8)[:, None], 16, 1)
    A = S.Fp4SparseMatrix.from_codes(32, 128, rowptr, colidx, F.pack(codes), scales, "mxfp4")
    x = torch.from_numpy(rng.standard_normal((3, 128))).half().cuda()
    C = torch.empty((32, 3), dtype=torch.float16, device="cuda")
    S.Fp4Plan(A).spmm(x, C, check=True)
    _close(C, *F.multiply(F.block_values(codes, scales, None, rowptr, "mxfp4"), rowptr, colidx, x.double().cpu().numpy()), 3)


def test_plans_made_on_several_threads():
    """Layers of very different K: the shared memory that one creation asks for does not bound another's."""
    Ks = [16 * 16, 16 * 512 * 64, 16 * 16 * 512 * 256 - 16]
    made = []
    for K in Ks:
        rowptr, colidx = np.array([0, 8], np.int32), np.arange(8, dtype=np.int32) * 16
        made.append(S.Fp4SparseMatrix.from_codes(16, K, rowptr, colidx, np.full((8, 16, 8), 0x22, np.uint8), np.full((8, 16), 56, np.uint8)))
    errors = []

    def work(A, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(300):
                    S.Fp4Plan(A).close()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(A, torch.cuda.Stream())) for A in made * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_builders_on_several_threads():
    """The same for the builder of the blocks."""
    errors = []

    def work(K, stream):
        try:
            rowptr, colidx = np.arange(17, dtype=np.int32), np.arange(16, dtype=np.int32) * (K // 16)
            with torch.cuda.stream(stream):
                for _ in range(100):
                    assert S.SparseMatrix.from_csr(16, K, rowptr, colidx, np.ones(16, np.float16)).nnzb > 0
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(K, torch.cuda.Stream())) for K in (256, 16 * 30000, 16 * 700000) * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_an_error_does_not_outlive_its_call():
    """A plan whose tiles do not fit the device (193 GB for blocks in scattered ranges of columns) is refused, and what is asked for next
    on the thread, the same plan without tiles, is made."""
    torch.cuda.empty_cache()
    steps, groups = 1 << 18, 20  # ranges of 256 columns, groups of 16 block-rows; four blocks in each
    K = steps * 256 - 256
    per_row = (steps - 1) // 4
    n = groups * 16 * per_row
    rowptr = torch.arange(groups * 16 + 1, device="cuda", dtype=torch.int32) * per_row
    row = torch.arange(per_row, device="cuda", dtype=torch.int32)
    # block-row e of a group has blocks in the ranges e / 4 modulo 4, so that four of them meet in every one
    colidx = torch.stack([(row * 4 + e // 4) * 256 + e % 4 * 16 for e in range(16)]).reshape(-1).repeat(groups)
    A = S.Fp4SparseMatrix.from_codes(groups * 256, K, rowptr, colidx, torch.full((n, 16, 8), 0x22, dtype=torch.uint8, device="cuda"),
                                     torch.full((n, 16), 56, dtype=torch.uint8, device="cuda"))
    with pytest.raises(S.SmatError) as e:
        S.Fp4Plan(A)
    assert e.value.code == -2
    plan = S.Fp4Plan(A, tiles=False)
    x = torch.ones((1, K), dtype=torch.float16, device="cuda")
    C = torch.empty((groups * 256, 1), dtype=torch.float16, device="cuda")
    x *= 2.0 ** -12
    plan.spmm(x, C, check=True)
    assert bool((C == 256).all())  # 16 * 65535 * 2^-12, rounded to fp16


@pytest.mark.parametrize("rows,n", [(3, 5), (16385, 1 << 20)])
def test_row_pointers_that_run_to_and_fro(rows, n):
    """Block-rows over the same blocks again and again: more blocks in all than are stored, up to more than 32 bits count."""
    K = n * 16
    rowptr = (torch.arange(rows + 1, device="cuda", dtype=torch.int32) % 2 * n).int()
    colidx = torch.arange(n, device="cuda", dtype=torch.int32) * 16
    A = S.Fp4SparseMatrix.from_codes(rows * 16, K, rowptr, colidx, torch.full((n, 16, 8), 0x22, dtype=torch.uint8, device="cuda"),
                                     torch.full((n, 16), 56, dtype=torch.uint8, device="cuda"))
    x = torch.ones((3, K), dtype=torch.float16, device="cuda")
    C = torch.full((rows * 16, 3), float("nan"), dtype=torch.float16, device="cuda")
    plan = S.Fp4Plan(A)
    with pytest.raises(S.SmatError) as e:
        plan.spmm(x, C, check=True)
    assert e.value.code == -6 and bool((C == 0).all())
    C.fill_(float("nan"))
    plan.spmm(S.Fp4Matrix.quantize(x), C, check=True)
    assert bool((C == 0).all())


def test_sparse_matrix_whose_arrays_do_not_fit():
    rowptr, colidx = np.array([0, 2, 3], np.int32), np.array([0, 32, 16], np.int32)
    for name, spoil in (("bcsrVal", lambda t: t[:512]), ("bcsrVal", lambda t: torch.cat([t, t])[::2]), ("bcsrRowPtr", lambda t: t[:2]),
                        ("bcsrRowPtr", lambda t: t.long()), ("bcsrColIdx", lambda t: t[:2]), ("bcsrColIdx", lambda t: t.cpu())):
        A = S.SparseMatrix.from_bcsr(32, 48, rowptr, colidx, np.ones(768, np.float16))
        setattr(A, name, spoil(getattr(A, name)))
        with pytest.raises(S.SmatError) as e:
            S.Fp4SparseMatrix.quantize(A)
        assert e.value.code == -1
    A = S.SparseMatrix.from_bcsr(32, 48, rowptr, colidx, np.ones(768, np.float16))
    A.bcsrVal = A.bcsrVal.bfloat16()  # other types of values are fine
    # row scale 2^-11 (1 / 2688 lies above 2^-12), group scale 2^11 / 6 = 341.3 -> 352, code 2^11 / 352 = 5.8 -> 6: 6 * 352 * 2^-11
    assert bool((S.Fp4SparseMatrix.quantize(A, check=True).dequantize().bcsrVal == 1.03125).all())


@pytest.mark.parametrize("N", [24, 64, 128, 264])
@pytest.mark.parametrize("counts", [[100] * 40, [9] * 40])
def test_waits_that_run_out(N, counts):
    """Codes that never arrive: the kernel with tiles gives up, alone and in pairs, reports it, and products after that are right."""
    c = Case(N, counts, 130, "nvfp4")
    B, b = c.acts4(N)
    plan, C = S.Fp4Plan(c.A), torch.empty((c.M, N), dtype=torch.float16, device="cuda")
    L = S.lib()
    call = L.smat_selftest_fp4_plan_wait_timeout
    call.argtypes = S.fp4._lib().smat_fp4_plan_spmm_fp4.argtypes
    codes, scales, row = B._at
    torch.cuda.synchronize()
    assert call(plan._h, codes, scales, row, 0, C.data_ptr(), 0, N, None) == 0
    assert L.smat_device_status(None) == -3 and b"site code 6" in L.smat_last_error_string()
    for _ in range(3):
        C.fill_(float("nan"))
        plan.spmm(B, C, check=True)
        _close(C, *F.multiply(c.vals, c.rowptr, c.colidx, b), c.longest)
    none = S.Fp4Plan(c.A, tiles=False)
    assert call(none._h, codes, scales, row, 0, C.data_ptr(), 0, N, None) == -1
