"""Products of a block-sparse matrix in 4 bits against the definition in 64 bits.

Tolerance.  Codes, scales and their products are exact; what is rounded are the fp32 additions, at most one for a block, one for
each of the 16 products inside it and a few for joining parts, each by less than 2^-22 of the sum of magnitudes (an addition in the
matrix unit may truncate), the two row scales (2^-24 each) and the result (half a step of its type, or of its smallest value)."""
import numpy as np
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _close(C, ref, mag, longest):
    got = C.double().cpu().numpy()
    tol = (longest + 32) * 2.0 ** -22 * mag + HALF[C.dtype] * np.abs(ref) * (1 + 1e-3) + LEAST[C.dtype]
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    # fp16 ends at 65504: a sum of at least 65504 + half a step = 65520 is infinite
    over = (np.abs(ref) + tol >= 65520.0) if C.dtype == torch.float16 else np.zeros(ref.shape, bool)
    assert np.all(np.where(over & np.isinf(got), np.sign(got) == np.sign(ref), np.isfinite(got) | ~np.isfinite(ref)))
    assert np.all(np.isinf(got[(np.abs(ref) - tol >= 65520.0)])) or C.dtype != torch.float16
    fine = np.isfinite(ref) & ~(over & np.isinf(got))
    assert np.all(np.abs(got - ref)[fine] <= tol[fine]), float(np.max((np.abs(got - ref) / tol)[fine]))


class Case:
    def __init__(self, seed, counts, Kb, fmt, row_scale=True):
        rng = self.rng = np.random.default_rng(seed)
        self.fmt, self.M, self.K = fmt, len(counts) * 16, Kb * 16
        self.rowptr, self.colidx = F.random_blocks(rng, counts, Kb)
        n = int(self.rowptr[-1])
        self.codes = rng.integers(0, 16, (n, 16, 16)).astype(np.uint8)
        if fmt == "nvfp4":
            self.scales = rng.integers(30, 90, (n, 16)).astype(np.uint8)
            self.p = (rng.random(self.M) + 0.5).astype(np.float32) if row_scale else None
        else:
            brow = np.repeat(np.arange(len(counts)), counts)
            table = rng.integers(120, 130, (len(counts), Kb // 2 + 1, 16)).astype(np.uint8)  # one for a pair of blocks
            self.scales, self.p = table[brow, self.colidx // 32], None
        self.longest = max(counts, default=0)
        self.A = S.Fp4SparseMatrix.from_codes(self.M, self.K, self.rowptr, self.colidx, F.pack(self.codes), self.scales, fmt, self.p)
        self.vals = F.block_values(self.codes, self.scales, self.p, self.rowptr, fmt)

    def acts(self, N, dtype):
        return torch.from_numpy(self.rng.standard_normal((N, self.K))).to(dtype).cuda()

    def acts4(self, N):
        codes = self.rng.integers(0, 16, (N, self.K)).astype(np.uint8)
        groups = -(-self.K // F.GROUP[self.fmt])
        s = self.rng.integers(30, 90, (N, groups)) if self.fmt == "nvfp4" else self.rng.integers(120, 130, (N, groups))
        s = s.astype(np.uint8)
        p = (self.rng.random(N) + 0.5).astype(np.float32) if self.fmt == "nvfp4" else None
        B = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(codes)), torch.from_numpy(s), self.K, self.fmt, p)
        return B, F.dense_values(codes, s, p, self.fmt)


SHAPES = [
    ([1], 1),                       # one block
    ([0, 0, 0], 5),                 # nothing stored
    ([3, 0, 17, 1, 40], 40),        # empty and full block-rows
    ([9] * 21, 33),                 # two groups of eight block-rows and a part of one
    ([700, 0, 650], 701),           # long block-rows
]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,Kb", SHAPES)
@pytest.mark.parametrize("N", [1, 7, 8, 13, 32, 67, 130])
def test_16bit(fmt, dtype, counts, Kb, N):
    c = Case(N + Kb, counts, Kb, fmt)
    x = c.acts(N, dtype)
    C = torch.full((c.M, N), float("nan"), dtype=dtype, device="cuda")
    plan = S.Fp4Plan(c.A)
    plan.spmm(x, C, check=True)
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, x.double().cpu().numpy())
    _close(C, ref, mag, c.longest)
    again = torch.empty_like(C)
    plan.spmm(x, again)
    assert torch.equal(C, again)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,Kb", SHAPES + [([100] * 40, 130), ([16] * 3 + [0] * 40 + [13] * 10 + [0] * 30, 16), ([0] * 9 + [12], 12), ([5] * 300, 48)])
@pytest.mark.parametrize("N", [1, 8, 9, 31, 64, 106, 128, 129, 191, 300])
def test_4bit(fmt, dtype, counts, Kb, N):
    c = Case(N + Kb, counts, Kb, fmt)
    B, b = c.acts4(N)
    C = torch.full((c.M, N), float("nan"), dtype=dtype, device="cuda")
    plan = S.Fp4Plan(c.A)
    plan.spmm(B, C, check=True)
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, b)
    _close(C, ref, mag, c.longest)
    again = torch.empty_like(C)
    plan.spmm(B, again)
    assert torch.equal(C, again)


@pytest.mark.parametrize("four", [False, True])
def test_no_row_scales_and_block_row_ranges(four):
    c = Case(5, [4, 0, 30, 12, 7, 1, 9, 22, 30, 3, 2], 31, "nvfp4", row_scale=False)
    N = 24
    if four:
        B, b = c.acts4(N)
        B.row_scale, b = None, b / B.row_scale.double().cpu().numpy()[:, None]
    else:
        B = c.acts(N, torch.float16)
        b = B.double().cpu().numpy()
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, b)
    for lo, hi in [(0, 11), (3, 9), (10, 11), (4, 4)]:
        C = torch.full(((hi - lo) * 16, N), float("nan"), dtype=torch.float16, device="cuda")
        S.Fp4Plan(c.A, lo, hi).spmm(B, C, check=True)
        _close(C, ref[lo * 16:hi * 16], mag[lo * 16:hi * 16], c.longest)


def test_nan_of_16bit_activations_stays_where_blocks_are():
    """A column of B that no stored block meets may hold anything."""
    c = Case(6, [5, 0, 3, 8], 20, "mxfp4")
    x = c.acts(9, torch.float16)
    meets = np.zeros(20, bool)
    meets[c.colidx // 16] = True
    free = np.flatnonzero(~meets)
    assert len(free)
    x.view(9, 20, 16)[:, torch.from_numpy(free).cuda()] = float("nan")
    x[3, int(c.colidx[-1])] = float("inf")
    C = torch.empty((c.M, 9), dtype=torch.float16, device="cuda")
    S.Fp4Plan(c.A).spmm(x, C, check=True)
    xs = x.double().cpu().numpy()
    assert bool(torch.isfinite(C[:16]).all()) and bool((C[16:32] == 0).all())
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, xs)
    got = C.double().cpu().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(ref))


@pytest.mark.parametrize("four", [False, True])
def test_scale_nan_of_a_row_makes_nan(four):
    c = Case(7, [6, 6], 12, "nvfp4")
    c.A.scales[2, 5] = 0x7F
    B = c.acts4(40)[0] if four else c.acts(40, torch.bfloat16)
    C = torch.empty((32, 40), dtype=torch.bfloat16, device="cuda")
    S.Fp4Plan(c.A).spmm(B, C, check=True)
    bad = torch.isnan(C).all(1).cpu().numpy()
    assert bad[5] and bad.sum() == 1 and not bool(torch.isnan(C[:5]).any())


@pytest.mark.parametrize("kind", ["f16", "bf16", "4bit", "4bit, no tiles"])
def test_scales_from_end_to_end(kind):
    """mxfp4 scales over the whole of their range: each row of A has its own, activations bring the products back to ordinary size."""
    rng = np.random.default_rng(12)
    n = 40  # blocks of each of two block-rows, side by side
    bytes_of_row = np.array([0, 1, 2, 3, 10, 20, 40, 60, 80, 100, 127, 150, 180, 220, 240, 250])
    rowptr, colidx = np.array([0, n, 2 * n], np.int32), np.tile(np.arange(n, dtype=np.int32) * 16, 2)
    codes = rng.integers(0, 16, (2 * n, 16, 16)).astype(np.uint8)
    scales = np.tile(bytes_of_row.astype(np.uint8), (2 * n, 1))
    A = S.Fp4SparseMatrix.from_codes(32, n * 16, rowptr, colidx, F.pack(codes), scales, "mxfp4")
    vals = F.block_values(codes, scales, None, rowptr, "mxfp4")
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    tokens = np.arange(-100, 101, 50) if kind != "f16" else np.arange(-12, 13, 6)  # token t is of size 2^t
    if kind[0] == "4":
        bc = rng.integers(0, 16, (len(tokens), n * 16)).astype(np.uint8)
        bs = np.repeat((tokens + 127).astype(np.uint8)[:, None], n // 2, 1)
        B = S.Fp4Matrix.from_codes(torch.from_numpy(F.pack(bc)), torch.from_numpy(bs), n * 16, "mxfp4")
        b = F.dense_values(bc, bs, None, "mxfp4")
    else:
        B = torch.from_numpy(rng.standard_normal((len(tokens), n * 16)) * 2.0 ** tokens[:, None]).to(dtype).cuda()
        b = B.double().cpu().numpy()
    C = torch.empty((32, len(tokens)), dtype=dtype, device="cuda")
    S.Fp4Plan(A, tiles=kind != "4bit, no tiles").spmm(B, C, check=True)
    ref, mag = F.multiply(vals, rowptr, colidx, b)
    # what fp32 and the type of C hold: neither overflows nor loses digits below the normal numbers
    top = 2.0 ** 14 if kind == "f16" else 2.0 ** 120
    fine = (mag < top) & (mag > (2.0 ** -10 if kind == "f16" else 2.0 ** -100))
    assert fine.sum() >= (6 if kind == "f16" else 60)  # f16: scale 127 with tokens -12, -6, 0, scale 100 with token 12
    got = C.double().cpu().numpy()
    tol = (n + 32) * 2.0 ** -22 * mag + HALF[dtype] * np.abs(ref) * (1 + 1e-3) + LEAST[dtype]
    assert np.all(np.abs(got - ref)[fine] <= tol[fine]), np.max((np.abs(got - ref) / tol)[fine])


@pytest.mark.parametrize("four", [False, True])
def test_values_change(four):
    c = Case(8, [5, 9, 2], 11, "nvfp4")
    plan = S.Fp4Plan(c.A)
    x = c.acts4(5)[0] if four else c.acts(5, torch.float16)
    C, D = (torch.empty((c.M, 5), dtype=torch.float16, device="cuda") for _ in range(2))
    plan.spmm(x, C)
    c.A.codes ^= 0x88  # all signs
    plan.set_values()
    plan.spmm(x, D)
    assert torch.equal(C, -D)


@pytest.mark.parametrize("N", [1, 9, 40, 130])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_4bit_without_tiles(N, fmt):
    """Plans made without tiles, and those of scattered blocks, which have none either."""
    for counts, Kb, tiles in [([3, 0, 17, 1, 40], 40, False), ([2] * 40, 2000, True)]:
        c = Case(N, counts, Kb, fmt)
        B, b = c.acts4(N)
        C = torch.full((c.M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
        S.Fp4Plan(c.A, tiles=tiles).spmm(B, C, check=True)
        _close(C, *F.multiply(c.vals, c.rowptr, c.colidx, b), c.longest)


@pytest.mark.parametrize("four", [False, True])
def test_streams_and_graphs(four):
    """Products of one plan on two streams at a time, and captured twice; the graphs replay side by side."""
    c = Case(9, [90] * 40, 300, "nvfp4")
    Ns = (33, 150)
    Bs = [c.acts4(N)[0] if four else c.acts(N, torch.bfloat16) for N in Ns]
    plan = S.Fp4Plan(c.A)
    want = [torch.empty((c.M, N), dtype=torch.bfloat16, device="cuda") for N in Ns]
    for B, C in zip(Bs, want):
        plan.spmm(B, C, check=True)
    got = [torch.empty_like(C) for C in want]
    streams = [torch.cuda.Stream() for _ in Ns]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, B, C in zip(streams, Bs, got):
            with torch.cuda.stream(s):
                plan.spmm(B, C)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = [torch.cuda.CUDAGraph() for _ in Ns]
    for gph, B, C in zip(graphs, Bs, got):
        with torch.cuda.graph(gph):
            plan.spmm(B, C)
            plan.spmm(B, C)
    for C in got:
        C.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, gph in zip(streams, graphs):
            with torch.cuda.stream(s):
                gph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inconsistent_arrays_are_reported_and_left_out():
    c = Case(10, [4, 4, 4], 16, "nvfp4")
    x = c.acts(8, torch.float16)
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, x.double().cpu().numpy())
    for spoil in ("outside", "order", "unaligned"):
        ci = c.colidx.copy()
        if spoil == "outside":
            ci[7] = 16 * 16
        elif spoil == "order":
            ci[[5, 6]] = ci[[6, 5]]
        else:
            ci[5] += 8
        A = S.Fp4SparseMatrix.from_codes(c.M, c.K, c.rowptr, ci, F.pack(c.codes), c.scales, "nvfp4", c.p)
        plan = S.Fp4Plan(A)
        C = torch.full((c.M, 8), float("nan"), dtype=torch.float16, device="cuda")
        with pytest.raises(S.SmatError) as e:
            plan.spmm(x, C, check=True)
        assert e.value.code == -6
        assert bool((C[16:32] == 0).all())
        for lo in (0, 32):
            _close(C[lo:lo + 16], ref[lo:lo + 16], mag[lo:lo + 16], 4)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_nothing_stored(fmt):
    """A matrix without blocks goes all the way; its products are zeros, whatever B holds."""
    A = S.SparseMatrix.from_bcsr(64, 96, np.zeros(5, np.int32), np.zeros(0, np.int32), np.zeros(0, np.float16))
    A4 = S.Fp4SparseMatrix.quantize(A, fmt, check=True)
    assert A4.dequantize(check=True).nnzb == 0
    plan = S.Fp4Plan(A4)
    plan.set_values()
    x = torch.full((5, 96), float("nan"), dtype=torch.float16, device="cuda")
    for B in (x, S.Fp4Matrix.quantize(x, fmt)):
        C = torch.full((64, 5), float("nan"), dtype=torch.float16, device="cuda")
        plan.spmm(B, C, check=True)
        assert bool((C == 0).all())
    plan.spmm(x[:0], torch.empty((64, 0), dtype=torch.float16, device="cuda"), check=True)
    assert S.Fp4Matrix.quantize(x[:0], fmt).dequantize().shape == (0, 96)


@pytest.mark.parametrize("N", [40, 300])
def test_long_and_short_groups(N):
    """Groups of block-rows of very different lengths: their tiles of C are dealt out in ranges, and cut."""
    rng = np.random.default_rng(13)
    Kb, rows = 1600, 16 * 90
    cols = [np.sort(rng.choice(Kb, 500, replace=False)) if r // 16 in (3, 40) else np.arange(r % 7, r % 7 + 16) for r in range(rows)]
    rowptr = np.zeros(rows + 1, np.int32)
    rowptr[1:] = np.cumsum([len(c) for c in cols])
    colidx = np.concatenate(cols).astype(np.int32) * 16
    n = int(rowptr[-1])
    codes, scales = rng.integers(0, 16, (n, 16, 16)).astype(np.uint8), rng.integers(30, 60, (n, 16)).astype(np.uint8)
    A = S.Fp4SparseMatrix.from_codes(rows * 16, Kb * 16, rowptr, colidx, F.pack(codes), scales)
    vals = F.block_values(codes, scales, None, rowptr, "nvfp4")
    x = torch.from_numpy(rng.standard_normal((N, Kb * 16))).half().cuda()
    B = S.Fp4Matrix.quantize(x)
    C = torch.empty((rows * 16, N), dtype=torch.bfloat16, device="cuda")
    S.Fp4Plan(A).spmm(B, C, check=True)
    _close(C, *F.multiply(vals, rowptr, colidx, B.dequantize(torch.float32).double().cpu().numpy()), 500)


def test_arrays_that_were_replaced():
    """A plan keeps the arrays that it was made of: those that replace them in A are not its own, and the old ones stay alive."""
    A = S.SparseMatrix.from_bcsr(32, 64, np.array([0, 2, 4], np.int32), np.array([0, 32, 16, 48], np.int32),
                                 np.random.default_rng(3).standard_normal(1024).astype(np.float16))
    A4 = S.Fp4SparseMatrix.quantize(A)
    plan = S.Fp4Plan(A4)
    x = torch.randn((4, 64), dtype=torch.float16, device="cuda")
    before, after = (torch.empty((32, 4), dtype=torch.float16, device="cuda") for _ in range(2))
    plan.spmm(x, before)
    A4.row_scale = torch.zeros_like(A4.row_scale)
    junk = [torch.zeros(32, dtype=torch.float32, device="cuda") for _ in range(64)]  # would take a freed array's place
    plan.spmm(x, after)
    assert torch.equal(before, after) and bool((before != 0).any())
    with pytest.raises(S.SmatError, match="other arrays"):
        plan.set_values()
    del junk


def test_row_scales_given_are_copied():
    """Quantising into a matrix leaves the caller's row scales as they were."""
    x = torch.randn((5, 64), dtype=torch.float16, device="cuda") * 100
    given = torch.full((5,), 0.75, dtype=torch.float32, device="cuda")
    B = S.Fp4Matrix.quantize(x)
    codes, scales, own = B.codes[:, :32].clone(), B.group_scales(), B.row_scale.clone()
    B.row_scale = given
    assert torch.equal(B.row_scale, given)
    assert torch.equal(B.dequantize(torch.float32), S.Fp4Matrix.from_codes(codes, scales, 64, row_scale=given).dequantize(torch.float32))
    S.Fp4Matrix.quantize(x, out=B)
    assert bool((given == 0.75).all()) and torch.equal(B.row_scale, own)
    B.row_scale = None
    assert B.row_scale is None
    with pytest.raises(S.SmatError, match="no row scales"):
        S.Fp4Matrix.quantize(x, out=B)


def test_as_a_program_runs_them():
    """A layer in fp16 goes to 4 bits, decodes with 16-bit activations and prefills with 4-bit ones; both agree with the matrix that
    the codes stand for, multiplied by the framework's fp16 product."""
    rng = np.random.default_rng(11)
    rowptr, colidx = F.random_blocks(rng, rng.integers(0, 60, 24), 60)
    vals = (rng.standard_normal((rowptr[-1], 16, 16)) * 0.05).astype(np.float16)
    A = S.SparseMatrix.from_bcsr(24 * 16, 960, rowptr, colidx, vals.reshape(-1))
    for fmt in ("nvfp4", "mxfp4"):
        A4 = S.Fp4SparseMatrix.quantize(A, fmt, check=True)
        plan, back = S.Fp4Plan(A4), A4.dequantize()
        for N in (8, 40, 136):
            x = torch.randn((N, 960), device="cuda").half()
            got, want = (torch.empty((384, N), dtype=torch.float16, device="cuda") for _ in range(2))
            plan.spmm(x, got, check=True)
            S.spmm(back, x, want, check=True)
            _, mag = F.multiply(F.block_values(*F.quantize_blocks(vals, rowptr, colidx, fmt), rowptr, fmt), rowptr, colidx, x.double().cpu().numpy())
            tol = 2 * (2.0 ** -11 * want.double().abs().cpu().numpy() * 1.01 + 100 * 2.0 ** -22 * mag + 2.0 ** -25)
            # values below fp16's normal numbers are rounded on the way back
            tol = tol + 2.0 ** -25 * x.double().abs().sum(1).cpu().numpy()[None]
            assert np.all(np.abs((got.double() - want.double()).cpu().numpy()) <= tol)
            q = S.Fp4Matrix.quantize(x, fmt)
            plan.spmm(q, got, check=True)
            S.spmm(back, q.dequantize(torch.float16), want, check=True)
            assert np.all(np.abs((got.double() - want.double()).cpu().numpy()) <= 1.3 * tol + 1e-3)
