"""Products with both sides in 4 bits, wider than one CTA's tile: pairs of CTAs, several column tiles, cut and whole units, rows of C
that are stored 16 bytes at a time.  Reference and tolerance as in test_gpu_fp4_spmm."""
import pytest
import torch

import fp4_oracle as F
import smat_b200 as S
from test_gpu_fp4_spmm import Case, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("counts,Kb", [
    ([100] * 40, 130),                                        # three groups, long units: cut and joined
    ([9] * 21, 33),                                           # one group and a part of one
    ([16] * 3 + [0] * 40 + [13] * 10 + [0] * 30, 16),         # groups without a block
    ([5] * 300, 48),                                          # more units than pairs: whole ones
])
@pytest.mark.parametrize("N", [136, 256, 264, 520, 1000])
def test_pairs(fmt, counts, Kb, N):
    c = Case(N + Kb, counts, Kb, fmt)
    B, b = c.acts4(N)
    ref, mag = F.multiply(c.vals, c.rowptr, c.colidx, b)
    plan = S.Fp4Plan(c.A)
    for dtype in (torch.float16, torch.bfloat16):
        C = torch.full((c.M, N), float("nan"), dtype=dtype, device="cuda")
        plan.spmm(B, C, check=True)
        _close(C, ref, mag, c.longest)
    again = torch.empty_like(C)
    for _ in range(20):
        plan.spmm(B, again)
        assert torch.equal(C, again)
