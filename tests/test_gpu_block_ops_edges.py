"""RMS norm, linear with activation and differential attention at the ends of the numbers' range (-m gpu), against plain implementations in 64 bits.

Bounds: those of test_gpu_block_ops (U32 = 2^-24 is one fp32 rounding, u(t) one rounding to t, tiny(t) half the type's smallest number) unless a test derives its own."""
import pytest
import torch

from tests.test_gpu_block_ops import BF16, F16, F32, check_norm, gen, ops  # noqa: F401

pytestmark = pytest.mark.gpu

NORM_WIDTHS = [5, 64, 640, 1277, 2560, 10007, 12000]          # 16, 64 and 256 threads to a row, aligned and not, and the one-row form


# ------------------------------------------------------------------------------------------------------------- rmsnorm
@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
@pytest.mark.parametrize("xt,rt", [(F16, None), (BF16, BF16), (F32, None), (BF16, F32), (F32, F32)], ids=str)
def test_rmsnorm_rows_of_zeros_without_eps(ops, xt, rt, f8):
    """eps = 0: a row of zeros stays zeros (e4m3: with scale 0), the rows beside it are as ever."""
    for i, ch in enumerate(NORM_WIDTHS):
        randn = gen(900 + i)
        x, r = randn(6, ch).to(xt), randn(6, ch).to(rt) if rt is not None else None
        gamma = 1 + randn(ch, scale=0.1) if i % 2 else None
        for t in (x, r):
            if t is not None:
                t[1], t[4] = 0, 0
        got = ops.rmsnorm(x, gamma, eps=0.0, residual=r, f8=f8)
        got = list(got) if isinstance(got, tuple) else [got]
        for g in got:
            assert g[1].float().eq(0).all() and g[4].float().eq(0).all(), ch
        rest = [0, 2, 3, 5]
        check_norm(f"rmsnorm eps 0 {ch} {xt} {rt}", tuple(g[rest] for g in got), x[rest], r[rest] if r is not None else None, gamma, 0.0, f8)


@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_rmsnorm_rows_whose_squares_leave_fp32(ops, eps, f8):
    """Rows of 1e-38 to 1e37, and one with values of both ends: the result is the formula's, within the bounds of any row."""
    for i, ch in enumerate(NORM_WIDTHS):
        for xt, rt in ((F32, None), (BF16, None), (F32, F32), (BF16, F32)):
            randn = gen(920 + i)
            size = torch.tensor([1e-38, 1e-30, 1e-25, 1e-20, 1.0, 1e18, 1e20, 1e30, 1e37], device="cuda")[:, None]
            x = (randn(9, ch).clamp(-8, 8) * size).to(xt)
            x[4, 0], x[4, 1] = 1e30, 1e-30
            r = (randn(9, ch).clamp(-8, 8) * size).to(rt) if rt is not None else None
            gamma = 1 + randn(ch, scale=0.1) if i % 2 else None
            check_norm(f"rmsnorm squares out of range {ch} {xt} {rt}", ops.rmsnorm(x, gamma, eps=eps, residual=r, f8=f8), x, r, gamma, eps, f8)
