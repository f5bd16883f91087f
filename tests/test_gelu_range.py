"""CPU suite: the erf-GELU of svd_common.h outside [-7, 7], where t = |x| is held at 7: the sequence in float32 against x Phi(x), to both ends of float32."""
import os
import re

import numpy as np
from scipy.special import erfc

from tests.test_gelu_formula import ROOT, _kernel_coefficients


def _sources():
    return [open(os.path.join(ROOT, "streamingt2v_amd", "csrc", f)).read() for f in ("svd_common.h", "ff_fused.hip")]


def test_every_form_multiplies_with_the_held_argument():
    """One scalar form, one on pairs, two spelled out in the fused feed-forward: the last step is max(x, 0) - t q with the held t, and t keeps a NaN (or the comparison does)."""
    common, fused = _sources()
    assert "return fmaf(-t, q, x < 0.0f ? 0.0f : x);" in common and "return __builtin_elementwise_fma(-t, q, mx);" in common
    assert fused.count("__builtin_elementwise_fma(-gt, gq, gmx)") == 2
    assert not re.search(r'asm\("v_min_f32|fabsf\(x\), q|-ax', common + fused)
    assert len(re.findall(r'asm\("v_minimum3_f32 %0, \|%1\|, %2, %2"', common)) == 2 and len(re.findall(r'asm\("v_minimum3_f32 %0, \|%1\|, %2, %2"', fused)) == 4


def test_gelu_over_the_whole_range():
    c = np.array(_kernel_coefficients(), dtype=np.float32)
    far = np.logspace(0, 38.5, 200_001)
    x = np.concatenate([np.linspace(-12, 12, 2_000_001), far, -far]).astype(np.float32)
    t = np.minimum(np.abs(x), np.float32(7.0))
    r = c[0] * t + c[1]
    for k in range(2, 6):
        r = r * t + c[k]
    q = np.exp2((r * t - np.float32(1.0)).astype(np.float32)).astype(np.float32)
    got = (np.where(x < 0, np.float32(0), x).astype(np.float64) - t.astype(np.float64) * q).astype(np.float32)          # one rounding, as the fma does
    xd = x.astype(np.float64)
    want = 0.5 * xd * erfc(-xd / np.sqrt(2.0))
    err = np.abs(got - want)
    assert (err <= 4e-6 + 2.0 ** -24 * np.abs(want)).all(), err.max()          # (every multiplication above is rounded, which an fma does not do: twice the kernel's 2e-6)
    assert np.abs(got[xd < -7]).max() <= 1e-11
