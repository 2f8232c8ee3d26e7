"""Shaped attention at its edges, as far as that goes without a GPU."""
import os
import re

import numpy as np
import pytest

from smcsd_b200.ops import native as K
from smcsd_b200.ops import native_shaped as N

needs_library = pytest.mark.skipif(not os.path.exists(os.path.join(os.path.dirname(K.__file__), "libsmcsd_b200.so")), reason="kernel library not built")


@needs_library
@pytest.mark.parametrize("scale,cap", [(0.125, 1e-42), (0.125, 3e38), (0.125, 1e38), (1e30, 1e-10), (3e38, 0.0), (1e-40, 0.0), (1e-30, 1e9), (0.0, 5.0), (float("inf"), 5.0), (0.125, float("nan"))])
def test_scales_and_caps_outside_of_fp32_are_refused_ahead_of_any_launch(scale, cap):
    """scale log2(e), scale / cap or cap log2(e) is not a normal fp32 number."""
    L, p = N._library(), 1 << 20
    assert L.smc_shaped_prompt(p, 512, p, p, 7, p, 8, 1, None, 0, p, 1, p, 512, None, 4, 8, 2, 64, scale, cap, None, None, p, 0, None) == -143
    assert L.smc_shaped_mass(p, 512, p, 7, p, 8, 1, None, 0, p, 1, p, p, 8, 4, 8, 2, 64, scale, cap, None, None, p, 0, None) == -162
    assert L.smc_shaped_step(p, 512, p, p, 7, p, 8, 1, None, 0, p, p, p, 512, None, None, 8, 2, 1, 8, 2, 64, scale, cap, None, None, p, 1 << 30, p, 0, None) == -152


@needs_library
def test_pitches_are_refused_ahead_of_any_launch():
    """From row to row in the low 32 bits, columns above them: more columns than that, none at all, weights or positions of fewer."""
    L, p = N._library(), 1 << 20

    def calls(pitch, mass_stride=8, kp_stride=8):
        return (L.smc_shaped_prompt(p, 512, p, p, 7, p, pitch, 1, None, 0, p, 1, p, 512, None, 4, 8, 2, 64, 0.125, 0.0, None, None, p, 0, None),
                L.smc_shaped_mass(p, 512, p, 7, p, pitch, 1, None, 0, p, 1, p, p, mass_stride, 4, 8, 2, 64, 0.125, 0.0, None, None, p, 0, None),
                L.smc_shaped_step(p, 512, p, p, 7, p, pitch, 1, None, 0, p, p, p, 512, None, p, mass_stride, 2, 1, 8, 2, 64, 0.125, 0.0, None, None, p, 1 << 30, p, 0, None),
                L.smc_evict(p, pitch, p, kp_stride, p, mass_stride, p, 4, p, p, 3, 2, 8, 1, 1, p, p, p, p, 100, p, 1 << 20, p, None))
    for pitch in (0, -8, 8 | 9 << 32, 1 << 31, 1 << 40):
        assert calls(pitch) == (-142, -163, -153, -171), pitch
    assert calls(64 | 8 << 32, mass_stride=7)[1:] == (-163, -153, -171) and calls(64 | 8 << 32, kp_stride=7)[3] == -171


@needs_library
def test_pools_and_allocators_without_a_page_are_refused_ahead_of_any_launch():
    """Without its scratch page a pool has no page that a bad one could be replaced by, and no workspace belongs to an allocator of nothing."""
    L, p = N._library(), 1 << 20
    assert L.smc_shaped_prompt(p, 512, p, p, -1, p, 8, 1, None, 0, p, 1, p, 512, None, 4, 8, 2, 64, 0.125, 0.0, None, None, p, 0, None) == -142
    assert L.smc_shaped_mass(p, 512, p, -1, p, 8, 1, None, 0, p, 1, p, p, 8, 4, 8, 2, 64, 0.125, 0.0, None, None, p, 0, None) == -163
    assert L.smc_shaped_step(p, 512, p, p, -1, p, 8, 1, None, 0, p, p, p, 512, None, None, 8, 2, 1, 8, 2, 64, 0.125, 0.0, None, None, p, 1 << 30, p, 0, None) == -153
    for pages in (0, -5):
        assert L.smc_evict(p, 8, p, 8, p, 8, p, 4, p, p, 3, 2, 8, 1, 1, p, p, p, p, pages, p, 1 << 20, p, None) == -172
        with pytest.raises(ValueError, match="allocator"):
            N.evict_work_bytes(pages)


def test_polynomials_of_the_tanh_are_as_close_as_their_header_says():
    """Relative to tanh, over the reach of each, with the coefficients rounded to fp32 as the kernels have them."""
    text = open(os.path.join(os.path.dirname(K.__file__), "csrc", "shaped.cuh")).read()
    for n, reach, off in ((3, 0.35, 3.0e-6), (4, 0.35, 6.1e-8), (5, 0.75, 6.3e-7), (6, 0.625, 1.0e-8)):
        coef = [np.float64(np.float32(float(x.rstrip("f")))) for x in re.search(r"c%d\[%d\] = \{([^}]*)\}" % (n, n), text).group(1).split(",")]
        u = np.linspace(1e-4, reach, 400001)
        got = u * sum(c * u ** (2 * k) for k, c in enumerate(coef))
        worst = np.abs(got / np.tanh(u) - 1).max()
        assert len(coef) == n and 0.9 * off <= worst <= off, (n, worst)
