"""The YaRN frequencies, every pair against the ramp written out with exact pair turns."""
from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest

from qwen_mla_vllm_b200.rotary import rotary_frequencies


def yarn(rot, base, n, factor, fast, slow):
    """The published blend: pair i keeps 1 - r of its frequency and takes r of the interpolated one, r
    rising linearly over the pair index from the pair that makes `fast` turns in n positions (rounded down)
    to the one that makes `slow` (rounded up); both ends within [0, rot - 1]."""
    i = np.arange(rot // 2, dtype=np.longdouble)
    w = np.longdouble(base) ** (-2 * i / rot)
    # n * base^(-2 x / rot) / (2 pi) = turns, solved for x by bisection (no logarithm shared with the code)
    def at(turns):
        lo, hi = np.longdouble(-1000), np.longdouble(1000)
        for _ in range(200):
            mid = (lo + hi) / 2
            if n * np.longdouble(base) ** (-2 * mid / rot) / (2 * np.longdouble(np.pi)) > turns:
                lo = mid
            else:
                hi = mid
        return float(lo)

    a, b = max(int(np.floor(at(fast))), 0), min(int(np.ceil(at(slow))), rot - 1)
    r = [float(min(max(Fraction(k - a, max(b - a, 1)) if b > a else Fraction(int(k > a)), 0), 1)) for k in range(rot // 2)]
    return [float(x * (1 - y) + x * y / factor) for x, y in zip(w, r)], b


CASES = [(64, 1e4, 4096), (64, 1e6, 262144), (128, 5e5, 8192), (58, 1e7, 262144),
         (64, 1e4, 131072), (58, 1e4, 65536), (32, 1e4, 131072), (58, 1e6, 8388608),
         (64, 1e4, 1 << 30)]  # the last: even the end of the ramp is clamped


def test_the_cases_lie_on_both_sides():
    """The ramp ends within the pairs, or past them: the slowest pair then makes more than `slow` turns."""
    past = [yarn(rot, base, n, 4.0, 32.0, 1.0)[1] > rot // 2 - 1 for rot, base, n in CASES]
    assert past == [False] * 4 + [True] * 5


@pytest.mark.parametrize("rot,base,n", CASES)
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (16.0, 2.0)])
def test_every_pair(rot, base, n, fast, slow):
    want, _ = yarn(rot, base, n, 4.0, fast, slow)
    got, _ = rotary_frequencies(rot, base, {"type": "yarn", "factor": 4.0, "original_max_position": n, "beta_fast": fast,
                                            "beta_slow": slow})
    assert got == pytest.approx(want, rel=1e-12)
