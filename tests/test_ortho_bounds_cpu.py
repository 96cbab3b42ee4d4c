"""The bounds that csrc/ortho.hip states for its iteration, by evaluating the polynomial (no kernel runs)."""
import numpy as np

from tests import _mx4_ref as ref


def test_the_stated_bounds():
    a, b, c = ref.NS
    p = lambda s: a * s + b * s ** 3 + c * s ** 5
    s = np.linspace(0.005, 1, 2000001)
    for _ in range(5):
        s = p(s)
    # (between two of the points p^5 moves by at most its slope, 3.4445^5 = 485, times half their distance, 2.5e-7: 1.2e-4)
    assert 0.68 + 1.2e-4 <= s.min() and s.max() <= 1.16 - 1.2e-4
    t = np.linspace(0, 1.21, 200001)
    assert p(t).max() <= 1.21 and 1.21 ** 2 <= 1.47 and np.abs(a + b * t ** 2 + c * t ** 4).max() <= 3.45
