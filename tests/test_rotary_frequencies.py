"""The frequencies of rotary positions (host arithmetic) against their formulas, and what is refused."""
import ctypes as C
import math

import numpy as np
import pytest

import om_binding as omb


def plain(n, base):
    return [base ** (-2.0 * j / n) for j in range(n // 2)]


@pytest.mark.parametrize("n,base", [(2, 10000.0), (64, 10000.0), (96, 500000.0), (256, 1.5)])
def test_scalings(n, base):
    rel = 1e-13   # a double power is within a few units of 2^-53 times its exponent's size
    assert np.allclose(omb.rotary_frequencies(n, base)[: n // 2], plain(n, base), rtol=rel, atol=0)
    assert np.allclose(omb.rotary_frequencies(n, base, "linear", 4.0)[: n // 2], [f / 4 for f in plain(n, base)], rtol=rel, atol=0)
    if n > 2:
        got = omb.rotary_frequencies(n, base, "base", 8.0)[: n // 2]
        assert np.allclose(got, plain(n, base * 8.0 ** (n / (n - 2))), rtol=rel, atol=0)
        assert math.isclose(got[-1] * 8.0, plain(n, base)[-1], rel_tol=1e-12) and got[0] == 1.0
    got = omb.rotary_frequencies(n, base, "parts", 16.0, 8192.0, 1.0, 32.0)[: n // 2]
    for f, want in zip(got, plain(n, base)):
        kept = min(1.0, max(0.0, (8192 * want / (2 * math.pi) - 1.0) / 31.0))
        assert math.isclose(f, want * ((1 - kept) / 16 + kept), rel_tol=1e-12)


@pytest.mark.parametrize("change,status", [(dict(columns=0), 1), (dict(columns=3), 1), (dict(columns=258), 1), (dict(base=1.0), 8), (dict(base=float("nan")), 8),
                                           (dict(scaling=4), 8), (dict(scaling=-1), 8), (dict(scaling=1, factor=0.5), 8), (dict(scaling=2, columns=2, factor=2.0), 1),
                                           (dict(scaling=3, original_context=0.0), 8), (dict(scaling=3, low_turns=4.0, high_turns=4.0), 8),
                                           (dict(scaling=2, base=1e300, factor=1e300), 8)])
def test_refusals(change, status):
    spec = omb.RotarySpec(**(dict(columns=8, scaling=0, base=10000.0, factor=2.0, original_context=100.0, low_turns=1.0, high_turns=2.0) | change))
    out = (C.c_double * 128)()
    assert omb.kernel_lib().om_rotary_frequencies(None, C.byref(spec), out) == status
    assert omb.kernel_lib().om_rotary_frequencies(None, None, out) == 8
