"""The limits of paged_precision.py, on the host: the kernel's number formats
stay inside them, one 16-bit part less does not."""
import numpy as np
import pytest

import paged_precision as P
from helpers import rng


@pytest.mark.parametrize("case", P.CASES[:4] + P.CASES[5:6], ids=str)
def test_random_inputs_tell_f16_parts_apart(case):
    c, q = P.inputs(rng(case[0][0]), *case, "f16")
    scale = case[-1] ** -0.5
    want = P.attend(c, q, case[1], scale)
    assert P.off(P.attend(c, q, case[1], scale, "f16", 2, 2), want).max() < 0.2 * P.LIMIT
    for less in ((1, 2), (2, 1)):
        assert P.off(P.attend(c, q, case[1], scale, "f16", *less), want).min() > 5 * P.LIMIT, less


@pytest.mark.parametrize("a", [1.0, 8.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", P.ONE_SHAPES)
def test_one_channel_tells_every_part_apart(hq, hkv, d, dtype, a):
    c, q, scale, want, limit = P.one_channel(rng(hq + d), hq, hkv, d, dtype, a)
    np.testing.assert_allclose(P.attend(c, q, 16, scale), want, rtol=1e-12, atol=1e-15)
    n = P.PARTS[dtype]
    assert (np.abs(P.attend(c, q, 16, scale, dtype, n, n) - want) <= 0.5 * limit).all()
    less = (n - 1, n) if a > 2 else (n, n - 1)
    err = np.abs(P.attend(c, q, 16, scale, dtype, *less) - want)
    assert ((err / limit).max(-1) > 1.5).all(), (err / limit).max(-1).min()
