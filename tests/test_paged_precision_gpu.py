"""How near paged attention comes to 64 bits (measures and limits:
paged_precision.py)."""
import numpy as np
import pytest

import paged_precision as P
import paged_ref as R
from helpers import rng

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def attend(c, q, scale, dtype, mask=None):
    import b200_decode as bw

    dk, dv = R.to_device(c, dtype)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    out = bw.paged_attn(bw.PagedKV(dk, dv), dev(q), dev(c["table"]), dev(c["lens"]), scale, mask=mask)
    assert bw.device_status(reset=True) == 0
    return out.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", P.CASES, ids=str)
def test_random_inputs(case, dtype, masked):
    """With a mask of zeros too, which takes the other variant."""
    c, q = P.inputs(rng(case[0][0]), *case, dtype)
    scale = case[-1] ** -0.5
    mask = torch.zeros((len(q), c["table"].shape[1] * case[1]), dtype=torch.float16, device="cuda") if masked else None
    off = P.off(attend(c, q, scale, dtype, mask), P.attend(c, q, case[1], scale))
    print(f"worst head {off.max():.2e}, limit {P.LIMIT:.2e}")
    assert off.max() <= P.LIMIT


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("a", [1.0, 8.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", P.ONE_SHAPES)
def test_one_channel(hq, hkv, d, dtype, a, masked):
    c, q, scale, want, limit = P.one_channel(rng(hq + d), hq, hkv, d, dtype, a)
    mask = torch.zeros((d, 16), dtype=torch.float16, device="cuda") if masked else None
    err = np.abs(attend(c, q, scale, dtype, mask) - want) / limit
    print(f"worst {err.max():.2f} of the limit")
    assert np.isfinite(err).all() and err.max() <= 1.0
