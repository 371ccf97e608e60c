"""Rows that paged_prefill computes again: those that meet pages out of range,
infinities or NaN, against 64 bits within the bound of chunk_ref.chunk_ref (such
rows are summed in at least as many bits as the others)."""
import numpy as np
import pytest

import paged_ref as R
from chunk_ref import chunk_ref

torch = pytest.importorskip("torch")
from test_paged_chunk_gpu import B, BOUNDS, _status_clean, i32, make, run  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# past, new, page size, heads, KV heads, head dim: one tile, units that ranges cut, many units to a range
SHAPES = [([64], [16], 16, 8, 2, 128), ([700, 0, 130], [50, 200, 1], 24, 12, 2, 64), ([300], [140], 16, 4, 2, 256),
          ([1500], [9], 5, 16, 4, 128), ([900, 0], [600, 1500], 64, 24, 8, 64), ([500], [1000], 32, 16, 4, 256)]


def left_out(c, ps, blocks):
    """The mask that stands for the blocks' positions being left out."""
    m = np.zeros((len(c["lens"]), c["table"].shape[1] * ps), np.float16)
    for s, b in blocks:
        m[s, b * ps:(b + 1) * ps] = -np.inf
    return m


@pytest.mark.parametrize("also", ["", "mask", "infinity", "window"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d", SHAPES)
def test_positions_on_pages_out_of_range_are_left_out(past, new, ps, hq, hkv, d, dtype, also):
    """One page in the middle and the newest block's of the first sequence.  Scores are
    negative, so a position that counted with a score of 0 would take all the weight."""
    r, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    q[:] = q.abs()
    c["k"] = -np.abs(c["k"])
    blocks = R.ceil_div(int(c["lens"][0]), ps)
    lost = [(0, blocks // 2), (0, blocks - 1)]
    m = left_out(c, ps, lost)
    mask, window = None, 0
    if also == "mask":
        mask = r.standard_normal(m.shape).astype(np.float16)
        mask[r.random(m.shape) < 0.2] = -np.inf
        m += mask
    elif also == "window":
        window = 3 * ps + 1
    want, tol = chunk_ref(c, q, cu, ps, d ** -0.5, m, window)
    rows = torch.arange(q.shape[0], device="cuda")
    if also == "infinity":  # the key or value of one token of the second sequence, or of the newest token
        s = len(past) - 1
        p = int(c["lens"][s]) - 1
        c["v"][c["table"][s, p // ps], p % ps, 0, 3] = np.inf
        rows = rows[rows != int(cu[s + 1]) - 1]  # the one row that sees it
    bad = dict(c, table=c["table"].copy())
    bad["table"][0, lost[0][1]], bad["table"][0, lost[1][1]] = c["k"].shape[0], -1
    out = run(bad, q, cu, dtype, d ** -0.5, mask, window)
    assert B().device_status(reset=True) == BOUNDS
    rows = rows[rows < int(cu[-1])]
    off = (out.double() - want).abs()[rows] - tol[rows]
    assert (off <= 0).all(), f"{(~(off <= 0)).sum().item()} of {off.numel()} off"


def test_only_pages_out_of_range():
    """No position is left: zeros."""
    _, c, cu, q = make([0, 40], [30, 3], 16, 8, 2, 128, "f16")
    c["table"][:] = 10**6
    out = run(c, q, cu, "f16", 0.1)
    assert B().device_status(reset=True) == BOUNDS
    assert (out[: int(cu[-1])] == 0).all()


@pytest.mark.parametrize("past,new,ps,hq,hkv,d", [([64], [16], 16, 8, 2, 128), ([3000, 0], [5, 200], 16, 12, 2, 64),
                                                  ([300], [140], 5, 4, 2, 256), ([0], [1], 16, 2, 2, 128)])
def test_values_near_the_largest(past, new, ps, hq, hkv, d):
    """bf16 values whose weighted sums pass the f32 range, but no mean does: all of one
    sign in half of the channels, of both in the others."""
    r, c, cu, q = make(past, new, ps, hq, hkv, d, "bf16")
    most = float(torch.finfo(torch.bfloat16).max)
    v = r.choice([most, most / 2, 0.75 * most], c["v"].shape) * r.choice([1, -1], c["v"].shape)
    v[..., ::2] = np.abs(v[..., ::2])
    c["v"] = np.where(np.isnan(c["v"]), np.nan, R.rounded(v, "bf16"))
    out = run(c, q, cu, "bf16", d ** -0.5)
    want, tol = chunk_ref(c, q, cu, ps, d ** -0.5)
    rows = slice(0, int(cu[-1]))
    assert torch.isfinite(out[rows].float()).all()
    assert ((out.double() - want).abs()[rows] <= tol[rows]).all()
