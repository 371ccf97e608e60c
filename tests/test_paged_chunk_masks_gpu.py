"""Masks of paged_prefill over ranges of many key tiles, through the tiles themselves:
keys and values are finite under -inf too, so no row is computed again, and every CTA
has tens of tiles, so the slots of mask entries are used over and over."""
import numpy as np
import pytest

import paged_ref as R
from chunk_ref import chunk_ref

torch = pytest.importorskip("torch")
from test_paged_chunk_gpu import B, _status_clean, dev, i32, make, run  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# past, new, page size, heads, KV heads, head dim; key tiles to a CTA (of 128 positions, at head dim 256 of 64)
SHAPES = [([2048], [2048], 16, 64, 8, 128), ([1500, 0, 2900], [1500, 2000, 100], 24, 24, 4, 64),
          ([1000, 700], [1024, 900], 32, 16, 4, 256), ([3000], [1200], 100, 32, 8, 128)]


def mask_of(kind, r, shape):
    m = r.standard_normal(shape).astype(np.float32)
    pos = np.arange(shape[1])
    if kind == "scattered":
        m[r.random(shape) < 0.4] = -np.inf
        m[r.random(shape) < 0.05] = -65504
    elif kind == "rising":  # the reference moves with every tile
        m += 16.0 * pos / shape[1] - 8
    elif kind == "falling":
        m += 8 - 16.0 * pos / shape[1]
    elif kind == "holes":  # whole tiles at -inf, and parts of them
        m[:, (pos // 192) % 3 == 1] = -np.inf
    elif kind == "lowest":  # then zeros: the first rows see the lowest value alone
        m[:] = np.where(pos < 900, -65504, 0)
    return m.astype(np.float16)


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("kind", ["scattered", "rising", "falling", "holes", "lowest"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d", SHAPES)
def test_masks_over_many_tiles(past, new, ps, hq, hkv, d, dtype, kind, window):
    r, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    m = mask_of(kind, r, (len(past), c["table"].shape[1] * ps))
    out = run(c, q, cu, dtype, d ** -0.5, m, window)
    want, tol = chunk_ref(c, q, cu, ps, d ** -0.5, m, window)
    # The reference of a row is relative to the largest mask entry so far and moves with
    # it, at most once a tile and once a piece: entries within 25 of each other and scores
    # within 8 make it less than 48 (in powers of two), so its two roundings cost the weights
    # before less than 2 * 48 log(2) 2^-24 < 68 * 2^-24, in numerator and denominator.  (After
    # the lowest value they are nothing.)  sum w |v| is at most tol over half a step.
    tiles = max(a + b for a, b in zip(past, new)) // (64 if d == 256 else 128) + 1
    tol = tol * (1 + 2 * 2 * tiles * 68 * 2.0 ** -24 / (torch.finfo(q.dtype).eps / 2))
    rows = slice(0, int(cu[-1]))
    off = (out.double() - want).abs()[rows] - tol[rows]
    assert (off <= 0).all(), f"{(~(off <= 0)).sum().item()} of {off.numel()} off by up to {off.max().item():.3e}"
