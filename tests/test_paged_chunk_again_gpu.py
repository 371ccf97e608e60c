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


@pytest.mark.parametrize("ps", [16, 5])
@pytest.mark.parametrize("hides", ["window", "mask"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_out_of_range_that_no_row_sees_change_nothing(d, hides, ps):
    """Behind the window or under -inf: recorded, but the tiles' sums stay as they are."""
    _, c, cu, q = make([700], [30], ps, 8, 2, d, "f16")
    mask, window = None, 0
    if hides == "window":
        window = 300
        first = 700 - 300 + 1
    else:
        first = 333
        mask = np.zeros((1, c["table"].shape[1] * ps), np.float16)
        mask[0, :first] = -np.inf
    good = run(c, q, cu, "f16", 0.1, mask, window)
    c["table"][0, : first // ps] = -1
    out = run(c, q, cu, "f16", 0.1, mask, window)
    assert B().device_status(reset=True) == BOUNDS
    assert torch.equal(out, good)


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


def nonfinite_want(c, q, cu, ps, scale, mask, window):
    """The formula in 64 bits, infinities and NaN included: a position that is not seen
    has no part in it."""
    n_head, d = q.shape[1:]
    group = n_head // c["k"].shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    qs, k_all, v_all = q.double().cpu(), torch.from_numpy(c["k"]), torch.from_numpy(c["v"])
    for s in range(len(cu) - 1):
        n, length = int(cu[s + 1] - cu[s]), int(c["lens"][s])
        for i in range(n):
            at = length - n + i
            pos = np.arange(max(0, at - window + 1) if window else 0, at + 1)
            bias = np.zeros(pos.size)
            if mask is not None:
                pos = pos[mask[s, pos] != -np.inf]
                bias = mask[s, pos].astype(np.float64)
            if pos.size == 0:
                continue
            page = torch.from_numpy(c["table"][s, pos // ps].astype(np.int64))
            for j in range(n_head):
                k, v = k_all[page, pos % ps, j // group], v_all[page, pos % ps, j // group]
                x = (qs[cu[s] + i, j] * k).sum(-1) * scale + torch.from_numpy(bias)
                if (x == -np.inf).all():
                    continue
                w = (x - x.max()).exp()
                out[cu[s] + i, j] = (w[:, None] * v).sum(0) / w.sum()
    return out


@pytest.mark.parametrize("also", ["", "mask", "window"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d", [([2500, 0], [7, 40], 16, 12, 2, 128), ([1900], [5], 5, 24, 2, 64),
                                                  ([700, 300, 600, 100], [40, 1, 60, 9], 24, 4, 4, 256)])
def test_infinities_in_units_that_ranges_cut(past, new, ps, hq, hkv, d, dtype, also):
    """Far from each other, so that several pieces of a unit meet one."""
    r, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    for s, n in enumerate(past):
        for p, what in ((n // 9, np.inf), (n // 2, -np.inf), (n - n // 8, np.nan), (n + new[s] // 2, np.inf)):
            c["v"][c["table"][s, p // ps], p % ps, 0, int(r.integers(d))] = what
        c["k"][c["table"][s, (n // 3) // ps], (n // 3) % ps, hkv - 1] = np.inf if s % 2 else np.nan
    mask, window = None, 0
    if also == "mask":
        mask = r.standard_normal((len(past), c["table"].shape[1] * ps)).astype(np.float16)
        mask[r.random(mask.shape) < 0.3] = -np.inf
        mask[:, [n // 3 for n in past]] = -np.inf
    elif also == "window":
        window = 150
    out = run(c, q, cu, dtype, 0.07, mask, window)[: int(cu[-1])].double().cpu()
    want = nonfinite_want(c, q, cu, ps, 0.07, mask, window)[: int(cu[-1])]
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(torch.where(out.isinf(), out, 0.0), torch.where(want.isinf(), want, 0.0))
    fine = want.isfinite()
    assert fine.double().mean() > 0.2
    # two roundings to 16 bits of sums of values below 6, and f32 sums far below
    assert (out - want).abs()[fine].max() <= 2 * 6 * torch.finfo(q.dtype).eps / 2 * 1.1


def test_an_infinity_far_back_does_not_take_forever():
    """5 rows of 12 heads over 65536 positions: 3 ms with a CTA to a row (about 220 ms when
    a warp took a row and one position at a time)."""
    bw, n, new = B(), 65536, 5
    k = torch.randn((n // 16 + 1, 16, 2, 128), device="cuda").half()
    v = torch.randn_like(k)
    v[0, 3, :, 7] = float("inf")
    table = torch.arange(n // 16 + 1, device="cuda").int()[None]
    q = torch.randn((new, 12, 128), device="cuda").half()
    times = []
    for _ in range(3):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        out = bw.paged_prefill(bw.PagedKV(k, v), q, table, i32([n + new]), i32([0, new]), 0.1)
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    assert (out[:, :, 7] == float("inf")).all() and torch.isfinite(out[:, :, 8:].float()).all()
    assert min(times) < 20, times


def test_lists_start_empty_in_every_replay_and_streams_have_their_own():
    """A captured call whose infinity comes and goes, and two calls at once: every one
    gives the bits that it gives alone."""
    bw = B()
    _, c, cu, q = make([2500, 40], [9, 30], 16, 12, 2, 128, "f16", pad=0)
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    args = i32(c["table"]), i32(c["lens"]), i32(cu), 0.09
    size = bw.paged_prefill_workspace_size(128, q.shape[0], 2, 12, 2)
    ws = [torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    cells = [(int(c["table"][0, p // 16]), p % 16, h, 3) for p, h in ((7, 0), (1300, 1), (2400, 0))]
    alone = []
    for what in (1.0, float("inf")):
        for cell in cells:
            dv[cell] = what
        alone.append(bw.paged_prefill(cache, q, *args, workspace=ws[0]).clone())
    assert torch.isfinite(alone[0].float()).all() and (alone[1][: int(cu[1]), :, 3] == float("inf")).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bw.paged_prefill(cache, q, *args, out=outs[0], workspace=ws[0])
    for turn in (1, 0, 1, 1, 0):
        for cell in cells:
            dv[cell] = (1.0, float("inf"))[turn]
        outs[0].zero_()
        g.replay()
        assert torch.equal(outs[0], alone[turn])
    for cell in cells:
        dv[cell] = float("inf")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, w, out in zip(streams, ws, outs):
            with torch.cuda.stream(stream):
                bw.paged_prefill(cache, q, *args, out=out, workspace=w)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], alone[1]) and torch.equal(outs[1], alone[1])
