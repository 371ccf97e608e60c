"""Attention of chunks of new tokens over the paged cache (paged_prefill) against
64 bits, within the per-element bound that chunk_ref.chunk_ref derives.  Unowned
cache memory holds NaN throughout."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from chunk_ref import chunk_ref
from helpers import rng

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BOUNDS = 2


def B():
    import b200_decode

    return b200_decode


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(v):
    return dev(np.asarray(v, np.int32))


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert B().device_status(reset=True) == 0


def make(past, new, ps, hq, hkv, d, dtype, seed=0, k_scale=1.0, pad=2):
    r = rng(sum(past) + 31 * sum(new) + ps + d + seed)
    c = R.make_cache(r, [a + b for a, b in zip(past, new)], ps, hkv, d, dtype, k_scale=k_scale)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = dev(r.standard_normal((int(cu[-1]) + pad, hq, d)).astype(np.float32)).to(R.DTYPES[dtype])
    return r, c, cu, q


def run(c, q, cu, dtype, scale, mask=None, window=0, layout="token", **kw):
    dk, dv = R.to_device(c, dtype, layout)
    cache = B().PagedKV(dk, dv)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    got = B().paged_prefill(cache, q, i32(c["table"]), i32(c["lens"]), i32(cu), scale,
                            mask=None if mask is None else dev(mask), window=window, out=out, **kw)
    assert got.data_ptr() == out.data_ptr()
    return out


def check(c, q, cu, ps, dtype, mask=None, window=0, scale=None, **kw):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = run(c, q, cu, dtype, scale, mask, window, **kw)
    want, tol = chunk_ref(c, q, cu, ps, scale, mask, window)
    rows = torch.arange(q.shape[0], device="cuda")
    mine = (rows >= int(cu[0])) & (rows < int(cu[-1]))
    assert (out[~mine] == 7).all()  # rows of no sequence are left as they were
    off = (out.double() - want).abs()[mine] - tol[mine]
    assert not torch.isnan(out[mine]).any()
    assert (off <= 0).all(), f"{(off > 0).sum().item()} of {off.numel()} off by up to {off.max().item():.3e} more"


SHAPES = [
    # past, new, page size, heads, KV heads, head dim
    ([0], [1], 16, 4, 2, 64), ([0], [2], 1, 2, 2, 128), ([5], [3], 5, 12, 2, 128), ([0, 40], [33, 1], 16, 8, 2, 64),
    ([100, 0, 7], [0, 64, 9], 24, 12, 2, 128), ([127, 128, 129], [1, 1, 1], 16, 64, 8, 128),
    ([300], [200], 100, 6, 2, 64), ([0], [300], 300, 3, 1, 128), ([1000], [5], 16, 16, 4, 256),
    ([0, 3], [130, 70], 16, 4, 4, 256), ([2500], [40], 64, 24, 2, 64), ([63, 64, 65, 0], [65, 64, 63, 128], 32, 8, 8, 64),
    ([17], [129], 16, 32, 2, 128), ([4000], [1], 16, 64, 8, 128), ([0], [1030], 128, 8, 1, 128),
    ([10, 20, 30, 40, 50], [3, 0, 2, 0, 1], 7, 20, 4, 128), ([9000], [17], 16, 12, 2, 128), ([600], [300], 8, 130, 1, 64),
    ([40], [3], 16, 300, 1, 128), ([200], [257], 16, 1, 1, 256),
    ([0], [512], 16, 64, 8, 128), ([0, 100, 30], [400, 0, 250], 16, 32, 8, 64), ([64], [300], 16, 16, 4, 256),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d", SHAPES)
def test_chunks(past, new, ps, hq, hkv, d, dtype):
    _, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    check(c, q, cu, ps, dtype)


@pytest.mark.parametrize("past,new,ps,hq,hkv,d,dtype", [([500], [1000], 16, 16, 4, 256, "f16"),
                                                        ([2000, 500, 600, 100], [700] * 4, 24, 8, 2, 256, "bf16"),
                                                        ([900, 0], [600, 1500], 16, 16, 8, 128, "bf16"),
                                                        ([900, 0], [600, 1500], 64, 24, 8, 64, "f16")])
def test_ranges_of_many_tiles_and_units(past, new, ps, hq, hkv, d, dtype):
    """Work for every SM: ranges that hold the end of a unit, whole ones and the start of another."""
    _, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    check(c, q, cu, ps, dtype)
    check(c, q, cu, ps, dtype, window=700)


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 24), (256, 64)])
def test_every_tile_counts_once(d, ps):
    """Keys of 0 and values that name their position: every weight is 1 / length,
    over 300 sequences of 1 to 8 tiles of keys in ranges that cut them anywhere."""
    bw, n, most = B(), 300, 8 * 128
    r = rng(d)
    lens = r.integers(1, most + 1, n)
    nb = R.ceil_div(most, ps)
    v = torch.zeros((n * nb, ps, 1, d), dtype=torch.float16, device="cuda")
    table = torch.randperm(n * nb, device="cuda", generator=torch.Generator("cuda").manual_seed(d)).int().view(n, nb)
    pos = torch.arange(nb * ps, device="cuda")
    width = R.ceil_div(most, d)  # positions that share a channel
    v[table[:, pos // ps].long(), pos % ps, 0, (pos // width) % d] = 1
    cache = bw.PagedKV(torch.zeros_like(v), v)
    q = torch.randn((n, 1, d), device="cuda").half()
    out = bw.paged_prefill(cache, q, table, i32(lens), i32(np.arange(n + 1)), 1.0)[:, 0].double()
    end = dev(lens)[:, None]
    want = ((end - torch.arange(d, device="cuda") * width).clamp(0, width)).double() / end
    # sums of whole numbers below 2^24 are exact; the quotient is rounded in f32 twice and to f16
    assert ((out - want).abs() <= want * (2.0 ** -11 + 2.0 ** -22) + 2.0 ** -25).all()


@pytest.mark.parametrize("window", [1, 2, 100, 129, 1000])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d,dtype", [([0], [300], 16, 8, 2, 128, "f16"),
                                                        ([700, 0, 130], [50, 200, 1], 24, 12, 2, 64, "bf16"),
                                                        ([300], [140], 16, 4, 2, 256, "f16")])
def test_window(past, new, ps, hq, hkv, d, dtype, window):
    _, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    check(c, q, cu, ps, dtype, window=window)


@pytest.mark.parametrize("kind", ["mixed", "nothing", "lowest", "left", "tail", "one"])
@pytest.mark.parametrize("past,new,ps,hq,hkv,d,dtype", [([0, 100], [150, 3], 16, 8, 2, 128, "f16"),
                                                        ([700, 0, 130], [50, 200, 1], 24, 12, 2, 64, "bf16"),
                                                        ([300], [140], 16, 4, 2, 256, "bf16")])
def test_mask(past, new, ps, hq, hkv, d, dtype, kind):
    r, c, cu, q = make(past, new, ps, hq, hkv, d, dtype)
    width = c["table"].shape[1] * ps
    m = r.standard_normal((len(past), width + 5)).astype(np.float32)
    if kind == "mixed":
        m[r.random(m.shape) < 0.3] = -np.inf
        m[r.random(m.shape) < 0.05] = -65504
    elif kind == "nothing":
        m[0] = -np.inf
    elif kind == "lowest":
        m[:] = -65504
    elif kind == "left":  # padding on the left: the first rows see the lowest value alone
        m[:, :20] = -65504
        m[:, 20:] = 0
    elif kind == "tail":
        m[:, 40:] = -np.inf
    else:
        m[:] = -np.inf
        m[:, 7] = 3
    m = m.astype(np.float16)
    for s in range(len(past)):  # what the mask leaves out may hold anything
        for p in range(past[s] + new[s]):
            if m[s, p] == -np.inf:
                c["k"][c["table"][s, p // ps], p % ps] = np.nan
                c["v"][c["table"][s, p // ps], p % ps] = np.nan
    check(c, q, cu, ps, dtype, mask=m)


@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("ps", [1, 5, 16, 300])
def test_layouts_strided_queries_and_scales(layout, ps):
    _, c, cu, q = make([90, 0], [40, 133], ps, 8, 2, 128, "bf16")
    wide = torch.zeros((q.shape[0], 3 * 1024 + 8), dtype=q.dtype, device="cuda")
    wide[:, 1024:2048] = q.flatten(1)
    view = wide[:, 1024:2048].unflatten(1, (8, 128))
    for scale in (0.2, -0.3, 0.0):
        check(c, view, cu, ps, "bf16", scale=scale, layout=layout)


def test_one_table_and_one_mask_row_for_all():
    r, c, cu, q = make([200], [4], 16, 8, 2, 128, "f16")
    n = 3
    dk, dv = R.to_device(c, "f16")
    cache = B().PagedKV(dk, dv)
    m = np.zeros((1, c["table"].shape[1] * 16), np.float16)
    m[0, 5:50] = -np.inf
    cu3 = np.array([0, 4, 5, 6], np.int32)
    lens = [204, 100, 37]
    out = B().paged_prefill(cache, q, i32(c["table"]).expand(n, -1), i32(lens), i32(cu3), 0.1,
                            mask=dev(m).expand(n, -1))
    many = dict(c, table=np.repeat(c["table"], n, 0), lens=np.array(lens))
    want, tol = chunk_ref(many, q, cu3, 16, 0.1, np.repeat(m, n, 0))
    assert ((out.double() - want).abs()[:6] <= tol[:6]).all()


def test_near_equal_and_crowded_scores():
    """Scores of hundreds (one position takes all) and of nothing (all equal)."""
    for k_scale in (0.0, 60.0):
        _, c, cu, q = make([500, 0], [70, 200], 16, 8, 2, 128, "f16", k_scale=k_scale)
        check(c, q, cu, 16, "f16")


def test_growing_scores():
    """Every position's score exceeds the one before: the running maximum moves all the time."""
    for dtype in ("f16", "bf16"):
        _, c, cu, q = make([900], [130], 16, 4, 2, 128, dtype)
        for p in range(1030):
            c["k"][c["table"][0, p // 16], p % 16] = R.rounded(np.full((2, 128), p / 256.0, np.float32), dtype)
        q[:] = q.abs()
        check(c, q, cu, 16, dtype)


def test_lengths_that_the_plan_did_not_serve_and_bad_rows():
    """A sequence with fewer tokens than rows: the rows before its first token
    see nothing.  Starts that go back or past the rows are clamped and recorded."""
    _, c, cu, q = make([0, 50], [30, 20], 16, 8, 2, 128, "f16")
    c["lens"][0] = 12
    check(c, q, cu, 16, "f16")
    bad = cu.copy()
    bad[1], bad[2] = -5, 90
    out = run(c, q, bad, "f16", 0.1)
    assert B().device_status(reset=True) == BOUNDS
    assert torch.isfinite(out.float()).all()
    c["lens"][1] = 10**6
    run(c, q, cu, "f16", 0.1)
    assert B().device_status(reset=True) == BOUNDS


def test_starts_that_go_back_and_forth_stay_in_the_workspace():
    """Every other sequence names all rows: far more units than there is room for."""
    bw, n = B(), 400
    _, c, cu, q = make([0], [64], 16, 64, 8, 128, "f16", pad=0)
    dk, dv = R.to_device(c, "f16")
    dv[c["table"][0, 0], 3, :, 5] = float("inf")  # and every row is computed again
    size = bw.paged_prefill_workspace_size(128, 64, n, 64, 8)
    ws = torch.full((size + 4096,), 0x3C, dtype=torch.uint8, device="cuda")
    starts = i32([0 if i % 2 == 0 else 64 for i in range(n + 1)])
    out = bw.paged_prefill(bw.PagedKV(dk, dv), q, i32(c["table"]).expand(n, -1), i32([64] * n), starts, 0.1,
                           workspace=ws[:size])
    assert bw.device_status(reset=True) == BOUNDS
    assert (ws[size:] == 0x3C).all() and torch.isfinite(out[:, :, :5].float()).all()


def test_bad_pages_are_recorded_and_passed_over():
    _, c, cu, q = make([64], [16], 16, 8, 2, 128, "f16")
    good = run(c, q, cu, "f16", 0.1)
    c["table"][0, 1] = 10**6
    out = run(c, q, cu, "f16", 0.1)
    assert B().device_status(reset=True) == BOUNDS
    assert torch.isfinite(out.float()).all() and not torch.equal(out, good)


def nonfinite_want(c, q, cu, ps, scale):
    """The formula in 64 bits, infinities and NaN included, row by row."""
    n_head, d = q.shape[1:]
    group = n_head // c["k"].shape[2]
    out = np.zeros(tuple(q.shape))
    qs = q.double().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        for s in range(len(cu) - 1):
            n, length = int(cu[s + 1] - cu[s]), int(c["lens"][s])
            for i in range(n):
                pos = np.arange(length - n + i + 1)
                page = c["table"][s, pos // ps]
                for j in range(n_head):
                    k, v = c["k"][page, pos % ps, j // group], c["v"][page, pos % ps, j // group]
                    x = (qs[cu[s] + i, j] * k).sum(-1) * scale
                    w = np.exp(x - np.max(x)) if np.max(x) > -np.inf or np.isnan(x).any() else np.zeros_like(x)
                    t = w.sum()
                    out[cu[s] + i, j] = 0 if t == 0 else (w[:, None] * v).sum(0) / t
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("what", ["v_inf", "v_nan", "k_nan", "k_inf", "k_minus", "v_both"])
def test_infinities_and_nan(what, d, dtype):
    """In a token's key or value: the rows before it do not see it."""
    _, c, cu, q = make([100, 30], [60, 3], 16, 4, 2, d, dtype)
    at = [(0, 130, 0), (0, 40, 1), (1, 31, 1)]  # (sequence, position, KV head)
    for s, p, h in at:
        cell = (c["table"][s, p // 16], p % 16, h)
        if what == "v_inf":
            c["v"][cell][3] = np.inf
        elif what == "v_nan":
            c["v"][cell][5] = np.nan
        elif what == "k_nan":
            c["k"][cell][7] = np.nan
        elif what == "k_inf":
            c["k"][cell][:] = np.inf
        elif what == "k_minus":
            c["k"][cell][:] = -np.inf
            q[:] = q.abs()
        else:
            c["v"][cell][3] = np.inf
            p2 = p - 1
            c["v"][c["table"][s, p2 // 16], p2 % 16, h][3] = -np.inf
    out = run(c, q, cu, dtype, 0.05).double().cpu().numpy()
    want = nonfinite_want(c, q, cu, 16, 0.05)
    rows = slice(0, int(cu[-1]))
    out, want = out[rows], want[rows]
    np.testing.assert_array_equal(np.isnan(out), np.isnan(want))
    np.testing.assert_array_equal(np.where(np.isinf(out), out, 0), np.where(np.isinf(want), want, 0))
    fine = np.isfinite(want)
    assert fine.mean() > 0.2
    # two roundings to 16 bits of sums of values below 6, and f32 sums far below
    assert np.abs(out[fine] - want[fine]).max() <= 2 * 6 * torch.finfo(q.dtype).eps / 2 * 1.1


def test_captured_and_replayed_with_other_lengths_and_another_stream():
    _, c, cu, q = make([300, 0, 50], [4, 200, 1], 16, 8, 2, 128, "f16")
    bw = B()
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    table, lens, dcu = i32(c["table"]), i32(c["lens"]), i32(cu)
    ws = torch.empty(bw.paged_prefill_workspace_size(128, q.shape[0], 3, 8, 2), dtype=torch.uint8, device="cuda")
    ws.fill_(0xA5)  # needs no initial contents
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        bw.paged_prefill(cache, q, table, lens, dcu, 0.1, out=out, workspace=ws)
    for now in (c["lens"], np.array([270, 120, 11], np.int32)):
        lens.copy_(i32(now))
        g.replay()
        want, tol = chunk_ref(dict(c, lens=now), q, cu, 16, 0.1)
        assert ((out.double() - want).abs()[: cu[-1]] <= tol[: cu[-1]]).all()
    with torch.cuda.stream(side):
        again = bw.paged_prefill(cache, q, table, lens, dcu, 0.1, workspace=ws)
    side.synchronize()
    assert torch.equal(again[: cu[-1]], out[: cu[-1]])


def test_same_bits_every_time():
    _, c, cu, q = make([5000, 100, 0], [3, 90, 400], 16, 64, 8, 128, "bf16")
    first = run(c, q, cu, "bf16", 0.09)
    for _ in range(3):
        assert torch.equal(run(c, q, cu, "bf16", 0.09), first)


def test_many_sequences_of_one_token_agree_with_decode_attention():
    """Rows of one token each: what paged_attn computes in f32."""
    past = [int(x) for x in rng(5).integers(0, 400, 150)]
    _, c, cu, q = make(past, [1] * 150, 16, 8, 2, 128, "f16", pad=0)
    out = run(c, q, cu, "f16", 0.09)
    dk, dv = R.to_device(c, "f16")
    ref = B().paged_attn(B().PagedKV(dk, dv), q.float(), i32(c["table"]), i32(c["lens"]), 0.09)
    _, tol = chunk_ref(c, q, cu, 16, 0.09)
    assert ((out.double() - ref.double()).abs() <= 2 * tol).all()


def test_empty_calls():
    bw = B()
    _, c, cu, q = make([3], [2], 16, 4, 2, 64, "f16")
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    assert bw.paged_prefill(cache, q[:0], i32(c["table"]), i32(c["lens"]), i32([0, 0]), 1.0).shape == (0, 4, 64)
    out = torch.full_like(q, 3)
    bw.paged_prefill(cache, q, i32(c["table"]), i32(c["lens"]), i32([1, 1]), 1.0, out=out)
    assert (out == 3).all()


def test_out_that_overlaps_the_queries_is_refused():
    bw = B()
    _, c, cu, q = make([3], [2], 16, 4, 2, 64, "f16")
    dk, dv = R.to_device(c, "f16")
    with pytest.raises(bw.B200Error) as e:
        bw.paged_prefill(bw.PagedKV(dk, dv), q, i32(c["table"]), i32(c["lens"]), i32(cu), 1.0, out=q)
    assert e.value.code == bw.EINVAL
