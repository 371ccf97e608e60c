"""Paged cache operators where bounds, keys, values or queries are infinite or
NaN: what the definitions in include/b200_paged.h make of them, against plain
64-bit implementations."""
import numpy as np
import pytest

import paged_ref as R
from helpers import rng

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


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


# ------------------------------------------------------------------ select

def select_by_definition(q, lo, hi, table, n_blocks, n_sel):
    """One sequence: the newest block and the best others, NaN scores (a NaN
    product, a sum of both infinities, a NaN head) behind all others, ties to
    the lower block."""
    n_head, n_head_kv = q.shape[0], lo.shape[1]
    group = n_head // n_head_kv
    out = np.full((n_head_kv, n_sel), -1, np.int32)
    with np.errstate(invalid="ignore"):
        for h in range(n_head_kv):
            qs = q[h * group:(h + 1) * group].astype(np.float64)
            score = [np.maximum(qs * lo[p, h], qs * hi[p, h]).sum(-1).max() for p in table[:n_blocks - 1]]
            older = sorted(range(n_blocks - 1), key=lambda b: (np.isnan(score[b]), 0.0 if np.isnan(score[b]) else -score[b], b))
            chosen = sorted(older[:n_sel - 1] + [n_blocks - 1])
            out[h, :len(chosen)] = chosen
    return out


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["infinite bound, zero query", "one NaN bound", "both bounds NaN", "both infinities"])
def test_select_ranks_nan_scores_last(kind, dtype, d):
    """Pages of several rows (lo < hi), 3 query heads per KV head: one page in
    five holds something that makes its score NaN for at least one head."""
    r = rng(len(kind) + d)
    n_pages, hkv, hq = 160, 2, 6
    a, b = (R.rounded(r.standard_normal((n_pages, hkv, d)), dtype) for _ in range(2))
    lo, hi = np.minimum(a, b), np.maximum(a, b)
    q = r.standard_normal((1, hq, d)).astype(np.float32)
    table = r.permutation(n_pages).astype(np.int32)
    odd = table[3:n_pages - 1:5]
    if kind == "infinite bound, zero query":  # 0 * inf
        q[:, :, 7] = 0.0
        hi[odd, :, 7] = np.inf
    elif kind == "one NaN bound":
        lo[odd[::2], :, 9] = np.nan
        hi[odd[1::2], :, 9] = np.nan
    elif kind == "both bounds NaN":
        lo[odd, :, 9] = hi[odd, :, 9] = np.nan
    else:  # +inf in one channel, -inf in another
        lo[odd, :, 4] = hi[odd, :, 4] = np.inf
        lo[odd, :, 5] = hi[odd, :, 5] = -np.inf
        q[:, :, 4:6] = np.abs(q[:, :, 4:6]) + 0.1
    t = R.DTYPES[dtype]
    k = torch.zeros((n_pages, 4, hkv, d), dtype=t, device="cuda")
    cache = B().PagedKV(k, k.clone(), dev(lo).to(t), dev(hi).to(t))
    for n_sel in (2, 30, 128, 140, 159):  # 127 or 128 older blocks have a score
        want = select_by_definition(q[0], lo, hi, table, n_pages, n_sel)
        got = B().paged_select(cache, dev(q), i32(table[None]), i32([4 * n_pages - 1]), n_sel).cpu().numpy()[0]
        np.testing.assert_array_equal(got, want, err_msg=f"n_sel {n_sel}")


def test_select_after_a_store_that_overflows():
    """An f16 key past the type's range is stored as infinity and becomes a
    bound: its page ranks first, and last for a query that is zero there."""
    bw = B()
    n_pages, d = 8, 64
    k = torch.zeros((n_pages, 4, 1, d), dtype=torch.float16, device="cuda")
    bound = torch.zeros((n_pages, 1, d), dtype=torch.float16, device="cuda")
    cache = bw.PagedKV(k, k.clone(), bound, bound.clone())
    x = torch.randn((4 * n_pages, 1, d), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    x[4 * 5 + 1, 0, 10] = 1e6
    bw.paged_store(cache, x, x, torch.arange(4 * n_pages, device="cuda"))
    table, lens = i32([list(range(n_pages))]), i32([4 * n_pages])
    q = torch.ones((1, 1, d), device="cuda")
    assert bw.paged_select(cache, q, table, lens, 2).tolist() == [[[5, 7]]]
    q[..., 10] = 0.0
    assert bw.paged_select(cache, q, table, lens, 7).tolist() == [[[0, 1, 2, 3, 4, 6, 7]]]


# --------------------------------------------------------------- attention

SHAPES = [(12, 2, 128), (24, 2, 64), (4, 2, 256), (20, 1, 128), (64, 8, 128)]


def attend(c, q, page_size, dtype, scale, mask=None, sel=None):
    dk, dv = R.to_device(c, dtype)
    return B().paged_attn(B().PagedKV(dk, dv), dev(q), i32(c["table"]), i32(c["lens"]), scale,
                          mask=None if mask is None else dev(mask),
                          sel=None if sel is None else i32(sel)).cpu().numpy().astype(np.float64)


def within(got, want, tol):
    assert bool(np.isfinite(got).all())
    assert float(np.max(np.abs(got - want) / tol)) <= 1.0


def put(c, name, s, positions, page_size, channel, value):
    for p in positions:
        c[name][c["table"][s, p // page_size], p % page_size, :, channel] = value


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_attn_scores_of_minus_infinity_have_no_weight(hq, hkv, d, masked, dtype):
    """Keys with an infinite channel of the sign opposite to the query's: as
    if those positions were masked; zeros where every position is one."""
    r = rng(hq + d + masked)
    lens, ps = [700, 50, 1, 320, 0, 16, 33, 40], 7 if hq == 12 else 16
    c = R.make_cache(r, lens, ps, hkv, d, dtype)
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2
    width = c["table"].shape[1] * ps
    mask = np.zeros((len(lens), width), np.float16)
    if masked:
        mask = r.standard_normal((len(lens), width)).astype(np.float16)
        mask[r.random((len(lens), width)) < 0.3] = -np.inf
    gone = mask.astype(np.float32)
    for s, n in enumerate(lens):
        sign = 1.0 if s % 2 else -1.0
        q[s, :, 5] = sign * (np.abs(q[s, :, 5]) + 0.1)
        at = np.nonzero(r.random(n) < 0.2)[0].tolist()
        if s == 0:
            at = sorted(set(at) | set(range(16, 32)) | set(range(500, 700)))  # whole units, and the end
        if s in (2, 5):
            at = list(range(n))  # nothing but such positions
        put(c, "k", s, at, ps, 5, -sign * np.inf)
        gone[s, at] = -np.inf
    want, tol = R.attn_ref(c, q, ps, d ** -0.5, gone)
    got = attend(c, q, ps, dtype, d ** -0.5, mask if masked else None)
    within(got, want, tol)
    assert (got[[2, 4, 5]] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,length", [(4, 1, 128, 30000), (12, 1, 64, 20000), (3, 1, 256, 9000)])
def test_attn_scores_of_minus_infinity_in_a_segment_over_every_cta(hq, hkv, d, length, dtype):
    """The first third has such scores only, the rest here and there."""
    r = rng(length)
    c = R.make_cache(r, [length], 16, hkv, d, dtype)
    q = r.standard_normal((1, hq, d)).astype(np.float32) * 2
    q[:, :, 0] = np.abs(q[:, :, 0]) + 0.1
    at = sorted(set(range(length // 3)) | set(np.nonzero(r.random(length) < 0.01)[0].tolist()))
    put(c, "k", 0, at, 16, 0, -np.inf)
    gone = np.zeros((1, c["table"].shape[1] * 16), np.float32)
    gone[0, at] = -np.inf
    want, tol = R.attn_ref(c, q, 16, d ** -0.5, gone)
    within(attend(c, q, 16, dtype, d ** -0.5), want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_attn_infinities_reach_what_the_formula_says(hq, hkv, d, dtype):
    """A score of +inf, a NaN key, a NaN or infinite query make their heads'
    outputs NaN; infinite values their own columns infinite, or NaN where both
    signs meet.  Every other output is as without them."""
    r = rng(hq * d)
    lens, ps = [300, 700, 40, 100, 90, 17], 16
    c = R.make_cache(r, lens, ps, hkv, d, dtype)
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32)
    want, tol = R.attn_ref(c, q, ps, d ** -0.5)
    q[0, 0, 7] = np.nan
    want[0, 0] = np.nan
    put(c, "k", 1, [333], ps, 9, np.inf)  # the sign of q[9] decides: +inf or no weight
    gone = np.zeros((len(lens), c["table"].shape[1] * ps), np.float32)
    gone[1, 333] = -np.inf
    plain = np.where(np.isinf(c["k"]), 0.0, c["k"])
    w1, t1 = R.attn_ref(dict(c, k=plain), q, ps, d ** -0.5, gone)
    want[1], tol[1] = np.where(q[1, :, 9:10] > 0, np.nan, w1[1]), t1[1]
    put(c, "k", 2, [20], ps, 3, np.nan)
    want[2] = np.nan
    put(c, "v", 3, [5, 80], ps, 11, np.inf)
    put(c, "v", 3, [50], ps, 12, -np.inf)
    put(c, "v", 3, [50], ps, 13, np.inf)
    put(c, "v", 3, [51], ps, 13, -np.inf)
    want[3, :, 11], want[3, :, 12], want[3, :, 13] = np.inf, -np.inf, np.nan
    q[4, 1, 2] = np.inf  # scores of both infinities
    want[4, 1] = np.nan
    got = attend(c, q, ps, dtype, d ** -0.5)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    some = ~np.isnan(want)
    np.testing.assert_array_equal(np.where(np.isinf(got[some]), got[some], 0), np.where(np.isinf(want[some]), want[some], 0))
    rest = np.isfinite(want)
    assert float(np.max(np.abs(got[rest] - want[rest]) / tol[rest])) <= 1.0


def test_attn_selected_blocks_with_an_overflowed_key():
    """paged_store makes an infinity of an f16 key past the range; selection
    and attention over what was selected take it from there."""
    bw = B()
    r = rng(8)
    n, ps, d = 90, 16, 64
    k, v = (r.standard_normal((n, 1, d)).astype(np.float32) for _ in range(2))
    k[70, 0, 4] = -1e6
    pages = -(-n // ps)
    zeros = torch.zeros((pages, ps, 1, d), dtype=torch.float16, device="cuda")
    bound = torch.zeros((pages, 1, d), dtype=torch.float16, device="cuda")
    cache = bw.PagedKV(zeros, zeros.clone(), bound, bound.clone())
    bw.paged_store(cache, dev(k), dev(v), torch.arange(n, device="cuda"))
    q = r.standard_normal((1, 8, d)).astype(np.float32)
    q[:, :, 4] = np.abs(q[:, :, 4]) + 0.1
    table, lens = i32([list(range(pages))]), i32([n])
    sel = bw.paged_select(cache, dev(q), table, lens, 4)
    got = bw.paged_attn(cache, dev(q), table, lens, 0.125, sel=sel).cpu().numpy().astype(np.float64)
    c = dict(k=cache.k.double().cpu().numpy(), v=cache.v.double().cpu().numpy(), table=table.cpu().numpy(),
             lens=np.array([n], np.int32))
    gone = np.zeros((1, pages * ps), np.float32)
    gone[0, 70] = -np.inf
    within(got, *R.attn_ref(c, q, ps, 0.125, gone, sel.cpu().numpy()))


def test_attn_bf16_values_near_the_largest():
    """A value of 3e38 at the position of the largest weight: the weighted sum
    stays in f32's range, as it does with weights of at most one.  Of 60000
    positions the kernel takes several units of 16 with one reference for their
    weights."""
    r = rng(9)
    for d, n in ((64, 40), (128, 40), (256, 40), (64, 60000), (128, 60000), (256, 60000)):
        c = R.make_cache(r, [n], 16, 1, d, "bf16")
        c["k"][~np.isnan(c["k"])] = 0.0
        put(c, "k", 0, [20], 16, 0, 1.75)  # e^1.75 = 2^2.52 times the others' weight
        c["v"][~np.isnan(c["v"])] = 1.0
        put(c, "v", 0, [20], 16, slice(None), R.rounded(np.float32(3e38), "bf16"))
        q = np.zeros((1, 4, d), np.float32)
        q[:, :, 0] = 1.0
        want, tol = R.attn_ref(c, q, 16, 1.0)
        within(attend(c, q, 16, "bf16", 1.0), want, tol)
