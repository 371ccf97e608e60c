"""Paged key-value cache operators against plain 64-bit implementations
(paged_ref.py), through the Python layer and the C ABI.

Integers (plans, selections), stored rows and key bounds are compared bit for
bit; attention against the per-element bound that paged_ref.attn_ref derives.
Unowned cache memory holds NaN throughout."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
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


# -------------------------------------------------------------------- plan

def random_state(r, n, page_size, max_blocks, n_pages, max_len):
    """Sequences with lengths up to max_len (as the pool allows) in shuffled
    pages, and the stack of the pages left."""
    order = r.permutation(n_pages).astype(np.int32)
    table = r.integers(-5, 0, (n, max_blocks)).astype(np.int32)
    lens = np.zeros(n, np.int32)
    at = 0
    for s in range(n):
        length = int(r.integers(0, max_len + 1))
        b = R.ceil_div(length, page_size)
        if b > max_blocks or at + b > n_pages:
            continue
        table[s, :b] = order[at:at + b]
        lens[s] = length
        at += b
    stack = np.full(n_pages, -7, np.int32)
    stack[: n_pages - at] = order[at:]
    return lens, table, stack, n_pages - at


def run_plan(new, lens, table, stack, top, page_size, max_tokens, in_place):
    d = dict(new_lens=i32(new), seq_lens=i32(lens), block_table=i32(table), free_pages=i32(stack), n_free=i32([top]))
    kw = {}
    if not in_place:
        kw = dict(seq_lens_out=torch.full_like(d["seq_lens"], -9), n_free_out=torch.full_like(d["n_free"], -9))
    p = B().paged_plan(page_size=page_size, max_tokens=max_tokens, **d, **kw)
    if in_place:
        assert p.seq_lens.data_ptr() == d["seq_lens"].data_ptr() and p.n_free.data_ptr() == d["n_free"].data_ptr()
    got = [p.slots, p.positions, p.cu, p.seq_lens, p.n_free, d["block_table"], d["free_pages"]]
    return [t.cpu().numpy() for t in got]


def check_plan(new, lens, table, stack, top, page_size, max_tokens, in_place=False):
    want = R.plan_ref(new, lens, table, stack, top, page_size, max_tokens)
    got = run_plan(new, lens, table, stack, top, page_size, max_tokens, in_place)
    for name, g, w in zip(("slots", "positions", "cu", "seq_lens", "n_free", "table"), got, want):
        np.testing.assert_array_equal(g, np.asarray(w).reshape(g.shape), err_msg=name)
    # the stack up to where pushes reached; what was popped stays as it was pushed
    np.testing.assert_array_equal(got[6], want[6], err_msg="free_pages")
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,page_size,max_len,chunk", [(1, 16, 40, 1), (1, 1, 5, 9), (3, 5, 30, 7), (64, 16, 900, 1),
                                                       (257, 16, 300, 40), (1023, 8, 100, 3), (1025, 32, 400, 65),
                                                       (8192, 4, 20, 3)])
def test_plan_matches_reference(n, page_size, max_len, chunk, in_place):
    r = rng(n + page_size)
    max_blocks = R.ceil_div(max_len + chunk, page_size)
    lens, table, stack, top = random_state(r, n, page_size, max_blocks, n * max_blocks + 3, max_len)
    new = r.integers(-1, chunk + 1, n).astype(np.int32)
    tokens = int(np.maximum(new, 0).sum())
    check_plan(new, lens, table, stack, top, page_size, tokens + 5, in_place)


@pytest.mark.parametrize("seed", range(8))
def test_plan_refuses_what_does_not_fit(seed):
    """Too few pages, rows that outgrow the table and tokens past max_tokens,
    in one step with sequences that end and give pages to later ones."""
    r = rng(900 + seed)
    n, page_size, max_blocks = 50, 4, 6
    lens, table, stack, top = random_state(r, n, page_size, max_blocks, 130, 24)
    new = r.choice([-1, 0, 1, 2, 5, 13], n).astype(np.int32)
    tokens = int(np.maximum(new, 0).sum())
    want = check_plan(new, lens, table, stack, top, page_size, tokens - int(r.integers(0, 30)), in_place=seed % 2 == 0)
    assert (want[3] != np.where(new < 0, 0, lens + np.maximum(new, 0))).any()  # something was refused


def test_plan_idle_ending_and_empty_pool():
    lens = np.array([5, 0, 8], np.int32)
    table = np.array([[3, 1, -1], [-1, -1, -1], [0, 2, -1]], np.int32)
    stack = np.full(4, -1, np.int32)
    check_plan(np.array([0, 0, 0], np.int32), lens, table, stack, 0, 4, 0)  # nothing to do, no rows at all
    check_plan(np.array([-1, -1, -1], np.int32), lens, table, stack, 0, 4, 3)  # everything ends
    check_plan(np.array([3, 0, 0], np.int32), lens, table, stack, 0, 4, 3)  # fits its last page
    check_plan(np.array([4, 1, 1], np.int32), lens, table, stack, 0, 4, 6)  # needs pages, none are left
    check_plan(np.array([4, 5, -1], np.int32), lens, table, stack, 0, 4, 9)  # the third one's pages serve the others
    big = np.array([2**31 - 1, 1, 2**31 - 1], np.int32)  # sums past 32 bits
    check_plan(big, lens, table, stack, 0, 4, 9)


def test_plan_bad_state_is_reported_and_never_followed():
    bw = B()
    stack = np.arange(6, dtype=np.int32)
    table = np.full((2, 3), 77, np.int32)  # page 77 of 6
    out = run_plan([1, 0], [2, 1], table, stack, 6, 4, 2, False)
    assert bw.device_status(reset=True) == BOUNDS
    assert (out[0] == -1).all()
    run_plan([0, 0], [-3, 100], table, stack, 6, 4, 2, False)  # lengths outside the table
    assert bw.device_status(reset=True) == BOUNDS
    run_plan([0, 1], [0, 0], table, stack, 9, 4, 2, False)  # more free pages than pages
    assert bw.device_status(reset=True) == BOUNDS
    out = run_plan([-1, 0], [12, 0], np.zeros((2, 3), np.int32), stack, 5, 4, 2, False)  # 5 + 3 pages of 6
    assert bw.device_status(reset=True) == BOUNDS
    assert out[4][0] == 6


# ------------------------------------------------------------------- store

def bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("lens,chunk,page_size,n_head_kv,d", [
    ([0], 1, 16, 2, 128), ([15, 16, 17, 0, 31], 1, 16, 8, 128), ([3, 0, 250], 37, 5, 1, 64), ([7], 300, 128, 3, 256),
    ([0, 1], 1, 1, 2, 64), ([20, 64, 63], 130, 64, 2, 128)])
def test_store_rows_and_bounds(lens, chunk, page_size, n_head_kv, d, layout, dtype):
    r = rng(sum(lens) + chunk + d)
    after = [n + chunk for n in lens]
    c = R.make_cache(r, after, page_size, n_head_kv, d, dtype)
    for s, n in enumerate(lens):  # the new tokens' slots are not written yet
        for p in range(n, after[s]):
            c["k"][c["table"][s, p // page_size], p % page_size] = np.nan
            c["v"][c["table"][s, p // page_size], p % page_size] = np.nan
    lo, hi = R.bounds_of(c)
    dk, dv = R.to_device(c, dtype, layout)
    t = R.DTYPES[dtype]
    dlo, dhi = dev(lo).to(t), dev(hi).to(t)
    tokens = len(lens) * chunk
    slots = np.full(tokens + 2, -1, np.int64)  # two rows of padding behind the last sequence
    new = r.standard_normal((2, tokens + 2, n_head_kv, d)).astype(np.float32) * 3
    new[:, -2:] = np.nan
    for s, n in enumerate(lens):
        for j in range(chunk):
            p = n + j
            slots[s * chunk + j] = c["table"][s, p // page_size] * page_size + p % page_size
    cache = B().PagedKV(dk, dv, dlo, dhi)
    # rows of a wider matrix, as a fused projection leaves them
    fused = torch.zeros((tokens + 2, 2 * n_head_kv * d + 8), device="cuda")
    fused[:, :n_head_kv * d] = dev(new[0]).flatten(1)
    fused[:, n_head_kv * d + 4:-4] = dev(new[1]).flatten(1)
    B().paged_store(cache, fused[:, :n_head_kv * d], fused[:, n_head_kv * d + 4:-4], dev(slots))
    for i, name in enumerate("kv"):
        for row, slot in enumerate(slots[:tokens]):
            c[name][slot // page_size, slot % page_size] = R.rounded(new[i, row], dtype)
    wk, wv = R.to_device(c, dtype)
    np.testing.assert_array_equal(bits(dk), bits(wk))
    np.testing.assert_array_equal(bits(dv), bits(wv))
    wlo, whi = R.bounds_of(c)
    for s in range(len(lens)):
        for b in range(R.ceil_div(after[s], page_size)):
            p = c["table"][s, b]
            np.testing.assert_array_equal(dlo[p].double().cpu().numpy(), wlo[p])
            np.testing.assert_array_equal(dhi[p].double().cpu().numpy(), whi[p])
    if layout == "gap":  # the space between the rows is untouched
        n, h = dk.shape[0], n_head_kv
        whole = torch.as_strided(dk, (n, page_size + 1, h + 1, d + 8), dk.stride())
        assert torch.isnan(whole[:, page_size]).all() and torch.isnan(whole[:, :, h]).all()
        assert torch.isnan(whole[..., d:]).all()


def test_store_without_bounds_single_row_and_bad_slots():
    bw = B()
    k = torch.zeros((3, 4, 2, 64), dtype=torch.float16, device="cuda")
    cache = bw.PagedKV(k, torch.zeros_like(k))
    x = torch.randn((3, 2, 64), device="cuda")
    bw.paged_store(cache, x, -x, torch.tensor([5, -1, -100], device="cuda"))
    assert bw.device_status(reset=True) == 0
    want = torch.zeros_like(k)
    want[1, 1] = x[0].half()
    assert torch.equal(k, want) and torch.equal(cache.v, -want)
    bw.paged_store(cache, x, x, torch.tensor([12, 2**40, 0], device="cuda"))  # 12 slots: 0 .. 11
    assert bw.device_status(reset=True) == BOUNDS
    want[0, 0] = x[2].half()
    assert torch.equal(k, want)


def test_store_extreme_values():
    """Values past the f16 range become infinities; NaN keys leave bounds alone."""
    bw = B()
    for dtype in (torch.float16, torch.bfloat16):
        k = torch.zeros((2, 2, 1, 64), dtype=dtype, device="cuda")
        lo, hi = torch.zeros((2, 1, 64), dtype=dtype, device="cuda"), torch.zeros((2, 1, 64), dtype=dtype, device="cuda")
        cache = bw.PagedKV(k, k.clone(), lo, hi)
        x = torch.randn((2, 1, 64), device="cuda")
        x[0, 0, :4] = torch.tensor([1e30, -1e30, float("nan"), 1e-30], device="cuda")
        x[1, 0, 2] = 0.5
        bw.paged_store(cache, x, x, torch.tensor([2, 3], device="cuda"))
        assert torch.equal(torch.nan_to_num(k[1]), torch.nan_to_num(x.to(dtype)))
        assert (lo[1, 0, 2] == 0.5) and (hi[1, 0, 2] == 0.5)
        keep = torch.arange(64, device="cuda") != 2
        assert torch.equal(lo[1][:, keep], x.to(dtype).amin(0)[:, keep])
        assert torch.equal(hi[1][:, keep], x.to(dtype).amax(0)[:, keep])


# ------------------------------------------------------------------ select

def select_inputs(r, lens, page_size, n_head, n_head_kv, d, dtype, ties=False):
    c = R.make_cache(r, lens, page_size, n_head_kv, d, dtype)
    if ties:  # pages that hold the same few rows over and over
        few = R.rounded(r.standard_normal((3, n_head_kv, d)), dtype)
        for p in range(c["k"].shape[0]):
            live = ~np.isnan(c["k"][p, :, 0, 0])
            c["k"][p, live] = few[p % 3]
    q = r.standard_normal((len(lens), n_head, d)).astype(np.float32)
    return c, q


def run_select(c, q, page_size, n_sel, dtype, table=None, workspace=None, stream=None):
    lo, hi = R.bounds_of(c)
    dk, dv = R.to_device(c, dtype)
    t = R.DTYPES[dtype]
    cache = B().PagedKV(dk, dv, dev(lo).to(t), dev(hi).to(t))
    return B().paged_select(cache, dev(q), i32(c["table"] if table is None else table), i32(c["lens"]), n_sel,
                            workspace=workspace)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,page_size,heads,d,n_sel", [
    ([1], 16, (2, 2), 128, 1), ([0, 5, 0], 4, (4, 1), 64, 3), ([1000, 16, 17, 999, 0], 16, (64, 8), 128, 7),
    ([333, 2000], 5, (24, 2), 64, 64), ([700], 3, (16, 4), 256, 1), ([4000, 123], 7, (12, 4), 128, 571),
    ([700, 31], 1, (8, 8), 128, 300), ([90], 1, (26, 2), 64, 200)])
def test_select_matches_reference(lens, page_size, heads, d, n_sel, dtype):
    r = rng(sum(lens) + d + n_sel)
    c, q = select_inputs(r, lens, page_size, *heads, d, dtype)
    lo, hi = R.bounds_of(c)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], page_size, n_sel)
    np.testing.assert_array_equal(run_select(c, q, page_size, n_sel, dtype).cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,n_sel", [(8193, 500), (8194, 8100), (20001, 64), (3000, 1), (1025, 1024), (1026, 512)])
def test_select_many_blocks(n, n_sel, dtype):
    """More blocks than a CTA's threads hold at once, and around that number."""
    r = rng(n + n_sel)
    c, q = select_inputs(r, [n, n // 3], 1, 4, 2, 64, dtype)
    lo, hi = R.bounds_of(c)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], 1, n_sel)
    np.testing.assert_array_equal(run_select(c, q, 1, n_sel, dtype).cpu().numpy(), want)


@pytest.mark.parametrize("n", [300, 2000, 9000])
@pytest.mark.parametrize("kinds", [1, 2, 5])
def test_select_crowds_of_equal_scores(n, kinds):
    """Hundreds of blocks with the same keys: nothing but the 64-bit order and
    the lower block decide."""
    r = rng(n + kinds)
    c = R.make_cache(r, [n], 1, 1, 64, "bf16")
    few = R.rounded(r.standard_normal((kinds, 1, 64)), "bf16")
    for b in range(n):
        c["k"][c["table"][0, b], 0] = few[r.integers(kinds)]
    q = r.standard_normal((1, 2, 64)).astype(np.float32)
    lo, hi = R.bounds_of(c)
    for n_sel in (2, n // 4, n // 2, n - 1):
        want = R.select_ref(q, lo, hi, c["table"], c["lens"], 1, n_sel)
        np.testing.assert_array_equal(run_select(c, q, 1, n_sel, "bf16").cpu().numpy(), want)


def test_select_scores_that_differ_in_the_last_bits():
    """Keys that differ by one step of their type in one channel: scores that
    agree to six digits, in an order that 32 bits would not find."""
    r = rng(14)
    for dtype, step in (("f16", 2.0 ** -10), ("bf16", 2.0 ** -7)):
        n = 600
        c = R.make_cache(r, [n], 1, 1, 128, dtype)
        base = R.rounded(1 + r.random(128) * 0.9, dtype)
        for b in range(n):
            row = base.copy()
            row[r.integers(128)] -= step * int(r.integers(0, 3))
            c["k"][c["table"][0, b], 0, 0] = row
        q = r.standard_normal((1, 3, 128)).astype(np.float32)
        q[:, :, ::7] *= 1e-4
        lo, hi = R.bounds_of(c)
        for n_sel in (10, 300):
            want = R.select_ref(q, lo, hi, c["table"], c["lens"], 1, n_sel)
            np.testing.assert_array_equal(run_select(c, q, 1, n_sel, dtype).cpu().numpy(), want)


def test_select_not_finite():
    """Infinite bounds rank first, NaN queries leave the lower blocks."""
    r = rng(15)
    c, q = select_inputs(r, [500], 1, 2, 1, 64, "f16")
    q = np.abs(q) + 0.1
    for b in (7, 300, 450):
        c["k"][c["table"][0, b], 0, 0, 3] = np.inf
    lo, hi = R.bounds_of(c)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], 1, 6)
    got = run_select(c, q, 1, 6, "f16").cpu().numpy()
    np.testing.assert_array_equal(got, want)
    assert set((7, 300, 450)) <= set(got[0, 0].tolist())
    q[:] = np.nan
    np.testing.assert_array_equal(run_select(c, q, 1, 6, "f16").cpu().numpy()[0, 0], [0, 1, 2, 3, 4, 499])


@pytest.mark.parametrize("n_seq", [31, 33, 129, 400])
def test_select_and_attn_of_many_sequences(n_seq):
    r = rng(n_seq)
    lens = [int(v) for v in r.integers(0, 60, n_seq)]
    lens[0], lens[-1], lens[n_seq // 2] = 0, 0, 333
    c, q = select_inputs(r, lens, 4, 6, 2, 64, "f16")
    lo, hi = R.bounds_of(c)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], 4, 5)
    np.testing.assert_array_equal(run_select(c, q, 4, 5, "f16").cpu().numpy(), want)
    check_attn(c, q, 4, "f16", 0.125)
    check_attn(c, q, 4, "f16", 0.125, sel=want)


@pytest.mark.parametrize("n_sel", [1, 2, 50, 66, 67, 99, 100, 101])
def test_select_ties_take_the_lower_block(n_sel):
    r = rng(11)
    c, q = select_inputs(r, [400, 398], 4, 8, 2, 64, "f16", ties=True)
    lo, hi = R.bounds_of(c)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], 4, n_sel)
    np.testing.assert_array_equal(run_select(c, q, 4, n_sel, "f16").cpu().numpy(), want)
    q[:] = 0  # every score is zero
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], 4, n_sel)
    np.testing.assert_array_equal(run_select(c, q, 4, n_sel, "f16").cpu().numpy(), want)


def test_select_tiny_and_huge_scores():
    """Subnormal f16 bounds, and queries whose products leave the f32 range."""
    r = rng(12)
    for scale, dtype in ((2.0 ** -22, "f16"), (1e30, "bf16"), (1e-38, "bf16")):
        c, q = select_inputs(r, [777], 7, 4, 2, 64, dtype)
        live = ~np.isnan(c["k"])
        c["k"][live] = R.rounded(c["k"][live] * scale, dtype)
        q *= 1e20 if scale > 1 else 1.0
        lo, hi = R.bounds_of(c)
        want = R.select_ref(q, lo, hi, c["table"], c["lens"], 7, 30)
        np.testing.assert_array_equal(run_select(c, q, 7, 30, dtype).cpu().numpy(), want)


def test_select_bad_pages_come_last_and_are_reported():
    bw = B()
    r = rng(13)
    c, q = select_inputs(r, [40], 4, 2, 1, 64, "f16")
    lo, hi = R.bounds_of(c)
    table = c["table"].copy()
    table[0, 3], table[0, 5] = -1, 10**6
    got = run_select(c, q, 4, 8, "f16", table=table).cpu().numpy()[0, 0]
    assert bw.device_status(reset=True) == BOUNDS
    np.testing.assert_array_equal(got, [0, 1, 2, 4, 6, 7, 8, 9])
    lens = c["lens"].copy()
    c["lens"][:] = 4000  # past the table: clamped to its ten blocks
    got = run_select(c, q, 4, 12, "f16").cpu().numpy()[0, 0]
    assert bw.device_status(reset=True) == BOUNDS
    np.testing.assert_array_equal(got, list(range(10)) + [-1, -1])
    c["lens"] = lens


# --------------------------------------------------------------- attention

def make_mask(r, kind, n_seq, width):
    if kind is None:
        return None
    m = r.standard_normal((n_seq, width)).astype(np.float16)
    if kind == "holes":
        m[r.random((n_seq, width)) < 0.4] = -np.inf
        m[r.random((n_seq, width)) < 0.1] = -65504.0
    elif kind == "lowest":  # nothing but the type's lowest value
        m[:] = -65504.0
    elif kind == "rows":  # whole rows without a position, one with a single one
        m[::2] = -np.inf
        m[1] = -np.inf
        m[1, 0] = 3.0
    elif kind == "steep":  # falls by 2 per position from the newest
        m[:] = np.maximum(-2.0 * np.arange(width, dtype=np.float32)[::-1], -65504).astype(np.float16)
    return m


def check_attn(c, q, page_size, dtype, scale, mask=None, sel=None, layout="token", **kw):
    dk, dv = R.to_device(c, dtype, layout)
    out = B().paged_attn(B().PagedKV(dk, dv), kw.pop("dq", None) if "dq" in kw else dev(q), i32(c["table"]),
                         i32(c["lens"]), scale, mask=None if mask is None else dev(mask),
                         sel=None if sel is None else i32(sel), **kw)
    want, tol = R.attn_ref(c, q, page_size, scale, mask, sel)
    got = out.cpu().numpy().astype(np.float64)
    worst = np.max(np.abs(got - want) / tol)
    assert bool(np.isfinite(got).all()) and float(worst) <= 1.0, f"{worst:.2f} of the bound"
    return out


LENS = [([1], 16), ([37], 16), ([0, 1, 15, 16, 17, 0], 16), ([127, 128, 129, 255, 256, 257], 32), ([63, 500, 5], 5),
        ([1000], 1), ([2048, 3, 777], 100), ([4160], 16), ([9000, 0, 1], 64), ([5000, 4096, 17], 2048), ([2500, 1], 1000)]
SHAPES = [(12, 2, 128), (24, 2, 64), (4, 4, 256), (64, 8, 128), (8, 8, 64), (16, 4, 256), (40, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,page_size", LENS)
def test_attn_lengths(lens, page_size, dtype):
    r = rng(sum(lens) + page_size)
    c = R.make_cache(r, lens, page_size, 2, 128, dtype)
    q = r.standard_normal((len(lens), 12, 128)).astype(np.float32) * 2
    check_attn(c, q, page_size, dtype, 128 ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_attn_head_shapes_and_layouts(hq, hkv, d, layout, dtype):
    lens, page_size = [300, 0, 33, 1], 24
    r = rng(hq + d)
    c = R.make_cache(r, lens, page_size, hkv, d, dtype)
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2
    check_attn(c, q, page_size, dtype, d ** -0.5, layout=layout)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["plain", "holes", "lowest", "rows", "steep"])
@pytest.mark.parametrize("hq,hkv,d,page_size", [(12, 2, 128, 16), (24, 2, 64, 24), (4, 2, 256, 7)])
def test_attn_masks(kind, hq, hkv, d, page_size, dtype):
    lens = [700, 50, 1, 320, 0, 16]
    r = rng(len(kind) + d)
    c = R.make_cache(r, lens, page_size, hkv, d, dtype)
    mask = make_mask(r, kind, len(lens), c["table"].shape[1] * page_size + 3)
    # what a mask of -inf leaves out may hold anything
    for s, n in enumerate(lens):
        for p in np.nonzero(np.isneginf(mask[s, :n]))[0]:
            c["k"][c["table"][s, p // page_size], p % page_size] = np.nan
            c["v"][c["table"][s, p // page_size], p % page_size] = np.inf
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2
    out = check_attn(c, q, page_size, dtype, d ** -0.5, mask=mask)
    if kind == "rows":
        assert (out[::2] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,page_size,hq,hkv,d,n_sel", [
    ([500, 16, 1, 0, 333], 16, 12, 2, 128, 4), ([999, 40], 5, 24, 2, 64, 30), ([600, 64, 65], 32, 16, 4, 256, 1),
    ([3000], 8, 64, 8, 128, 40)])
def test_attn_selected_blocks(lens, page_size, hq, hkv, d, n_sel, dtype):
    r = rng(sum(lens) + n_sel)
    c = R.make_cache(r, lens, page_size, hkv, d, dtype)
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2
    sel = np.full((len(lens), hkv, n_sel), -1, np.int32)
    for s, n in enumerate(lens):
        nb = R.ceil_div(n, page_size)
        for h in range(hkv):
            pick = np.sort(r.permutation(nb)[:n_sel])
            sel[s, h, :pick.size] = pick
    check_attn(c, q, page_size, dtype, d ** -0.5, sel=sel)
    mask = make_mask(r, "holes", len(lens), c["table"].shape[1] * page_size)
    check_attn(c, q, page_size, dtype, d ** -0.5, sel=sel, mask=mask)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,length,page_size", [(4, 1, 128, 30000, 16), (12, 1, 64, 50000, 48),
                                                       (20, 1, 128, 9000, 16), (3, 1, 256, 20000, 100)])
def test_attn_one_segment_over_every_cta(hq, hkv, d, length, page_size, dtype):
    """A long sequence of one KV head: over a hundred pieces to join."""
    r = rng(length + hq)
    c = R.make_cache(r, [length], page_size, hkv, d, dtype)
    q = r.standard_normal((1, hq, d)).astype(np.float32) * 2
    check_attn(c, q, page_size, dtype, d ** -0.5)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (14, 2), (16, 1), (17, 1), (33, 1)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attn_group_sizes(hq, hkv, d):
    r = rng(hq * d)
    lens = [200, 3, 0, 90]
    c = R.make_cache(r, lens, 16, hkv, d, "f16")
    q = r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2
    mask = make_mask(r, "holes", len(lens), c["table"].shape[1] * 16)
    check_attn(c, q, 16, "f16", d ** -0.5)
    check_attn(c, q, 16, "f16", d ** -0.5, mask=mask)


def test_attn_keys_and_values_in_different_layouts():
    r = rng(44)
    c = R.make_cache(r, [100, 37], 16, 2, 128, "f16")
    q = r.standard_normal((2, 8, 128)).astype(np.float32)
    for a, b in (("token", "head"), ("head", "gap"), ("gap", "token")):
        cache = B().PagedKV(R.to_device(c, "f16", a)[0], R.to_device(c, "f16", b)[1])
        got = B().paged_attn(cache, dev(q), i32(c["table"]), i32(c["lens"]), 0.1).cpu().numpy()
        want, tol = R.attn_ref(c, q, 16, 0.1)
        assert (np.abs(got - want) <= tol).all(), (a, b)


def test_attn_one_workspace_for_all_shapes():
    """Calls of other head dims, groups, batches and masks in between leave a
    workspace ready for the next."""
    bw = B()
    r = rng(52)
    ws = torch.zeros(4 << 20, dtype=torch.uint8, device="cuda")
    for hq, hkv, d, n in ((3, 3, 256, 2), (4, 2, 64, 300), (12, 1, 128, 3), (64, 8, 128, 5), (1, 1, 256, 40), (14, 1, 64, 7),
                          (8, 8, 64, 64), (3, 3, 256, 2)):
        lens = [int(v) for v in r.integers(0, 9000 // n + 200, n)]
        c = R.make_cache(r, lens, 16, hkv, d, "f16")
        q = r.standard_normal((n, hq, d)).astype(np.float32)
        assert ws.numel() >= bw.paged_attn_workspace_size(d, n, hq, hkv)
        check_attn(c, q, 16, "f16", d ** -0.5, workspace=ws)


def test_empty_batch_and_no_tokens():
    bw = B()
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16, device="cuda")
    b = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda")
    cache = bw.PagedKV(k, k.clone(), b, b.clone())
    q = torch.zeros((0, 4, 64), device="cuda")
    table, lens = torch.zeros((0, 3), dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert bw.paged_attn(cache, q, table, lens, 1.0).shape == (0, 4, 64)
    assert bw.paged_select(cache, q, table, lens, 2).shape == (0, 2, 2)
    x = torch.zeros((0, 2, 64), device="cuda")
    bw.paged_store(cache, x, x, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert (cache.k == 0).all()


FIRST_CALL = """
import sys
sys.path[:0] = {path!r}
import torch, b200_decode as B
k = torch.randn((8, 16, 2, 128), device="cuda").half()
cache = B.PagedKV(k, k.clone(), k.amin(1).contiguous(), k.amax(1).contiguous())
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
table, lens, n_free, free, new = i32([[0, 1, 2, -1]]), i32([40]), i32([3]), i32([5, 6, 7, 0, 0, 0, 0, 0]), i32([3])
x, q = torch.randn((3, 2, 128), device="cuda"), torch.randn((1, 4, 128), device="cuda")
ws = torch.zeros(B.paged_attn_workspace_size(128, 1, 4, 2), dtype=torch.uint8, device="cuda")
out_lens, out_free = i32([0]), i32([0])
def step():
    p = B.paged_plan(new, lens, table, free, n_free, 16, 3, seq_lens_out=out_lens, n_free_out=out_free)
    B.paged_store(cache, x, x, p.slots)
    sel = B.paged_select(cache, q, table, p.seq_lens, 2)
    return B.paged_attn(cache, q, table, p.seq_lens, 0.1, workspace=ws), \
        B.paged_attn(cache, q, table, p.seq_lens, 0.1, sel=sel)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
want = step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) and a.abs().sum() > 0 for a, b in zip(got, want))
assert int(out_lens.item()) == 43 and B.device_status() == 0
print("captured")
"""


def test_first_calls_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(B().__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(path=[here])], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_attn_selected_blocks_any_order_repeats_and_gaps():
    """-1 anywhere, a block listed twice, blocks past the sequence, the
    partial block first: what the list says is what is attended to."""
    r = rng(77)
    c = R.make_cache(r, [70, 9], 16, 1, 64, "f16")
    q = r.standard_normal((2, 4, 64)).astype(np.float32)
    sel = np.array([[[4, -1, 2, 2, 0, -5]], [[-1, -1, -1, -1, -1, -1]]], np.int32)
    out = check_attn(c, q, 16, "f16", 0.125, sel=sel)
    assert (out[1] == 0).all()
    sel = np.array([[[1, 4, 5, 4, 1000, 2**31 - 1]], [[0, 1, 3, 3, 3, 3]]], np.int32)
    check_attn(c, q, 16, "f16", 0.125, sel=sel)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attn_peaked_and_extreme_queries(dtype):
    """Scores in the hundreds (one position takes all), tiny and huge query
    magnitudes, scale 0 and a negative scale."""
    r = rng(31)
    c = R.make_cache(r, [400, 90], 16, 2, 128, dtype)
    for mag, scale in ((60.0, 128 ** -0.5), (1e-6, 128 ** -0.5), (1e5, 1e-5), (1e30, 1e-30), (1e-30, 1e30), (1.0, 0.0),
                       (1.0, -0.3)):
        q = (r.standard_normal((2, 8, 128)) * mag).astype(np.float32)
        check_attn(c, q, 16, dtype, scale)


def test_attn_values_at_the_end_of_their_range():
    """f16 values of 60000, bf16 values of 1e36: the weighted sums stay in
    range as far as f32 sums of weights of at most one would."""
    r = rng(32)
    for dtype, big in (("f16", 6e4), ("bf16", 1e36)):
        c = R.make_cache(r, [40, 3], 16, 2, 128, dtype)
        live = ~np.isnan(c["v"])
        c["v"][live] = R.rounded(np.sign(c["v"][live]) * big * (0.5 + 0.5 * r.random(live.sum())), dtype)
        q = r.standard_normal((2, 8, 128)).astype(np.float32)
        check_attn(c, q, 16, dtype, 0.1)


def test_attn_strided_queries_tables_and_masks():
    r = rng(41)
    lens, ps = [100, 333], 16
    c = R.make_cache(r, lens, ps, 2, 128, "f16")
    q = r.standard_normal((2, 12, 128)).astype(np.float32)
    fused = torch.zeros((2, 16 * 128 + 4), device="cuda")
    fused[:, :12 * 128] = dev(q).flatten(1)
    view = fused[:, :12 * 128].view(2, 12, 128)
    check_attn(c, q, ps, "f16", 0.1, dq=view)
    odd = torch.zeros((2, 12 * 128 + 1), device="cuda")  # rows that are not 16-byte aligned
    odd[:, 1:] = dev(q).flatten(1)
    check_attn(c, q, ps, "f16", 0.1, dq=odd[:, 1:].view(2, 12, 128))
    wide = torch.full((2, 50), 10**8, dtype=torch.int32, device="cuda")
    wide[:, :c["table"].shape[1]] = i32(c["table"])
    dk, dv = R.to_device(c, "f16")
    cache = B().PagedKV(dk, dv)
    want = B().paged_attn(cache, dev(q), i32(c["table"]), i32(lens), 0.1)
    got = B().paged_attn(cache, dev(q), wide[:, :c["table"].shape[1]], i32(lens), 0.1)
    assert torch.equal(got, want)
    # entries of the table past the sequence's blocks are never followed
    got = B().paged_attn(cache, dev(q), wide, i32(lens), 0.1)
    assert torch.equal(got, want)


def test_attn_bad_pages_and_lengths_are_reported():
    bw = B()
    r = rng(43)
    c = R.make_cache(r, [64, 20], 16, 2, 64, "f16")
    q = r.standard_normal((2, 4, 64)).astype(np.float32)
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    table = c["table"].copy()
    table[0, 1], table[0, 2] = -1, 10**7
    got = bw.paged_attn(cache, dev(q), i32(table), i32(c["lens"]), 0.125).cpu().numpy()
    assert bw.device_status(reset=True) == BOUNDS
    sel = np.array([[[0, 3]] * 2, [[0, 1]] * 2], np.int32)  # as if the bad blocks were not there
    want, tol = R.attn_ref(c, q, 16, 0.125, sel=sel)
    assert (np.abs(got - want) <= tol).all()
    c["table"] = c["table"][:, :2]  # 64 tokens, a table of 2 blocks: clamped
    got = bw.paged_attn(cache, dev(q), i32(c["table"]), i32([64, -4]), 0.125).cpu().numpy()
    assert bw.device_status(reset=True) == BOUNDS
    c["lens"] = np.array([32, 0], np.int32)
    want, tol = R.attn_ref(c, q, 16, 0.125)
    assert (np.abs(got - want) <= tol).all()


def test_attn_same_bits_every_time_and_on_any_workspace():
    """Split and joined in a fixed order: repeated calls agree bit for bit,
    whatever other shapes used the workspace in between."""
    bw = B()
    r = rng(51)
    c = R.make_cache(r, [5000, 10, 0, 2600], 16, 8, 128, "f16")
    q = dev(r.standard_normal((4, 64, 128)).astype(np.float32))
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    table, lens = i32(c["table"]), i32(c["lens"])
    first = bw.paged_attn(cache, q, table, lens, 0.09)
    ws = torch.zeros(bw.paged_attn_workspace_size(128, 4, 64, 8), dtype=torch.uint8, device="cuda")
    for i in range(5):
        assert torch.equal(bw.paged_attn(cache, q, table, lens, 0.09, workspace=ws), first)
        n = 1 + i % 4
        got = bw.paged_attn(cache, q[:n].contiguous(), table[:n], lens[:n], 0.09, workspace=ws)
        want, tol = R.attn_ref(dict(c, table=c["table"][:n], lens=c["lens"][:n]), q[:n].cpu().numpy(), 16, 0.09)
        assert (np.abs(got.cpu().numpy() - want) <= tol).all()


def test_attn_offsets_past_32_bits():
    """Pages beyond byte 2^32 of the cache (a 9 GiB allocation of which few
    pages are touched)."""
    ps, hkv, d = 64, 8, 128
    n_pages = (9 << 30) // (ps * hkv * d * 2)
    r = rng(61)
    small = R.make_cache(r, [200, 130], ps, hkv, d, "f16", extra_pages=0)
    big = torch.empty((n_pages, ps, hkv, d), dtype=torch.float16, device="cuda")
    lo = torch.empty((n_pages, hkv, d), dtype=torch.float16, device="cuda")
    hi = torch.empty_like(lo)
    sk, sv = R.to_device(small, "f16")
    slo, shi = R.bounds_of(small)
    far = np.linspace(n_pages // 2, n_pages - 1, sk.shape[0]).astype(np.int64)
    big[dev(far)] = sk
    cache = B().PagedKV(big, big, lo, hi)
    q = r.standard_normal((2, 64, d)).astype(np.float32)
    small["v"] = small["k"]
    table = i32(np.where(small["table"] >= 0, far[small["table"]], -1))
    out = B().paged_attn(cache, dev(q), table, i32(small["lens"]), 0.1).cpu().numpy()
    want, tol = R.attn_ref(small, q, ps, 0.1)
    assert (np.abs(out - want) <= tol).all()
    lo[dev(far)], hi[dev(far)] = dev(slo).half(), dev(shi).half()
    sel = B().paged_select(cache, dev(q), table, i32(small["lens"]), 3).cpu().numpy()
    np.testing.assert_array_equal(sel, R.select_ref(q, slo, shi, small["table"], small["lens"], ps, 3))
    row = torch.randn((1, hkv, d), device="cuda")
    last = n_pages * ps - 1
    B().paged_store(cache, row, row, torch.tensor([last], device="cuda"))
    assert torch.equal(big[-1, -1], row[0].half())


def test_refusals_of_the_python_layer_on_device():
    bw = B()
    k = torch.zeros((4, 16, 2, 128), dtype=torch.float16, device="cuda")
    cache = bw.PagedKV(k, k.clone())
    q = torch.zeros((2, 4, 128), device="cuda")
    table, lens = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(q=q.cpu()), dict(table=table.long()),
           dict(table=table[:1]), dict(table=table.cpu()), dict(table=table.t().contiguous().t()), dict(lens=lens[:1]),
           dict(lens=lens.long()), dict(mask=torch.zeros((2, 31), dtype=torch.float16, device="cuda")),
           dict(mask=torch.zeros((2, 32), device="cuda")),
           dict(sel=torch.zeros((2, 1, 3), dtype=torch.int32, device="cuda")),
           dict(sel=torch.zeros((2, 2, 0), dtype=torch.int32, device="cuda")),
           dict(out=torch.zeros((2, 4, 64), device="cuda")), dict(out=q),
           dict(workspace=torch.zeros(64, device="cuda")),
           dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))]
    for over in bad:
        a = dict(q=q, table=table, lens=lens)
        a.update(over)
        kw = {n: a[n] for n in ("mask", "sel", "out", "workspace") if n in a}
        with pytest.raises(bw.B200Error):
            bw.paged_attn(cache, a["q"], a["table"], a["lens"], 1.0, **kw)
    with pytest.raises(bw.B200Error):
        bw.paged_select(cache, q, table, lens, 2)  # no key bounds
    with pytest.raises(bw.B200Error):
        bw.paged_store(cache, q, q, torch.zeros(2, dtype=torch.int64, device="cuda"))  # 4 heads into a cache of 2
    with pytest.raises(bw.B200Error):
        bw.paged_store(cache, q[:, :2], q[:, :2], torch.zeros(2, dtype=torch.int32, device="cuda"))
    for badk in (k.cpu(), k[..., ::2], k[:, :, :, 1:65]):
        with pytest.raises(bw.B200Error):
            bw.PagedKV(badk, badk)
    assert (bw.paged_attn(cache, q, table, lens, 1.0) == 0).all()  # a batch of empty sequences


# -------------------------------------------------- the operators together

class Server:
    """A toy serving loop on the host's reference: what the device loop must
    reproduce step by step."""

    def __init__(self, n, ps, width, n_pages, hq, hkv, d, dtype, seed):
        self.r = rng(seed)
        self.n, self.ps, self.hq, self.hkv, self.d, self.dtype = n, ps, hq, hkv, d, dtype
        self.lens = np.zeros(n, np.int32)
        self.table = np.full((n, width), -1, np.int32)
        self.stack, self.top = self.r.permutation(n_pages).astype(np.int32), n_pages
        self.k = np.full((n_pages, ps, hkv, d), np.nan)
        self.v = self.k.copy()

    def step(self, new, max_tokens):
        k, v = (self.r.standard_normal((max_tokens, self.hkv, self.d)).astype(np.float32) for _ in range(2))
        out = R.plan_ref(new, self.lens, self.table, self.stack, self.top, self.ps, max_tokens)
        slots, positions, cu, self.lens, self.top, self.table, self.stack = out
        self.stack[self.top:] = -1
        for t, slot in enumerate(slots):
            if slot >= 0:
                page, row = slot // self.ps, slot % self.ps
                if row == 0:  # a recycled page starts afresh
                    self.k[page], self.v[page] = np.nan, np.nan
                self.k[page, row], self.v[page, row] = R.rounded(k[t], self.dtype), R.rounded(v[t], self.dtype)
        q = self.r.standard_normal((self.n, self.hq, self.d)).astype(np.float32) * 2
        return k, v, q, slots, positions

    def attend(self, q, n_sel, scale):
        c = dict(k=self.k, v=self.v, table=self.table, lens=self.lens)
        lo, hi = R.bounds_of(c)
        sel = R.select_ref(q, lo, hi, self.table, self.lens, self.ps, n_sel)
        return R.attn_ref(c, q, self.ps, scale), sel, R.attn_ref(c, q, self.ps, scale, sel=sel)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,d,ps,n_pages", [("f16", 12, 2, 128, 16, 10), ("bf16", 8, 2, 64, 5, 30)])
def test_serving_loop(dtype, hq, hkv, d, ps, n_pages, graph):
    """Prompts, decode steps, requests that end and start, refusals when pages
    run out: plan -> store -> select -> attention (all blocks, then the
    selected ones), eager or as one captured graph that every step replays."""
    bw = B()
    n, width, max_tokens, n_sel, scale = 6, 12, 96, 3, 0.2
    srv = Server(n, ps, width, n_pages, hq, hkv, d, dtype, 5)
    t = R.DTYPES[dtype]
    dk = torch.full((n_pages, ps, hkv, d), float("nan"), dtype=t, device="cuda")
    cache = bw.PagedKV(dk, dk.clone(), torch.full((n_pages, hkv, d), float("nan"), dtype=t, device="cuda"),
                       torch.full((n_pages, hkv, d), float("nan"), dtype=t, device="cuda"))
    lens, n_free = torch.zeros(n, dtype=torch.int32, device="cuda"), i32([n_pages])
    table, stack = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), i32(srv.stack)
    new = torch.zeros(n, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros((max_tokens, hkv, d), device="cuda") for _ in range(2))
    q = torch.zeros((n, hq, d), device="cuda")
    ws_a = torch.zeros(bw.paged_attn_workspace_size(d, n, hq, hkv), dtype=torch.uint8, device="cuda")
    ws_s = torch.empty(bw.paged_select_workspace_size(n, hkv, width), dtype=torch.uint8, device="cuda")
    res = {}

    def once():
        p = bw.paged_plan(new, lens, table, stack, n_free, ps, max_tokens)
        bw.paged_store(cache, k, v, p.slots)
        res["plan"] = p
        res["dense"] = bw.paged_attn(cache, q, table, p.seq_lens, scale, workspace=ws_a)
        res["sel"] = bw.paged_select(cache, q, table, p.seq_lens, n_sel, workspace=ws_s)
        res["sparse"] = bw.paged_attn(cache, q, table, p.seq_lens, scale, sel=res["sel"], workspace=ws_a)

    g = None
    if graph:
        once()  # new is zero: a step that changes nothing
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            once()
    refused = 0
    for step in range(25):
        want_new = srv.r.choice([-1, 0, 1, 1, 1, 1, 9, 21], n, p=[.06, .04, .2, .2, .2, .2, .05, .05]).astype(np.int32)
        if step == 0:
            want_new[:] = [7, 30, 1, 0, 16, 12]
        before = srv.lens.copy()
        hk, hv, hq_, slots, positions = srv.step(want_new, max_tokens)
        refused += int((srv.lens != np.where(want_new < 0, 0, before + np.maximum(want_new, 0))).sum())
        new.copy_(i32(want_new))
        k.copy_(dev(hk))
        v.copy_(dev(hv))
        q.copy_(dev(hq_))
        if g is None:
            once()
        else:
            g.replay()
        (dense, tol), sel, (sparse, stol) = srv.attend(hq_, n_sel, scale)
        np.testing.assert_array_equal(res["plan"].slots.cpu().numpy(), slots, err_msg=f"step {step}")
        np.testing.assert_array_equal(res["plan"].positions.cpu().numpy(), positions)
        np.testing.assert_array_equal(lens.cpu().numpy(), srv.lens)
        assert int(n_free.item()) == srv.top
        np.testing.assert_array_equal(res["sel"].cpu().numpy(), sel, err_msg=f"step {step}")
        assert (np.abs(res["dense"].cpu().numpy() - dense) <= tol + 1e-30).all(), step
        assert (np.abs(res["sparse"].cpu().numpy() - sparse) <= stol + 1e-30).all(), step
    assert refused > 0


def test_two_streams_with_their_own_workspaces():
    bw = B()
    r = rng(91)
    jobs = []
    for i, lens in enumerate(([3000, 17], [900, 2500])):
        c = R.make_cache(r, lens, 16, 8, 128, "f16")
        dk, dv = R.to_device(c, "f16")
        q = r.standard_normal((2, 64, 128)).astype(np.float32)
        jobs.append((c, q, bw.PagedKV(dk, dv), dev(q), i32(c["table"]), i32(lens), torch.cuda.Stream(),
                     torch.zeros(bw.paged_attn_workspace_size(128, 2, 64, 8), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (c, q, cache, dq, table, lens, st, ws) in enumerate(jobs):
            with torch.cuda.stream(st):
                outs[i].append(bw.paged_attn(cache, dq, table, lens, 0.09, workspace=ws))
                outs[i].append(bw.paged_attn(cache, dq, table, lens, 0.09))  # a workspace of its own
    torch.cuda.synchronize()
    for i, (c, q, *_) in enumerate(jobs):
        want, tol = R.attn_ref(c, q, 16, 0.09)
        for o in outs[i]:
            assert (np.abs(o.cpu().numpy() - want) <= tol).all()
            assert torch.equal(o, outs[i][0])
