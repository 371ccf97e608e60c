"""Paths of the paged store and the block selection that only larger calls
take: store tiles of many tokens, selection at head dim 256."""
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


# ------------------------------------------------------------------- store

def ragged_slots(r, tokens, page_size):
    """(slots, pages): sequences of 1 to 3000 new tokens behind cached ones of any
    number, in shuffled pages, with 0 to 4 rows of padding between them."""
    owners, at = [], 0
    while at < tokens:
        n = min(tokens - at, int(r.choice([1, 2, int(r.integers(3, 70)), int(r.integers(70, 3000))])))
        owners.append((int(r.integers(0, 5 * page_size)), n))
        at += n + int(r.integers(0, 5))
    blocks = [R.ceil_div(old + n, page_size) for old, n in owners]
    order = r.permutation(sum(blocks))
    slots, first = [], 0
    for (old, n), b in zip(owners, blocks):
        p = np.arange(old, old + n)
        slots.append(order[first + p // page_size].astype(np.int64) * page_size + p % page_size)
        slots.append(np.full(int(r.integers(0, 5)), -1 - int(r.integers(0, 9)), np.int64))
        first += b
    return np.concatenate(slots), sum(blocks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,n_head_kv,d,page_size,tile", [
    (2000, 2, 128, 16, 2), (8195, 8, 128, 64, 28), (9600, 8, 64, 64, 33), (9600, 8, 64, 100, 33), (20000, 8, 64, 64, 64),
    (20000, 8, 64, 100, 64), (6000, 25, 64, 2048, 64), (20000, 4, 64, 5, 5), (5000, 16, 256, 24, 24), (9000, 8, 64, 33, 31),
    (20000, 2, 64, 1, 1)])
def test_store_tiles_of_many_tokens(tokens, n_head_kv, d, page_size, tile, dtype):
    """Several runs of tokens per CTA, runs that begin anywhere in a tile and
    end in a later one: rows and bounds bit for bit, all else untouched."""
    r = rng(tokens + page_size + d)
    slots, n_pages = ragged_slots(r, tokens, page_size)
    want_tile = min(64, page_size, R.ceil_div(len(slots) * n_head_kv, 2368))
    assert abs(want_tile - tile) <= 1  # (the padding's rows count too)
    t = R.DTYPES[dtype]
    shape = (n_pages, page_size, n_head_kv, d)
    gen = torch.Generator("cuda").manual_seed(tokens)
    k = torch.full(shape, float("nan"), dtype=t, device="cuda")
    v = k.clone()
    lo = torch.randn((n_pages, n_head_kv, d), generator=gen, device="cuda").to(t)
    hi = lo + 1
    new_k, new_v = (torch.randn((len(slots), n_head_kv, d), generator=gen, device="cuda") * 2 for _ in range(2))
    ds = dev(slots)
    for x in (new_k, new_v):
        x[ds < 0] = float("nan")
    rows = ds >= 0
    page, off = ds[rows] // page_size, ds[rows] % page_size
    wk, wv, wlo, whi = k.clone(), v.clone(), lo.float(), hi.float()
    kk = new_k[rows].to(t)
    wk[page, off], wv[page, off] = kk, new_v[rows].to(t)
    first = page[off == 0]
    wlo[first], whi[first] = float("inf"), -float("inf")
    wlo.index_reduce_(0, page, kk.float(), "amin")
    whi.index_reduce_(0, page, kk.float(), "amax")
    B().paged_store(B().PagedKV(k, v, lo, hi), new_k, new_v, ds)
    for name, got, want in (("k", k, wk), ("v", v, wv), ("k_lo", lo, wlo.to(t)), ("k_hi", hi, whi.to(t))):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), name


# ------------------------------------------------------------------ select

def run_select(c, q, page_size, n_sel, dtype):
    lo, hi = R.bounds_of(c)
    dk, dv = R.to_device(c, dtype)
    t = R.DTYPES[dtype]
    got = B().paged_select(B().PagedKV(dk, dv, dev(lo).to(t), dev(hi).to(t)), dev(q), i32(c["table"]), i32(c["lens"]), n_sel)
    want = R.select_ref(q, lo, hi, c["table"], c["lens"], page_size, n_sel)
    np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,page_size,heads,n_sel", [
    ([700, 31], 3, (16, 4), 60), ([700, 31, 0, 1], 3, (4, 4), 60), ([500, 77], 4, (24, 2), 20), ([2000], 1, (10, 1), 700),
    ([9000], 1, (3, 1), 33), ([330, 331, 332], 5, (34, 2), 2), ([160, 17], 1, (8, 8), 100)])
def test_select_at_head_dim_256(lens, page_size, heads, n_sel, dtype):
    r = rng(sum(lens) + n_sel)
    c = R.make_cache(r, lens, page_size, heads[1], 256, dtype)
    q = r.standard_normal((len(lens), heads[0], 256)).astype(np.float32)
    run_select(c, q, page_size, n_sel, dtype)
    q *= 2.0 ** -130  # below the range in which the scores are scaled exactly
    run_select(c, q, page_size, n_sel, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [300, 2000])
@pytest.mark.parametrize("kinds", [1, 3])
def test_select_crowds_of_equal_scores_at_head_dim_256(n, kinds, dtype):
    """Blocks that only the 64-bit scores and their numbers tell apart, ranked in
    shared memory (300) and by bisection (2000)."""
    r = rng(n + kinds)
    c = R.make_cache(r, [n], 1, 1, 256, dtype)
    few = R.rounded(r.standard_normal((kinds, 1, 256)), dtype)
    for b in range(n):
        c["k"][c["table"][0, b], 0] = few[r.integers(kinds)]
    q = r.standard_normal((1, 11, 256)).astype(np.float32)
    for n_sel in (2, n // 3, n - 1):
        run_select(c, q, 1, n_sel, dtype)


def test_select_scores_that_differ_in_the_last_bits_at_head_dim_256():
    r = rng(19)
    for dtype, step in (("f16", 2.0 ** -10), ("bf16", 2.0 ** -7)):
        c = R.make_cache(r, [500], 1, 1, 256, dtype)
        base = R.rounded(1 + r.random(256) * 0.9, dtype)
        for b in range(500):
            row = base.copy()
            row[r.integers(256)] -= step * int(r.integers(0, 3))
            c["k"][c["table"][0, b], 0, 0] = row
        q = r.standard_normal((1, 3, 256)).astype(np.float32)
        q[:, :, ::7] *= 1e-4
        for n_sel in (10, 250):
            run_select(c, q, 1, n_sel, dtype)
