"""Forks of block tables and copies of pages against chunk_ref.fork_ref: every
integer and every bit."""
import numpy as np
import pytest

import paged_ref as R
from chunk_ref import fork_ref
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


def state(r, n, ps, width, n_pages, max_len):
    order = r.permutation(n_pages).astype(np.int32)
    table = r.integers(-5, 0, (n, width)).astype(np.int32)
    lens = np.zeros(n, np.int32)
    at = 0
    for s in range(n):
        m = int(r.integers(0, max_len + 1))
        b = R.ceil_div(m, ps)
        if b > width or at + b > n_pages:
            continue
        table[s, :b] = order[at:at + b]
        lens[s] = m
        at += b
    stack = np.full(n_pages, -7, np.int32)
    stack[: n_pages - at] = order[at:]
    return lens, table, stack, n_pages - at


def run(src, keep, lens, table, stack, top, ps, in_place, gap=0):
    n, width = table.shape
    wide = torch.full((n, width + gap), 99, dtype=torch.int32, device="cuda")
    wide[:, :width] = i32(table)
    t = wide[:, :width]
    d = dict(src=i32(src), keep=i32(keep), seq_lens=i32(lens), block_table=t, free_pages=i32(stack), n_free=i32([top]))
    kw = {}
    if not in_place:
        kw = dict(table_out=torch.full((n, width), 55, dtype=torch.int32, device="cuda"),
                  seq_lens_out=torch.full_like(d["seq_lens"], -9), n_free_out=torch.full_like(d["n_free"], -9))
    size = B().paged_fork_workspace_size(n, width, len(stack))
    ws = torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda")
    f = B().paged_fork(page_size=ps, workspace=ws, **d, **kw)
    if gap:
        assert (wide[:, width:] == 99).all()
    if not in_place:
        assert torch.equal(t, i32(table))
    got = [f.block_table, f.seq_lens, f.n_free, d["free_pages"], torch.stack([f.copy_src, f.copy_dst, f.copy_rows])]
    return [x.cpu().numpy() for x in got]


def check(src, keep, lens, table, stack, top, ps, in_place=False, gap=0):
    src, keep = np.asarray(src, np.int32), np.asarray(keep, np.int32)
    want = fork_ref(src, keep, lens, table, stack, top, ps)
    got = run(src, keep, lens, table, stack, top, ps, in_place, gap)
    for name, g, w in zip(("table", "seq_lens", "n_free", "free_pages", "copies"), got, want):
        np.testing.assert_array_equal(g, np.asarray(w).reshape(g.shape), err_msg=name)
    return want


def owners(table, lens, stack, top, ps, n_pages):
    """No page is lost, none is both free and held, and a page that receives
    tokens has one row."""
    held, parts = set(), []
    for i, m in enumerate(lens):
        row = [int(p) for p in table[i, : R.ceil_div(int(m), ps)]]
        held |= set(row)
        if m % ps:
            parts.append(row[-1])
    free = [int(p) for p in stack[:top]]
    assert len(free) == len(set(free)) and not held & set(free) and len(held) + len(free) == n_pages
    for p in parts:
        assert sum(int(p) in [int(x) for x in table[i, : R.ceil_div(int(m), ps)]] for i, m in enumerate(lens)) == 1


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,ps,max_len", [(1, 16, 40), (2, 1, 5), (4, 5, 30), (64, 16, 900), (257, 24, 300),
                                          (1024, 16, 100), (1500, 7, 60), (9, 16, 40000)])
def test_random_forks_and_the_steps_after_them(n, ps, max_len, in_place):
    r = rng(n + ps)
    width = R.ceil_div(max_len, ps) + 1
    n_pages = n * width + 3
    lens, table, stack, top = state(r, n, ps, width, n_pages, max_len)
    for step in range(4):
        src = r.integers(-1, n, n)
        stay = r.random(n) < 0.5
        src[stay] = np.arange(n)[stay]
        keep = np.where(r.random(n) < 0.5, 10**9, r.integers(-2, max_len + 2, n))
        table, lens, top, stack, _ = check(src, keep, lens, table, stack, top, ps, in_place, gap=3 * step)
        owners(table, lens, stack, top, ps, n_pages)


@pytest.mark.parametrize("second", [False, True])
def test_tables_in_two_halves_of_one_tensor(second):
    r, n, ps, width = rng(8), 33, 16, 6
    lens, table, stack, top = state(r, n, ps, width, 150, 90)
    both = torch.full((n, 2 * width), 44, dtype=torch.int32, device="cuda")
    old, new = (both[:, width:], both[:, :width]) if second else (both[:, :width], both[:, width:])
    old.copy_(i32(table))
    src, keep = r.integers(-1, n, n), r.integers(0, 90, n)
    want = fork_ref(src, keep, lens, table, stack, top, ps)
    f = B().paged_fork(i32(src), i32(keep), i32(lens), old, i32(stack), i32([top]), ps, table_out=new)
    np.testing.assert_array_equal(f.block_table.cpu().numpy(), want[0])
    np.testing.assert_array_equal(f.seq_lens.cpu().numpy(), want[1])
    assert torch.equal(old, i32(table))


def test_beams_share_all_but_their_last_page():
    lens = np.array([37, 0, 0, 0], np.int32)
    table = np.full((4, 5), -1, np.int32)
    table[0, :3] = 9, 4, 6
    stack = np.array([0, 1, 2, 3, 5, 7, 8, -1, -1, -1], np.int32)
    want = check([0, 0, 0, 0], [37] * 4, lens, table, stack, 7, 16)
    assert want[0].tolist() == [[9, 4, 6, -1, -1], [9, 4, 8, -1, -1], [9, 4, 7, -1, -1], [9, 4, 5, -1, -1]]
    # shorter forks of a full page, the owner stays: every one needs a page
    want = check([0, 0, 0, -1], [37, 20, 9, 4], lens, table, stack, 7, 16)
    assert want[4].tolist() == [[-1, 4, 9, -1], [-1, 8, 7, -1], [0, 4, 9, 0]]
    # whole blocks need none
    assert check([0, 0, -1, -1], [37, 32, 0, 0], lens, table, stack, 7, 16)[2] == 7


def test_no_page_left_ends_a_row_with_its_last_full_block():
    lens = np.array([37, 37, 5], np.int32)
    table = np.array([[0, 1, 2], [3, 4, 5], [6, -1, -1]], np.int32)
    stack = np.full(7, -1, np.int32)
    want = check([0, 0, 0], [37, 37, 37], lens, table, stack, 0, 16)  # freed pages serve them
    assert want[1].tolist() == [37, 37, 37] and want[2] == 2
    want = check([0, 1, 0], [37, 37, 37], lens, table, stack, 0, 16)  # one freed page: row 2 has it
    assert want[1].tolist() == [37, 37, 37] and want[2] == 0
    want = check([0, 0, 1], [30, 37, 37], np.array([37, 37, 0], np.int32), table, stack, 0, 16)
    assert want[1].tolist()[0] == 16  # nothing is free: row 1 keeps page 1 in full


def test_bad_pages_sources_and_lengths_are_recorded():
    lens = np.array([20, 20], np.int32)
    table = np.array([[0, 99], [1, 2]], np.int32)
    stack = np.full(4, -1, np.int32)
    stack[0] = 3
    got = run([0, 7], [20, 20], lens, table, stack, 1, 16, False)
    assert B().device_status(reset=True) == BOUNDS
    assert got[0].tolist() == [[0, 99], [-1, -1]] and got[1].tolist() == [20, 0]
    assert got[2].tolist() == [3] and got[3].tolist() == [3, 1, 2, -1]
    run([0, 1], [20, 20], np.array([20, 500], np.int32), np.array([[0, 1], [2, 3]], np.int32), stack, 0, 16, False)
    assert B().device_status(reset=True) == BOUNDS
    run([0, 1], [20, 20], lens, np.array([[0, 1], [2, 3]], np.int32), stack, 9, 16, False)
    assert B().device_status(reset=True) == BOUNDS


def test_captured_in_place_and_replayed():
    r = rng(8)
    n, ps, width = 40, 8, 30
    n_pages = n * width
    lens, table, stack, top = state(r, n, ps, width, n_pages, 200)
    bw = B()
    d = dict(src=i32(np.arange(n)), keep=i32(lens), seq_lens=i32(lens), block_table=i32(table), free_pages=i32(stack),
             n_free=i32([top]))
    ws = torch.empty(bw.paged_fork_workspace_size(n, width, n_pages), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f = bw.paged_fork(page_size=ps, workspace=ws, **d)
    for _ in range(4):
        src, keep = r.integers(-1, n, n).astype(np.int32), r.integers(0, 220, n).astype(np.int32)
        d["src"].copy_(i32(src))
        d["keep"].copy_(i32(keep))
        g.replay()
        table, lens, top, stack, copies = fork_ref(src, keep, lens, table, stack, top, ps)
        for x, y in ((f.block_table, table), (f.seq_lens, lens), (f.n_free, [top]), (d["free_pages"], stack),
                     (torch.stack([f.copy_src, f.copy_dst, f.copy_rows]), copies)):
            np.testing.assert_array_equal(x.cpu().numpy(), np.asarray(y))


# ------------------------------------------------------------------- copies

@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("bounds", [False, True])
@pytest.mark.parametrize("n,ps,h,d,dtype", [(1, 16, 2, 64, "f16"), (3, 1, 1, 128, "bf16"), (70, 5, 3, 64, "bf16"),
                                            (40, 300, 2, 256, "f16"), (300, 16, 8, 128, "f16"), (2, 2000, 1, 64, "f16")])
def test_copies(n, ps, h, d, dtype, bounds, layout):
    r = rng(n + ps + d)
    n_pages = 2 * n + 1
    c = dict(k=r.standard_normal((n_pages, ps, h, d)), v=r.standard_normal((n_pages, ps, h, d)))
    c["k"][r.random(c["k"].shape) < 0.01] = np.nan
    dk, dv = R.to_device(c, dtype, layout)
    kw = {}
    if bounds:
        kw = dict(k_lo=dk.amin(1).contiguous(), k_hi=dk.amax(1).contiguous())
    cache = B().PagedKV(dk, dv, **kw)
    order = r.permutation(n_pages)
    src, dst = np.full(n + 3, -1), np.full(n + 3, -1)
    src[1:n + 1], dst[2:n + 1] = order[:n], order[n:2 * n - 1]  # one entry without a target
    rows = r.integers(0, ps + 1, n + 3)
    for given in (None, rows):
        before = [t.clone() for t in (dk, dv)] + [t.clone() for t in kw.values()]
        B().paged_copy(cache, i32(src), i32(dst), None if given is None else i32(given))
        for i in range(n + 3):
            if src[i] >= 0 and dst[i] >= 0:
                m = ps if given is None else int(given[i])
                for x in before[:2]:
                    x[dst[i], :m] = x[src[i], :m]
                for x in before[2:]:
                    if m:
                        x[dst[i]] = x[src[i]]
        for x, y in zip((dk, dv, *kw.values()), before):
            assert torch.equal(x.contiguous().view(torch.int16), y.contiguous().view(torch.int16))
    if layout == "gap":
        whole = torch.as_strided(dk, (n_pages, ps + 1, h + 1, d + 8), dk.stride())
        assert torch.isnan(whole[:, ps]).all() and torch.isnan(whole[:, :, h]).all() and torch.isnan(whole[..., d:]).all()


def test_copies_of_bad_entries():
    k = torch.randn((4, 16, 2, 64), device="cuda").half()
    cache = B().PagedKV(k, k.clone())
    before = k.clone()
    B().paged_copy(cache, i32([0, 9, 1, 2]), i32([7, 1, 1, -3]), i32([16, 16, 16, 16]))
    assert B().device_status(reset=True) == BOUNDS
    assert torch.equal(k, before)
    B().paged_copy(cache, i32([0, 2]), i32([1, 3]), i32([99, -4]))
    assert B().device_status(reset=True) == BOUNDS
    before[1] = before[0]
    assert torch.equal(k, before)
    B().paged_copy(cache, i32([]), i32([]))
