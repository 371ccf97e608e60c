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
