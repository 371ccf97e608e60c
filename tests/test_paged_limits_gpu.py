"""Paged cache operators at the ends of their ranges, and what their
documentation allows beyond the ordinary call."""
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


@pytest.mark.parametrize("max_tokens", [2**31 - 2, 2**31 - 4096])
def test_plan_with_the_most_token_rows(max_tokens):
    """26 GB of slots and positions: the last steps over the rows end, and
    every row behind the first sequence says -1 (the second one's position 5 lies
    in a block whose page is -1: recorded, never followed)."""
    free = torch.cuda.mem_get_info()[0]
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    slots = torch.zeros(max_tokens, dtype=torch.int64, device="cuda")
    positions = torch.zeros(max_tokens, dtype=torch.int32, device="cuda")
    p = B().paged_plan(i32([3, 2]), i32([0, 5]), i32([[-1, -1], [2, -1]]), i32([0, 1, -1, -1]), i32([2]), 4, max_tokens,
                       slots=slots, positions=positions)
    assert B().device_status(reset=True) == 2
    assert p.slots[:6].tolist() == [4, 5, 6, -1, -1, -1] and p.positions[:6].tolist() == [0, 1, 2, -1, -1, -1]
    assert p.seq_lens.tolist() == [3, 7] and p.cu.tolist() == [0, 3, 5] and p.n_free.tolist() == [1]
    for at in range(5, max_tokens, 1 << 28):
        assert bool((slots[at:at + (1 << 28)] == -1).all()) and bool((positions[at:at + (1 << 28)] == -1).all()), at
    del slots, positions, p
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n_seq", [2, 5, 140])
def test_one_row_of_table_and_mask_for_every_sequence(n_seq):
    """Expanded tensors (row stride 0): many queries of one cached prompt, one
    mask for the whole batch; the same bits as with rows written out."""
    bw = B()
    r = rng(n_seq)
    ps, d = 16, 64
    c = R.make_cache(r, [300], ps, 2, d, "f16")
    dk, dv = R.to_device(c, "f16")
    lo, hi = R.bounds_of(c)
    cache = bw.PagedKV(dk, dv, dev(lo).half(), dev(hi).half())
    q = r.standard_normal((n_seq, 8, d)).astype(np.float32)
    lens = r.integers(0, 301, n_seq).astype(np.int32)
    width = c["table"].shape[1]
    mask = r.standard_normal((1, width * ps)).astype(np.float16)
    mask[0, ::3] = -np.inf
    table = i32(c["table"]).expand(n_seq, width)
    full = table.contiguous()
    dmask = dev(mask).expand(n_seq, width * ps)
    assert table.stride(0) == dmask.stride(0) == 0 and full.stride(0) == width
    dq, dl = dev(q), i32(lens)
    for m, fm in ((None, None), (dmask, dmask.contiguous())):
        for sel in (None, bw.paged_select(cache, dq, table, dl, 4)):
            got = bw.paged_attn(cache, dq, table, dl, 0.125, mask=m, sel=sel)
            assert torch.equal(got, bw.paged_attn(cache, dq, full, dl, 0.125, mask=fm, sel=sel))
    assert torch.equal(bw.paged_select(cache, dq, table, dl, 4), bw.paged_select(cache, dq, full, dl, 4))
    want, tol = R.attn_ref(dict(c, table=np.repeat(c["table"], n_seq, 0), lens=lens), q, ps, 0.125,
                           np.repeat(mask, n_seq, 0))
    got = bw.paged_attn(cache, dq, table, dl, 0.125, mask=dmask).cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
