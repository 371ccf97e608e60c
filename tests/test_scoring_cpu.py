"""Argument checks of chunk attention, forks, copies and log probabilities,
without a device: a refused call touches no memory and launches nothing, so
made-up addresses serve as pointers."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_ref as R
from chunk_ref import fork_ref
from test_paged_cpu import BAD_KV, PTR, UNSUPPORTED_KV, B, kv_struct

# A call that is not refused would use the made-up addresses: never where there
# is a device to use them.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must not reach a device")

FAR = PTR + (1 << 20)
PREFILL = dict(q=PTR, q_stride=512, n_tokens=3, n_head=4, block_table=PTR, table_stride=4, n_seq=2, max_blocks=4,
               seq_lens=PTR, cu=PTR, mask=None, mask_stride=0, window=0, scale=1.0, out=FAR, workspace=PTR,
               workspace_size=1 << 40, stream=None)


def prefill(kv=None, **over):
    kv = kv_struct() if kv is None else kv
    return B().lib().b200_paged_prefill(C.byref(kv), *{**PREFILL, **over}.values())


@pytest.mark.parametrize("over", [
    dict(q=None), dict(q=PTR + 8), dict(q_stride=508), dict(q_stride=504), dict(n_tokens=-1), dict(n_head=0),
    dict(n_head=3), dict(n_head=65538), dict(block_table=None), dict(table_stride=3), dict(n_seq=-1),
    dict(n_seq=65536), dict(max_blocks=0), dict(max_blocks=1 << 28, table_stride=1 << 28), dict(seq_lens=None),
    dict(cu=None), dict(mask=PTR + 1, mask_stride=64), dict(mask=PTR, mask_stride=63), dict(window=-1),
    dict(out=None), dict(out=FAR + 8), dict(workspace=None), dict(workspace=PTR + 8), dict(workspace_size=8),
    dict(out=PTR), dict(out=PTR + 1024), dict(out=PTR - 3 * 1024 + 16), dict(q_stride=1 << 62)])
def test_prefill_refuses(over):
    assert prefill(**over) == B().EINVAL


def test_prefill_refuses_more_rows_than_it_counts():
    assert prefill(n_tokens=1 << 29, out=PTR + (1 << 45)) == B().EUNSUPPORTED
    assert prefill(max_blocks=(1 << 27) - 1, table_stride=1 << 27) == B().EUNSUPPORTED  # the last tile passes 2^31
    assert prefill(scale=float("nan")) == B().EINVAL


def test_prefill_refuses_rows_that_its_last_tiles_would_count_past():
    """Rows are counted in int up to two tiles of 128 from the last one on."""
    far = PTR + (1 << 45)
    for n_tokens, n_head in [((1 << 31) // 4 - 1, 4), ((1 << 31) // 4 - 64, 4), ((1 << 31) // 2 - 100, 2)]:
        assert prefill(n_tokens=n_tokens, n_head=n_head, out=far) == B().EUNSUPPORTED


@pytest.mark.parametrize("over", BAD_KV)
def test_bad_cache_is_refused(over):
    kv = kv_struct(**over)
    assert prefill(kv) == B().EINVAL
    assert B().lib().b200_paged_copy(C.byref(kv), PTR, PTR, None, 3, None) == B().EINVAL


@pytest.mark.parametrize("over", UNSUPPORTED_KV)
def test_unsupported_cache_is_refused(over):
    kv = kv_struct(**over)
    assert prefill(kv) == B().EUNSUPPORTED
    assert B().lib().b200_paged_copy(C.byref(kv), PTR, PTR, None, 3, None) == B().EUNSUPPORTED


FORK = dict(src=PTR, keep=PTR, seq_lens=PTR, n_seq=2, block_table=PTR, table_stride=4, max_blocks=4, page_size=16,
            free_pages=PTR, n_pages=8, n_free=PTR, table_out=PTR, table_out_stride=4, seq_lens_out=PTR, n_free_out=PTR,
            copy_src=PTR, copy_dst=PTR, copy_rows=PTR, workspace=PTR, workspace_size=1 << 40, stream=None)


@pytest.mark.parametrize("over", [{k: None} for k in FORK if FORK[k] == PTR] + [
    dict(n_seq=0), dict(n_seq=-1), dict(table_stride=3), dict(table_out_stride=3), dict(max_blocks=0),
    dict(page_size=0), dict(n_pages=0), dict(n_pages=1 << 28), dict(max_blocks=1 << 28, table_stride=1 << 28),
    dict(workspace=PTR + 4), dict(workspace_size=100), dict(table_out=PTR + 16), dict(table_out=PTR + 4),
    dict(table_out_stride=8), dict(table_out=PTR - 16)])
def test_fork_refuses(over):
    assert B().lib().b200_paged_fork(*{**FORK, **over}.values()) == B().EINVAL


def test_fork_takes_tables_that_stand_between_each_others_rows():
    """Two parts of one tensor: apart, whichever comes first, as long as no entry is in both
    (no device here: a call that is not refused ends with a CUDA error)."""
    def fork(at, stride, blocks=4):
        over = dict(table_out=PTR + 4 * at, table_stride=stride, table_out_stride=stride, max_blocks=blocks)
        return B().lib().b200_paged_fork(*{**FORK, **over}.values())

    for at, stride in [(4, 8), (-4, 8), (5, 9), (4, 9), (-4, 9), (12, 8), (6, 10)]:
        assert fork(at, stride) not in (B().OK, B().EINVAL), (at, stride)
    for at, stride in [(3, 8), (5, 8), (-3, 8), (-5, 8), (3, 9), (6, 9), (4, 7), (2, 100), (-2, 100), (8, 8), (0, 8)]:
        if at:
            assert fork(at, stride) == B().EINVAL, (at, stride)


def test_fork_refuses_more_entries_than_it_counts():
    a = {**FORK, "n_seq": 1 << 16, "max_blocks": 1 << 16, "table_stride": 1 << 16, "table_out_stride": 1 << 16}
    assert B().lib().b200_paged_fork(*a.values()) == B().EUNSUPPORTED
    for bad in [(0, 4, 8), (2, 0, 8), (2, 4, 0), (1 << 16, 1 << 16, 8), (2, 4, 1 << 31)]:
        assert B().paged_fork_workspace_size(*bad) == 0
    assert B().paged_fork_workspace_size(2, 4, 8) >= 8 * 10


def test_copy_refuses():
    L = B().lib()
    kv = kv_struct()
    for args in [(None, PTR, PTR, 3), (PTR, None, PTR, 3), (PTR, PTR, None, -1), (PTR, PTR, None, 1 << 31)]:
        assert L.b200_paged_copy(C.byref(kv), *args, None) == B().EINVAL
    assert L.b200_paged_copy(C.byref(kv), None, None, None, 0, None) == B().OK
    kv = kv_struct(n_head_kv=65536, k_head=0, v_head=0)
    assert L.b200_paged_copy(C.byref(kv), PTR, PTR, None, 1, None) == B().EINVAL


LOGPROBS = dict(logits=PTR, type=0, ld=100, n_rows=2, n_vocab=100, tokens=PTR, k=3, logprob=PTR, entropy=PTR,
                top_ids=PTR, top_logprobs=PTR, stream=None)


@pytest.mark.parametrize("over", [
    dict(logits=None), dict(logits=PTR + 2), dict(ld=99), dict(n_rows=-1), dict(n_vocab=0), dict(n_vocab=2**31 - 1),
    dict(tokens=None), dict(logprob=None), dict(k=-1), dict(k=33), dict(n_vocab=2), dict(k=0), dict(top_ids=None),
    dict(top_logprobs=None), dict(ld=1 << 62), dict(type=1, logits=PTR + 1)])
def test_logprobs_refuses(over):
    assert B().lib().b200_token_logprobs(*{**LOGPROBS, **over}.values()) == B().EINVAL


def test_logprobs_types_and_empty_calls():
    L = B().lib()
    for t in (2, 8, 99, -1):
        assert L.b200_token_logprobs(*{**LOGPROBS, "type": t}.values()) == B().EUNSUPPORTED
    assert L.b200_token_logprobs(*{**LOGPROBS, "n_rows": 0}.values()) == B().OK
    assert prefill(n_seq=0) == prefill(n_tokens=0) == B().OK


def test_workspace_sizes():
    bw = B()
    for bad in [(96, 1, 1, 4, 2), (128, -1, 1, 4, 2), (128, 1, -1, 4, 2), (128, 1, 65536, 4, 2), (128, 1, 1, 0, 2),
                (128, 1, 1, 4, 0), (128, 1, 1, 5, 2), (128, 1 << 31, 1, 4, 2)]:
        assert bw.paged_prefill_workspace_size(*bad) == 0
    assert all(bw.paged_prefill_workspace_size(d, t, 3, 64, 8) > 0 for d in (64, 128, 256) for t in (1, 8192))


def test_python_layer_refuses_host_tensors():
    bw = B()
    x = torch.zeros((2, 10))
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: bw.token_logprobs(x), lambda: bw.paged_fork(i, i, i, torch.zeros((2, 4), dtype=torch.int32),
                                                                     i, i[:1], 16)):
        with pytest.raises(bw.B200Error) as e:
            call()
        assert e.value.code == bw.EINVAL


def test_fork_reference_keeps_every_page_once():
    """The reference itself: no page is lost or handed out twice, and a page that
    receives tokens has one row."""
    r = np.random.default_rng(4)
    n, ps, width, n_pages = 9, 4, 8, 50
    lens, table = np.zeros(n, np.int32), np.full((n, width), -1, np.int32)
    stack, top = r.permutation(n_pages).astype(np.int32), n_pages
    for _ in range(300):
        new = r.choice([0, 0, 1, 1, 3, 9], n).astype(np.int32)
        *_, lens, top, table, stack = R.plan_ref(new, lens, table, stack, top, ps, int(new.sum()))[2:]
        src = np.where(r.random(n) < 0.7, np.arange(n), r.integers(-1, n, n))
        table, lens, top, stack, copies = fork_ref(src, r.integers(0, 40, n), lens, table, stack, top, ps)
        rows = [[int(p) for p in table[i, : R.ceil_div(int(m), ps)]] for i, m in enumerate(lens)]
        held, free = {p for row in rows for p in row}, [int(p) for p in stack[:top]]
        assert len(set(free)) == len(free) and not held & set(free) and len(held) + len(free) == n_pages
        for i, m in enumerate(lens):
            assert m % ps == 0 or sum(rows[i][-1] in row for row in rows) == 1
        assert not set(copies[0][copies[0] >= 0]) & set(copies[1][copies[1] >= 0])
