"""Argument checks of the paged key-value cache entry points, through the C
ABI and the Python layer, without a device: a refused call touches no memory
and launches nothing, so made-up addresses serve as pointers."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_ref as R

# A call that is not refused would use the made-up addresses: never where there
# is a device to use them.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must not reach a device")

PTR = 4096  # an aligned address nothing reads


def B():
    import b200_decode

    return b200_decode


def kv_struct(**over):
    bw = B()
    f = dict(type=bw.TYPE_F16, head_dim=128, n_head_kv=2, page_size=16, n_pages=8, k=PTR, v=PTR, k_page=16 * 512,
             k_row=512, k_head=256, v_page=16 * 512, v_row=512, v_head=256, k_lo=PTR, k_hi=PTR)
    f.update(over)
    return bw._PagedKVStruct(*[f[n] for n, _ in bw._PagedKVStruct._fields_])


PLAN = dict(new_lens=PTR, seq_lens=PTR, n_seq=2, block_table=PTR, table_stride=4, max_blocks=4, page_size=16,
            free_pages=PTR, n_pages=8, n_free=PTR, max_tokens=4, slots=PTR, positions=PTR, cu=PTR, seq_lens_out=PTR,
            n_free_out=PTR, stream=None)


@pytest.mark.parametrize("over", [dict(new_lens=None), dict(seq_lens=None), dict(n_seq=0), dict(n_seq=-1),
                                  dict(block_table=None), dict(table_stride=3), dict(max_blocks=0),
                                  dict(page_size=0), dict(free_pages=None), dict(n_pages=0), dict(n_free=None),
                                  dict(max_tokens=-1), dict(slots=None), dict(positions=None), dict(cu=None),
                                  dict(seq_lens_out=None), dict(n_free_out=None),
                                  dict(max_blocks=1 << 28, table_stride=1 << 28), dict(n_pages=1 << 28),
                                  dict(max_tokens=2**31 - 1)])
def test_plan_refuses(over):
    assert B().lib().b200_paged_plan(*{**PLAN, **over}.values()) == B().EINVAL


def test_plan_refuses_more_sequences_than_it_scans():
    assert B().lib().b200_paged_plan(*{**PLAN, "n_seq": 8193}.values()) == B().EUNSUPPORTED


BAD_KV = [dict(k=None), dict(v=None), dict(n_head_kv=0), dict(page_size=0), dict(n_pages=0), dict(k=PTR + 8),
          dict(v=PTR + 2), dict(k_page=8), dict(k_row=520), dict(k_head=2), dict(v_page=-16), dict(v_row=264),
          dict(v_head=8), dict(k_lo=None), dict(k_hi=None), dict(k_lo=PTR + 8), dict(k_hi=PTR + 4),
          dict(page_size=1 << 20, n_pages=1 << 12)]
UNSUPPORTED_KV = [dict(type=0), dict(type=2), dict(type=99), dict(head_dim=96), dict(head_dim=512), dict(head_dim=0),
                  dict(k_page=1 << 36), dict(v_row=1 << 40), dict(k_page=1 << 34), dict(v_page=1 << 34),
                  dict(v_head=1 << 36), dict(n_pages=1 << 26, k_page=1 << 10)]


def calls(kv):
    L = B().lib()
    ref = None if kv is None else C.byref(kv)
    return [L.b200_paged_store(ref, PTR, 256, PTR, 256, PTR, 3, None),
            L.b200_paged_select(ref, PTR, 512, 2, 4, PTR, 4, 4, PTR, 2, PTR, PTR, 1 << 20, None),
            L.b200_paged_attn(ref, PTR, 512, 2, 4, PTR, 4, 4, PTR, None, 0, None, 0, 1.0, PTR, PTR, 1 << 30, None)]


@pytest.mark.parametrize("over", BAD_KV)
def test_bad_cache_is_refused_by_every_call(over):
    assert calls(kv_struct(**over)) == [B().EINVAL] * 3


@pytest.mark.parametrize("over", UNSUPPORTED_KV)
def test_unsupported_cache_is_refused_by_every_call(over):
    assert calls(kv_struct(**over)) == [B().EUNSUPPORTED] * 3


def test_null_cache_is_refused():
    assert calls(None) == [B().EINVAL] * 3


STORE = dict(k=PTR, k_ld=256, v=PTR, v_ld=256, slots=PTR, n_tokens=3, stream=None)


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(slots=None), dict(n_tokens=-1), dict(k=PTR + 4),
                                  dict(v=PTR + 8), dict(k_ld=255), dict(v_ld=250), dict(k_ld=252), dict(v_ld=128),
                                  dict(n_tokens=2**31)])
def test_store_refuses(over):
    kv = kv_struct()
    assert B().lib().b200_paged_store(C.byref(kv), *{**STORE, **over}.values()) == B().EINVAL


BATCH = dict(q=PTR, q_stride=512, n_seq=2, n_head=4, block_table=PTR, table_stride=4, max_blocks=4, seq_lens=PTR)
BAD_BATCH = [dict(q=None), dict(q=PTR + 4), dict(q_stride=510), dict(q_stride=508), dict(n_seq=-1),
             dict(n_seq=65536), dict(n_head=0), dict(n_head=3), dict(n_head=-2), dict(block_table=None),
             dict(table_stride=3), dict(max_blocks=0), dict(seq_lens=None),
             dict(max_blocks=1 << 28, table_stride=1 << 28)]
SELECT = dict(n_sel=2, sel=PTR, workspace=PTR, workspace_size=1024, stream=None)
ATTN = dict(mask=None, mask_stride=0, sel=None, n_sel=0, scale=1.0, out=PTR, workspace=PTR, workspace_size=1 << 30,
            stream=None)


@pytest.mark.parametrize("over", BAD_BATCH + [dict(n_sel=0), dict(n_sel=-1), dict(sel=None), dict(workspace=None),
                                              dict(workspace=PTR + 8), dict(workspace_size=1023)])
def test_select_refuses(over):
    kv = kv_struct()
    a = {**BATCH, **SELECT, **over}
    assert B().lib().b200_paged_select(C.byref(kv), *a.values()) == B().EINVAL


def test_select_refuses_a_cache_without_bounds_and_too_many_blocks():
    L = B().lib()
    kv = kv_struct(k_lo=None, k_hi=None)
    a = {**BATCH, **SELECT}
    assert L.b200_paged_select(C.byref(kv), *a.values()) == B().EINVAL
    kv = kv_struct(page_size=1, n_pages=1 << 21)
    a.update(max_blocks=(1 << 20) + 1, table_stride=1 << 21, workspace_size=1 << 40)
    assert L.b200_paged_select(C.byref(kv), *a.values()) == B().EUNSUPPORTED


@pytest.mark.parametrize("over", BAD_BATCH + [dict(out=None), dict(out=PTR + 8), dict(workspace=None),
                                              dict(workspace=PTR + 4), dict(workspace_size=8),
                                              dict(sel=PTR, n_sel=0), dict(sel=PTR, n_sel=-3),
                                              dict(mask=PTR + 1, mask_stride=64), dict(mask=PTR, mask_stride=63)])
def test_attn_refuses(over):
    kv = kv_struct()
    a = {**BATCH, **ATTN, **over}
    assert B().lib().b200_paged_attn(C.byref(kv), *a.values()) == B().EINVAL


def test_empty_batches_are_nothing_to_do():
    L = B().lib()
    kv = kv_struct()
    assert L.b200_paged_store(C.byref(kv), None, 256, None, 256, None, 0, None) == B().OK
    assert L.b200_paged_select(C.byref(kv), *{**BATCH, **SELECT, "n_seq": 0}.values()) == B().OK
    assert L.b200_paged_attn(C.byref(kv), *{**BATCH, **ATTN, "n_seq": 0}.values()) == B().OK


def test_workspace_sizes():
    bw = B()
    assert bw.paged_select_workspace_size(2, 2, 4) == 1024  # four arrays of at most 256 bytes
    assert bw.paged_select_workspace_size(16, 8, 2048) == 16 * 8 * (2048 * 12 + 128 * 4 + 8)
    assert bw.paged_select_workspace_size(-1, 2, 5) == bw.paged_select_workspace_size(3, 0, 5) == 0
    assert bw.paged_select_workspace_size(3, 2, 0) == bw.paged_select_workspace_size(1, 1, (1 << 20) + 1) == 0
    for bad in [(96, 2, 4, 2), (128, -1, 4, 2), (128, 2, 0, 2), (128, 2, 4, 0), (128, 2, 5, 2)]:
        assert bw.paged_attn_workspace_size(*bad) == 0
    sizes = [bw.paged_attn_workspace_size(d, n, 64, 8) for d in (64, 128, 256) for n in (1, 16, 4096)]
    assert all(s > 0 and s % 16 == 0 for s in sizes)


def test_python_layer_refuses_host_tensors_and_wrong_types():
    bw = B()
    k = torch.zeros((4, 16, 2, 128), dtype=torch.float16)
    with pytest.raises(bw.B200Error) as e:
        bw.PagedKV(k, k.clone())
    assert e.value.code == bw.EINVAL
    with pytest.raises(bw.B200Unsupported):
        bw.PagedKV(k.float(), k.float())
    with pytest.raises(bw.B200Error):
        bw.PagedKV(k[0], k[0])
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(bw.B200Error):
        bw.paged_plan(i, i, torch.zeros((2, 4), dtype=torch.int32), i, i[:1], 16, 4)


def test_plan_reference_gives_back_what_it_hands_out():
    """The reference allocator itself: over random steps no page is owned
    twice and none is lost."""
    r = np.random.default_rng(3)
    n, ps, width, n_pages = 7, 4, 9, 40
    lens = np.zeros(n, np.int32)
    table = np.full((n, width), -1, np.int32)
    stack, top = r.permutation(n_pages).astype(np.int32), n_pages
    for _ in range(200):
        new = r.choice([-1, 0, 1, 1, 3, 11], n).astype(np.int32)
        out = R.plan_ref(new, lens, table, stack, top, ps, int(np.maximum(new, 0).sum()))
        slots, positions, cu, lens, top, table, stack = out
        owned = [int(table[s, b]) for s in range(n) for b in range(R.ceil_div(int(lens[s]), ps))]
        assert sorted(owned + [int(p) for p in stack[:top]]) == list(range(n_pages))
        assert ((slots >= 0) == (positions >= 0)).all()
