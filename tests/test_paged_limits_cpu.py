"""Limits of the paged cache's arithmetic that need no device: sizes at which a
check or an index could wrap around."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

# A call that is not refused would use made-up addresses: never where there is a
# device to use them.
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must not reach a device")

PTR = 4096


def B():
    import b200_decode

    return b200_decode


@no_device
@pytest.mark.parametrize("over", [
    dict(page_size=(1 << 29) + 1, n_pages=1, k_row=1 << 35, v_row=1 << 35),
    dict(page_size=(1 << 29) + 1, n_pages=1, k_row=1 << 35, v_row=3 << 34),
    dict(n_head_kv=(1 << 29) + 1, k_head=1 << 35, v_head=1 << 35),
    dict(page_size=(1 << 29) + 1, n_pages=2, k_row=1 << 35, v_row=1 << 35, k_page=0, v_page=0),
    dict(n_pages=(1 << 27) - 2, k_page=1 << 35, v_page=1 << 35)])
def test_cache_spans_past_64_bits_are_refused(over):
    """Rows and heads whose last byte lies past 2^63 of the first: the sum must
    not wrap around to a span that looks small."""
    bw = B()
    f = dict(type=bw.TYPE_F16, head_dim=128, n_head_kv=2, page_size=16, n_pages=8, k=PTR, v=PTR, k_page=16 * 512,
             k_row=512, k_head=256, v_page=16 * 512, v_row=512, v_head=256, k_lo=PTR, k_hi=PTR)
    f.update(over)
    kv = bw._PagedKVStruct(*[f[n] for n, _ in bw._PagedKVStruct._fields_])
    L, ref = bw.lib(), C.byref(kv)
    assert [L.b200_paged_store(ref, PTR, 256, PTR, 256, PTR, 3, None),
            L.b200_paged_select(ref, PTR, 512, 2, 4, PTR, 4, 4, PTR, 2, PTR, PTR, 1 << 20, None),
            L.b200_paged_attn(ref, PTR, 512, 2, 4, PTR, 4, 4, PTR, None, 0, None, 0, 1.0, PTR, PTR, 1 << 30, None)
            ] == [bw.EUNSUPPORTED] * 3
