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
