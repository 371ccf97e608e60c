"""token_logprobs against 64 bits: ids exactly, log probabilities and entropies
within a bound counted in roundings."""
import math

import numpy as np
import pytest

from chunk_ref import logprobs_ref
from helpers import rng

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def B():
    import b200_decode

    return b200_decode


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert B().device_status(reset=True) == 0


def check(x, tokens, k):
    """Bound: with t = x - M (one rounding of |t|, and one of its product with
    log2 e: 2 u |t| in the exponent) and ex2's 2 units, a term of the sums is off
    by (2 |t| + 8) u of itself; e^t |t| is below 0.37 and e^t t^2 below 0.55, so
    sums are off by the terms' (8 u + 2 u |t|) weighted with e^t, plus adding n terms in
    chains of at most ceil(n / 512) + 16 additions.  log(n1) + log1p(s / n1) then
    moves by that share of s / (n1 + s) and adds 4 roundings of itself; t itself
    is rounded once and so is the difference."""
    r = B().token_logprobs(x, tokens, k)
    y = x.double()
    lp, ent, ids, top = logprobs_ref(y, tokens, k)
    m = y.amax(1, keepdim=True)
    t = torch.where(y == -math.inf, 0.0, y - m)
    e = torch.where(y == -math.inf, 0.0, t.exp())
    n = x.shape[1]
    chain = n / 512 + 16
    z = e.sum(1)
    others_sum = (e * (t != 0)).sum(1)
    others = ((e * (t != 0)) * (8 + 2 * t.abs() + chain)).sum(1) / z * U
    top1 = (e * (t == 0)).sum(1)
    lse = top1.log() + (others_sum / top1).log1p()
    tol_lse = others + 4 * U * lse
    tol = lambda v: tol_lse + 2 * U * (v.abs() + lse)  # noqa: E731
    weighted = ((e * t.abs()) * (12 + 2 * t.abs() + chain)).sum(1) / z * U
    tol_ent = tol_lse + weighted + (others + 4 * U) * ((e * t.abs()).sum(1) / z) + 2 * U * ent
    seen = torch.isfinite(lp)
    assert torch.equal(torch.where(seen, 0.0, r.logprob.double()), torch.where(seen, 0.0, lp))
    assert ((r.logprob.double() - lp).abs()[seen] <= tol(lp)[seen] + 1e-37).all()
    assert ((r.entropy.double() - ent).abs() <= tol_ent + 1e-37).all()
    if k:
        assert torch.equal(r.top_ids, ids)
        fine = torch.isfinite(top)
        off = (r.top_logprobs.double() - top).abs()
        assert (off[fine] <= (tol_lse[:, None] + 2 * U * (top.abs() + lse[:, None]) + 1e-37)[fine]).all()
        assert torch.equal(torch.where(fine, 0.0, r.top_logprobs.double()), torch.where(fine, 0.0, top))
    else:
        assert r.top_ids is None and r.top_logprobs is None


def logits(r, rows, vocab, dtype, scale=3.0):
    x = torch.from_numpy((r.standard_normal((rows, vocab)) * scale).astype(np.float32)).cuda().to(DTYPES[dtype])
    return x, torch.from_numpy(r.integers(-1, vocab, rows).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 33), (5, 511), (1, 4096), (7, 8191), (1, 128256),
                                        (2, 151936), (40, 151936), (400, 5003), (1000, 777), (70000, 40)])
def test_rows(rows, vocab, dtype):
    r = rng(rows + vocab)
    x, t = logits(r, rows, vocab, dtype)
    for k in sorted({0, 1, min(7, vocab), min(32, vocab)}):
        check(x, t, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5])
def test_strided_and_unaligned_rows(shift, dtype):
    r = rng(shift)
    for vocab in (3, 9, 1001, 20011):
        x, t = logits(r, 9, vocab + 9, dtype)
        check(x[:, shift:shift + vocab], t.clamp(max=vocab - 1), min(5, vocab))


def test_banned_tokens_ties_and_confident_rows():
    r = rng(2)
    x, t = logits(r, 6, 50021, "f32")
    x[0, ::2] = -math.inf
    x[1] = 1.25                                # all equal: the lowest ids
    x[2, 1:] = -math.inf                       # one token
    x[3, 777] = 60.0                           # nearly all of it: log p = -1e-20
    x[4, 100:160] = 9.0                        # more ties than k
    x[5] = torch.round(x[5] * 2) / 2           # ties everywhere, zeros of both signs
    x[5, ::7] *= -0.0
    t[:] = torch.tensor([1, 40000, 0, 777, 130, -1], dtype=torch.int32)
    for k in (0, 1, 20, 32):
        check(x, t, k)
    got = B().token_logprobs(x, t, 1)
    assert -1e-15 < got.logprob[3].item() < 0 and got.logprob[2].item() == 0 and got.entropy[2].item() == 0
    assert got.logprob[5].item() == 0


@pytest.mark.parametrize("order", ["up", "down", "clustered", "striped"])
def test_adversarial_orders(order):
    """The largest logits in ascending or descending order, all with one thread,
    or in every thread's last vector."""
    r = rng(3)
    for rows, vocab in ((1, 65536), (300, 20000)):
        x, t = logits(r, rows, vocab, "f32")
        if order == "up":
            x = x.sort(1).values
        elif order == "down":
            x = x.sort(1, descending=True).values
        elif order == "clustered":  # 40 of them 2048 logits apart: one thread's vectors
            x[:, 5:5 + 2048 * (vocab // 2048):2048] += 50
        else:
            x[:, -3000:] += 50
        check(x.contiguous(), t, 32)


def test_rows_without_a_distribution():
    r = rng(4)
    x, t = logits(r, 5, 3000, "f32")
    t[:] = 5
    x[0] = -math.inf
    x[1, 17] = math.nan
    x[2, 18] = math.inf
    x[3, 5] = -math.inf
    x[4, ::2] = math.nan
    x[4, 1::2] = -math.inf
    got = B().token_logprobs(x, t, 4)
    for i in (0, 1, 2, 4):
        assert got.logprob[i].isnan() and got.entropy[i].isnan() and got.top_logprobs[i].isnan().all()
    assert got.logprob[3] == -math.inf and got.entropy[3].isfinite()
    assert got.top_ids[0].tolist() == [0, 1, 2, 3] and got.top_ids[4].tolist() == [1, 3, 5, 7]
    assert got.top_ids[2, 0].item() == 18 and 17 not in got.top_ids[1].tolist()
    want = logprobs_ref(x.double(), t, 4)[2]
    assert torch.equal(got.top_ids, want)
    x = torch.full((1, 20), math.nan, device="cuda")
    assert B().token_logprobs(x, None, 3).top_ids.tolist() == [[0, 1, 2]]


def test_tokens_past_the_vocabulary_are_recorded():
    x = torch.zeros((2, 10), device="cuda")
    got = B().token_logprobs(x, torch.tensor([10, 3], dtype=torch.int32, device="cuda"), 0)
    assert B().device_status(reset=True) == 2
    assert got.logprob[0].item() == 0 and abs(got.logprob[1].item() + math.log(10)) < 1e-6


def test_refusals():
    bw = B()
    x = torch.zeros((2, 10), device="cuda")
    for bad in (dict(k=11), dict(k=-1), dict(tokens=torch.zeros(2, device="cuda")),
                dict(tokens=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(bw.B200Error) as e:
            bw.token_logprobs(x, **bad)
        assert e.value.code == bw.EINVAL
    with pytest.raises(bw.B200Unsupported):
        bw.token_logprobs(x.double())
    with pytest.raises(bw.B200Error):
        bw.token_logprobs(x.T)
    assert bw.token_logprobs(x[:0], None, 3).top_ids.shape == (0, 3)
    assert bw.token_logprobs(x[:1].expand(4, -1), None, 1).top_ids.tolist() == [[0]] * 4


def test_captured_and_replayed():
    r = rng(6)
    x, t = logits(r, 3, 128256, "f32")
    g = torch.cuda.CUDAGraph()
    B().token_logprobs(x, t, 20)
    with torch.cuda.graph(g):
        got = B().token_logprobs(x, t, 20)
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        g.replay()
        want = logprobs_ref(x.double(), t, 20)
        assert torch.equal(got.top_ids, want[2]) and (got.logprob.double() - want[0]).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k", [1, 4, 20, 32])
@pytest.mark.parametrize("rows", [1, 700])
def test_alternatives_that_share_threads(rows, k, dtype):
    """The largest logits in one vector, in one thread's vectors, in neighbours, and
    mixes of these with ties, at every rank where one kind gives way to another."""
    r = rng(7 * k + rows)
    vocab, vec = 128 * 256, 16 // (4 if dtype == "f32" else 2)
    x, tokens = logits(r, rows, vocab, dtype, 1.0)
    stride = 256 * vec  # of a thread's vectors
    for i in range(rows):
        near = int(r.integers(0, 256)) * vec
        n = int(r.integers(1, k + 1))
        places = [near + np.arange(vec),  # one vector
                  near + stride * np.arange(min(k, vocab // stride)),  # one thread
                  near + vec * np.arange(k),  # a thread each
                  np.concatenate([near + stride * np.arange(min(n, vocab // stride)), near + vec * np.arange(1, k - n + 1)])]
        at = places[i % 4] % vocab
        high = np.full(len(at), 8.0) if i % 3 == 0 else 8.0 + np.arange(len(at)) * 0.125 * (-1) ** (i % 2)
        x[i, torch.from_numpy(at).cuda()] = torch.from_numpy(high.astype(np.float32)).cuda().to(x.dtype)
    check(x, tokens, k)
