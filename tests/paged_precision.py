"""How near the paged attention comes to 64 bits: two measures with their limits,
and what the kernel's number formats alone would do to them.

Random inputs.  The measure of one (sequence, query head) is the RMS of the error
over the head dim divided by the RMS of the exact output.  A weight
w = 2^(f q.k - m) is off, relative to itself and in the RMS, by
  - the parts of q: one rounding to 22 bits per product, whose errors add up at
    random: 2^-23 of the score's standard deviation, here 2: 2.4e-7;
  - the score's additions: at most D / 16 of them (D = 256), each off by 2^-24 of a partial
    sum no larger than the score's spread, at random: 4 x 2 x 2^-24 = 4.8e-7;
  - the argument of ex2, up to 16 in size: 2^-21 / sqrt(12) = 1.4e-7; ex2
    itself 2^-22 / sqrt(3) = 1.4e-7; the parts of w the same.
In quadrature 6e-7.  The errors of different positions are independent, so
sum w v carries the same share of its own RMS; a head where few weights matter
may have three times that: LIMIT is 2^-19 = 1.9e-6.  With one f16 part less it
would be 14 times LIMIT or more; bf16's third part is too small to show here.

One channel.  Sequence s has 16 cached tokens; the queries are zero but for
channel s (all channels in turn), the keys there 0 for the first token and -1
for the others, the first value is zero.  Every head's weights are then 1 and
w0 = exp(-scale q), known exactly, and every output is w0 (sum v) / (1 + 15 w0):
an error of q's or w's parts shows undiluted.  With u = 2^-24, p = 2^-22 what two
f16 parts leave out (three bf16 parts: nothing) and a = scale q: the score is off by a (p + 6 u) (the
product is exact, f takes four roundings, the argument two); w0 by ex2's 4 u and
by p.  The values are between 0.5 and 1.5, so the largest of the 15 products is
at most a fifth of their sum: two instructions that truncate 17 terms to 2^-24 of
the largest are off by 7 u, joining their sums by 2 u, the sum of the weights by 5 u,
the division and the product with it by 2 u; in all fewer than 20 u.  A part less
of q or of w, where it leaves out more than 0.6 of 2^-17 (f16: 2^-12) of the
value, is off by more than 1.5 times the limit."""
import numpy as np
import torch

import paged_ref as R

LIMIT = 2.0 ** -19

# (lengths, page size, query heads, KV heads, head dim)
CASES = [([300, 90], 16, 12, 2, 128), ([4160], 16, 8, 1, 128), ([900], 24, 24, 2, 64), ([700], 16, 16, 4, 256),
         ([1000], 16, 16, 1, 128), ([20000], 16, 4, 1, 64), ([9000], 64, 12, 1, 128)]


def inputs(r, lens, page_size, hq, hkv, d, dtype):
    c = R.make_cache(r, lens, page_size, hkv, d, dtype)
    return c, r.standard_normal((len(lens), hq, d)).astype(np.float32) * 2


def parts(x, dtype, n):
    """x as the sum of n values of the type, each the rounding of what is left."""
    t = R.DTYPES[dtype]
    left, total = torch.from_numpy(np.ascontiguousarray(x, np.float64)), 0.0
    for _ in range(n):
        p = left.float().to(t).double()
        total, left = total + p, left - p
    return total.numpy()


def attend(c, q, page_size, scale, dtype=None, q_parts=None, w_parts=None):
    """Attention in 64 bits; with q (scaled to [1, 2) per head) or the weights
    (times 2^12 for f16) replaced by so many parts of the type."""
    n_seq, n_head, d = q.shape
    hkv = c["k"].shape[2]
    group = n_head // hkv
    out = np.zeros(q.shape)
    for s in range(n_seq):
        n = int(c["lens"][s])
        pos = np.arange(n)
        page = c["table"][s, pos // page_size]
        for h in range(hkv):
            k, v = c["k"][page, pos % page_size, h], c["v"][page, pos % page_size, h]
            qs = q[s, h * group:(h + 1) * group].astype(np.float64)
            if q_parts:
                up = 2.0 ** -np.floor(np.log2(np.abs(qs).max(-1, keepdims=True)))
                qs = parts(qs * up, dtype, q_parts) / up
            x = qs @ k.T * scale
            w = np.exp(x - x.max(-1, keepdims=True))
            total = w.sum(-1, keepdims=True)
            if w_parts:
                up = 4096.0 if dtype == "f16" else 1.0
                w = parts(w * up, dtype, w_parts) / up
            out[s, h * group:(h + 1) * group] = w @ v / total
    return out


def off(got, want):
    """The measure, per (sequence, query head)."""
    return np.sqrt(((got - want) ** 2).mean(-1) / (want ** 2).mean(-1))


# (query heads, KV heads, head dim): one and two groups of 8 heads a pass
ONE_SHAPES = [(12, 2, 128), (24, 2, 64), (16, 1, 128), (4, 2, 256), (8, 1, 64)]
PARTS = {"f16": 2, "bf16": 3}


def remainder(x, dtype):
    """What one part less leaves out of x, relative to x, in units of 2^-12
    (f16) or 2^-17 (bf16)."""
    return np.abs(x - parts(x, dtype, PARTS[dtype] - 1)) / x * (2.0 ** 12 if dtype == "f16" else 2.0 ** 17)


def one_channel(r, hq, hkv, d, dtype, a):
    """(cache, q, scale, exact, limit): scores of 0 and about -a.  Of the
    candidates for a query's one entry those are taken whose own remainder
    (a > 2) or whose weight's (a <= 2) is large."""
    scale = np.float32(a / 1.5)
    c = R.make_cache(r, [16] * d, 16, hkv, d, dtype, extra_pages=0)
    q = np.zeros((d, hq, d), np.float32)
    some = (1 + r.random(40000)).astype(np.float32)
    w0 = np.exp(-some.astype(np.float64) * float(scale))
    left = remainder(some.astype(np.float64), dtype) if a > 2 else remainder(w0 * (4096 if dtype == "f16" else 1), dtype)
    some = some[(left > 0.6) & (left < 0.9)]
    for s in range(d):
        q[s, :, s] = r.choice(some, hq, replace=False)
        page = c["table"][s, 0]
        c["k"][page, 0, :, s], c["k"][page, 1:, :, s] = 0.0, -1.0
        c["v"][page] = R.rounded(0.5 + r.random((16, hkv, d)), dtype)
        c["v"][page, 0] = 0.0
    v = np.stack([c["v"][c["table"][s, 0]] for s in range(d)])  # [sequence, token, KV head, dim]
    v = np.repeat(v, hq // hkv, 2)
    q0 = q[np.arange(d), :, np.arange(d)].astype(np.float64)
    w = np.exp(-q0 * float(scale))[..., None]
    want = w * v.sum(1) / (1 + 15 * w)
    u, p = 2.0 ** -24, 2.0 ** -22 if dtype == "f16" else 0.0
    rel = float(scale) * 2 * (p + 6 * u) + 24 * u + p
    limit = want * rel
    return c, q, float(scale), want, limit
