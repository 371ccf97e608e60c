"""Plain 64-bit implementations of chunk attention, forks and log
probabilities, and how far a result in fewer bits may be off."""
import math

import numpy as np
import torch

from paged_ref import ceil_div


def chunk_ref(c, q, cu, page_size, scale, mask=None, window=0):
    """(out, bound) f64 [n_tokens, n_head, D] for q (torch, 16-bit, on the GPU)
    over a cache of paged_ref.make_cache; NaN in rows of no sequence.

    Bound per element, u = 2^-24 and h half a step of the 16-bit type relative to
    the value: scores are sums of D exact products in f32, off by at most
    A (D / 8 + 6) 2u with A = scale sum_d |q_d k_d| (as paged_ref.attn_ref has
    it), so weights by a factor 1 +- (2 A e + 16 u), doubled for numerator and
    denominator; adding n weighted values costs (n / 4 + 32) 2u; each weight is
    rounded to 16 bits before its product with V (h) and the output is
    (h |out|).  An f16 weight below 2^-14 of the reference (itself within 2^8 of
    2^7) is off by 2^-25 absolutely: less than 2^-31 of the largest weight for
    each of n values, and an f16 output below 2^-14 by 2^-25; bf16 has neither."""
    n_tokens, n_head, d = q.shape
    n_head_kv = c["k"].shape[2]
    group = n_head // n_head_kv
    dev = q.device
    half = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    u = 2.0 ** -24
    k_all, v_all = (torch.from_numpy(c[n]).to(dev) for n in "kv")
    for s in range(len(cu) - 1):
        first, n, length = int(cu[s]), int(cu[s + 1] - cu[s]), int(c["lens"][s])
        for lo in range(0, n, 256):
            hi = min(n, lo + 256)
            rows = slice(first + lo, first + hi)
            out[rows] = 0
            tol[rows] = 1e-30
            at = torch.arange(length - n + lo, length - n + hi, device=dev)
            pos = np.arange(max(0, length - n + hi))
            if mask is not None:
                pos = pos[mask[s, pos] != -np.inf]
            if pos.size == 0:
                continue
            page = torch.from_numpy(c["table"][s, pos // page_size].astype(np.int64)).to(dev)
            p = torch.from_numpy(pos).to(dev)
            see = p <= at[:, None]
            if window:
                see &= p > (at - window)[:, None]
            some = see.any(1)
            for h in range(n_head_kv):
                heads = slice(h * group, (h + 1) * group)
                k, v = k_all[page, p % page_size, h], v_all[page, p % page_size, h]
                qs = q[rows, heads].double()
                x = qs @ k.T * scale
                if mask is not None:
                    x = x + torch.from_numpy(mask[s, pos].astype(np.float64)).to(dev)
                x = torch.where(see[:, None], x, -math.inf)
                w = torch.softmax(x, -1)
                w = torch.where(some[:, None, None], w, 0.0)
                a = torch.where(see[:, None], qs.abs() @ k.abs().T * abs(scale), 0.0).amax(-1, keepdim=True)
                o, wv = w @ v, w @ v.abs()
                rel = 2 * (2 * a * (d / 8 + 6) * 2 * u + 16 * u) + (pos.size / 4 + 32) * 2 * u
                big = torch.where(see[..., None], v.abs(), 0.0).sum(1)[:, None] if tiny else 0.0
                out[rows, heads] = o
                tol[rows, heads] = (1 + half) * wv * (half + rel) + half * o.abs() + tiny + 2.0 ** -31 * big * (tiny > 0) \
                    + 1e-30
    return out, tol


def fork_ref(src, keep, lens, table, stack, top, page_size):
    """(table, lens, top, stack, copies) after a fork; the inputs are left alone."""
    stack = stack.copy()
    n, width = table.shape
    new_lens = np.array([max(0, min(int(keep[i]), int(lens[j]))) if 0 <= j < n else 0 for i, j in enumerate(src)],
                        np.int32)
    rows = [list(table[j][: ceil_div(int(m), page_size)]) for j, m in zip(src, new_lens)]
    users = {}
    for i, row in enumerate(rows):
        for b, p in enumerate(row):
            users.setdefault(int(p), []).append((i, (b + 1) * page_size > new_lens[i]))
    before = {int(p) for i in range(n) for p in table[i][: ceil_div(int(lens[i]), page_size)]}
    for p in sorted(before - set(users)):
        stack[top] = p
        top += 1
    copies = np.array([[-1] * n, [-1] * n, [0] * n], np.int32)
    for i, row in enumerate(rows):
        part = int(new_lens[i]) % page_size
        if not part:
            continue
        mine = users[int(row[-1])]
        if all(p for _, p in mine) and mine[0][0] == i:
            continue
        if top == 0:
            row.pop()
            new_lens[i] -= part
            continue
        top -= 1
        copies[:, i] = row[-1], stack[top], part
        row[-1] = stack[top]
    out = np.full((n, width), -1, np.int32)
    for i, row in enumerate(rows):
        out[i, : len(row)] = row
    return out, new_lens, top, stack, copies


def logprobs_ref(x, tokens, k):
    """(logprob, entropy, ids, top) of f64 rows x (torch)."""
    # the largest left out of the sums: log(1 + 1e-20) is 0 in 64 bits too
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    n1 = (d == 0).sum(1, keepdim=True)
    lse = n1.double().log() + (torch.where(d == 0, 0.0, e).sum(1, keepdim=True) / n1).log1p()
    y = d - lse
    entropy = (lse - torch.where(e == 0, 0.0, e * d).sum(1, keepdim=True) / e.sum(1, keepdim=True))[:, 0]
    t = tokens.long()
    logprob = torch.where(t < 0, 0.0, y.gather(1, t.clamp(min=0)[:, None])[:, 0])
    order = torch.where(x.isnan(), -math.inf, x)
    # NaN last: after -inf, by id
    key = order.argsort(dim=1, descending=True, stable=True)
    if x.isnan().any():
        nan = x.gather(1, key).isnan().to(torch.int8)
        key = key.gather(1, nan.argsort(dim=1, stable=True))
    ids = key[:, :k]
    return logprob, entropy, ids.int(), y.gather(1, ids)
