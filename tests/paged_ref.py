"""Plain implementations of the paged key-value cache operators in 64 bits,
and seeded caches to run them on.

Everything is numpy on the host.  A cache is a dict: k, v float64 arrays
[n_pages, page_size, n_head_kv, head_dim] holding values of the cache type,
NaN wherever no cached token lives."""
import numpy as np
import torch

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def ceil_div(a, b):
    return -(-a // b)


def rounded(x, dtype):
    """x (f32) to the cache type and back, in float64."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(DTYPES[dtype]).double().numpy()


def plan_ref(new_lens, seq_lens, table, free_pages, n_free, page_size, max_tokens):
    """(slots, positions, cu, seq_lens, n_free, table, free_pages) after the
    step; the inputs are left alone."""
    table, stack, lens = table.copy(), free_pages.copy(), seq_lens.copy()
    max_blocks = table.shape[1]
    top = int(n_free)
    start = [0]
    for i, n in enumerate(seq_lens):
        if new_lens[i] < 0:
            for b in range(ceil_div(int(n), page_size)):
                stack[top] = table[i, b]
                top += 1
            lens[i] = 0
        start.append(start[-1] + max(int(new_lens[i]), 0))
    pool, asked = top, 0
    slots = np.full(max_tokens, -1, np.int64)
    positions = np.full(max_tokens, -1, np.int32)
    for i, n in enumerate(int(v) for v in seq_lens):
        new = int(new_lens[i])
        old_b, end_b = ceil_div(n, page_size), ceil_div(n + new, page_size)
        if new < 0 or start[i + 1] > max_tokens or end_b > max_blocks:
            continue
        asked += end_b - old_b
        if end_b > old_b and asked > pool:
            continue
        for b in range(old_b, end_b):
            top -= 1
            table[i, b] = stack[top]
        for j in range(new):
            slots[start[i] + j] = int(table[i, (n + j) // page_size]) * page_size + (n + j) % page_size
            positions[start[i] + j] = n + j
        lens[i] = n + new
    cu = np.minimum(np.array(start, np.int64), max_tokens).astype(np.int32)
    return slots, positions, cu, lens, top, table, stack


def make_cache(r, lens, page_size, n_head_kv, head_dim, dtype, extra_pages=2, k_scale=1.0):
    """A cache holding lens[s] tokens of N(0, k_scale^2) keys and N(0, 1)
    values per sequence in shuffled pages: dict(k, v, table, lens)."""
    blocks = [ceil_div(n, page_size) for n in lens]
    n_pages = sum(blocks) + extra_pages
    order = r.permutation(n_pages)
    shape = (n_pages, page_size, n_head_kv, head_dim)
    k, v = np.full(shape, np.nan), np.full(shape, np.nan)
    table = np.full((len(lens), max(1, max(blocks))), -1, np.int32)
    at = 0
    for s, n in enumerate(lens):
        table[s, :blocks[s]] = order[at:at + blocks[s]]
        at += blocks[s]
        for b in range(blocks[s]):
            rows = min(page_size, n - b * page_size)
            p = table[s, b]
            k[p, :rows] = rounded(r.standard_normal((rows,) + shape[2:]) * k_scale, dtype)
            v[p, :rows] = rounded(r.standard_normal((rows,) + shape[2:]), dtype)
    return dict(k=k, v=v, table=table, lens=np.array(lens, np.int32))


def bounds_of(c):
    """Per-page smallest and largest key per channel (rows that hold tokens);
    NaN for an empty page."""
    import warnings

    with warnings.catch_warnings():
        warnings.simplefilter("ignore", RuntimeWarning)  # pages of NaN only
        return np.nanmin(c["k"], axis=1), np.nanmax(c["k"], axis=1)


def select_ref(q, lo, hi, table, lens, page_size, n_sel):
    """int32 [n_seq, n_head_kv, n_sel]."""
    n_seq, n_head, _ = q.shape
    n_head_kv = lo.shape[1]
    group = n_head // n_head_kv
    out = np.full((n_seq, n_head_kv, n_sel), -1, np.int32)
    for s in range(n_seq):
        nb = ceil_div(int(lens[s]), page_size)
        if nb == 0:
            continue
        for h in range(n_head_kv):
            qs = q[s, h * group:(h + 1) * group].astype(np.float64)
            score = []
            for b in range(nb - 1):
                p = table[s, b]
                score.append(np.maximum(qs * lo[p, h], qs * hi[p, h]).sum(-1).max())
            older = sorted(range(nb - 1), key=lambda b: (-score[b], b))[:n_sel - 1]
            chosen = sorted(older + [nb - 1])
            out[s, h, :len(chosen)] = chosen
    return out


def attn_ref(c, q, page_size, scale, mask=None, sel=None):
    """(out, bound): the result in float64 and, per element, how far an f32
    computation of it may be off.

    With u = 2^-24: a score of D products, entering with 22 bits and added in
    f32 (D / 8 + 4 roundings or truncations of at most 2u each along any path),
    is off by at most A e, A = scale * sum_d |q_d k_d| and e = (D / 8 + 6) 2u;
    the subtraction of the maximum and the product with log2(e) add a few u of
    a score difference, where the weight exp(-x) makes x exp(-x) u < u.  The
    weights then differ by a factor within 1 +- (2 A e + 16 u) relative to one
    another, and adding n weighted values in f32 costs at most (n / 4 + 32) u.
    Numerator and denominator both carry these, relative to sum w |v| / sum w."""
    n_seq, n_head, d = q.shape
    n_head_kv = c["k"].shape[2]
    group = n_head // n_head_kv
    out, tol = np.zeros(q.shape), np.full(q.shape, 1e-30)
    u = 2.0 ** -24
    for s in range(n_seq):
        n = int(c["lens"][s])
        for h in range(n_head_kv):
            if sel is None:
                blocks = list(range(ceil_div(n, page_size)))
            else:
                blocks = [int(b) for b in sel[s, h] if b >= 0]
            pos = np.array([b * page_size + i for b in blocks for i in range(page_size)], np.int64)
            pos = pos[pos < n]
            if mask is not None:
                pos = pos[mask[s, pos] != -np.inf]
            if pos.size == 0:
                continue
            page = c["table"][s, pos // page_size]
            k, v = c["k"][page, pos % page_size, h], c["v"][page, pos % page_size, h]
            qs = q[s, h * group:(h + 1) * group].astype(np.float64)
            x = qs @ k.T * scale
            if mask is not None:
                x = x + mask[s, pos].astype(np.float64)
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            a = (np.abs(qs) @ np.abs(k).T * abs(scale)).max(-1, keepdims=True)
            rows = slice(h * group, (h + 1) * group)
            out[s, rows] = w @ v
            rel = 2 * (2 * a * (d / 8 + 6) * 2 * u + 16 * u) + (pos.size / 4 + 32) * 2 * u
            tol[s, rows] = (w @ np.abs(v)) * rel + 1e-30
    return out, tol


def to_device(c, dtype, layout="token"):
    """(k, v) CUDA tensors of the cache; layout "token": rows [page, row, head,
    dim] as stored, "head": [page, head, row, dim] in memory, "gap": rows with
    unused space between them."""
    out = []
    for name in ("k", "v"):
        t = torch.from_numpy(c[name]).to(DTYPES[dtype]).cuda()
        if layout == "head":
            t = t.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "gap":
            n, p, h, d = t.shape
            big = torch.full((n, p + 1, h + 1, d + 8), float("nan"), dtype=t.dtype, device="cuda")
            big[:, :p, :h, :d] = t
            t = big[:, :p, :h, :d]
        out.append(t)
    return out
