"""Cases of the operators that score and branch sequences of a paged
key-value cache: paged_prefill, paged_fork, paged_copy and token_logprobs
(b200_decode.py), each beside its plain form in elementary torch operations
and its definition in 64 bits.

A case is one call as a serving loop makes it.  Pages are handed out in
shuffled order and every slot that no cached token owns holds NaN (a recycled
page is never cleared).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# (query heads, KV heads, head dim) of the shapes this repository runs.
HEADS = [(12, 2, 128), (64, 8, 128), (24, 2, 64), (8, 2, 64), (16, 4, 256), (32, 8, 128), (4, 4, 256), (8, 8, 64)]
VOCABS = [128256, 151936]


def listed():
    return [
        # Draft tokens of 8 sequences checked in one step: latency counts.
        dict(name="prefill_8x5_drafts", op="prefill", n_seq=8, chunk=5, same=True, n_head=12, n_head_kv=2,
             head_dim=128, page_size=16, dtype="f16", max_past=4160, mask=False, window=0),
        # A prompt that starts a sequence.
        dict(name="prefill_1x512_new", op="prefill", n_seq=1, chunk=512, same=True, n_head=64, n_head_kv=8,
             head_dim=128, page_size=16, dtype="bf16", max_past=0, mask=False, window=0),
        # A step that mixes decodes with chunks of prompts; small heads, an odd page size, a mask and a window.
        dict(name="prefill_33_ragged", op="prefill", n_seq=33, chunk=300, same=False, n_head=24, n_head_kv=2,
             head_dim=64, page_size=24, dtype="bf16", max_past=3000, mask=True, window=2048),
        # Four chunks with the largest heads.
        dict(name="prefill_4x1000_d256", op="prefill", n_seq=4, chunk=1000, same=True, n_head=16, n_head_kv=4,
             head_dim=256, page_size=16, dtype="f16", max_past=2000, mask=False, window=0),
        # A whole long prompt at once.
        dict(name="prefill_1x8192_new", op="prefill", n_seq=1, chunk=8192, same=True, n_head=64, n_head_kv=8,
             head_dim=128, page_size=64, dtype="f16", max_past=0, mask=False, window=0),
        # The last chunk of a very long document: the largest work.
        dict(name="prefill_2k_at_128k", op="prefill", n_seq=1, chunk=2048, same=True, n_head=64, n_head_kv=8,
             head_dim=128, page_size=16, dtype="bf16", max_past=129024, mask=False, window=0),
        # Beam search: 16 requests of 4 beams change places after a step.
        dict(name="fork_beams_64", op="fork", n_seq=64, beams=4, page_size=16, max_len=4096, change=0.6),
        # A busy server's step: forks of shared prompts, rejected draft tokens taken back, finished requests.
        dict(name="fork_mixed_1024", op="fork", n_seq=1024, beams=1, page_size=16, max_len=8192, change=0.3),
        # The last pages of the beams that were forked, one layer.
        dict(name="copy_tails_48", op="copy", n_pairs=48, n_head_kv=8, head_dim=128, page_size=16, dtype="f16",
             bounds=True, part=True),
        # Pages of whole sequences moved to other places.
        dict(name="copy_4096_pages", op="copy", n_pairs=4096, n_head_kv=8, head_dim=128, page_size=16, dtype="bf16",
             bounds=False, part=False),
        # One sampled token with its alternatives.
        dict(name="logprobs_1x128256", op="logprobs", n_rows=1, n_vocab=128256, dtype="f32", k=20, banned=0.0),
        # A prompt's scores.
        dict(name="logprobs_1024x151936", op="logprobs", n_rows=1024, n_vocab=151936, dtype="f32", k=5, banned=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "prefill", "fork", "copy", "logprobs"])
    page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 128, 300])
    if op == "fork":
        beams = rng.choice([1, 1, 2, 3, 4, 5, 8])
        n_seq = beams * _log_int(rng, 1, 1024 // beams)
        return dict(op=op, n_seq=n_seq, beams=beams, page_size=page, max_len=_log_int(rng, 4, min(8192, 1024 * page)),
                    change=rng.choice([0.1, 0.3, 0.6, 1.0]))
    if op == "logprobs":
        rows = _log_int(rng, 1, 512)
        vocab = rng.choice(VOCABS + [_log_int(rng, 100, 200000), _log_int(rng, 100, 200000)])
        return dict(op=op, n_rows=rows, n_vocab=vocab, dtype=rng.choice(["f32", "f32", "f16", "bf16"]),
                    k=rng.choice([0, 1, 5, 7, 20, 32]), banned=rng.choice([0.0, 0.1, 0.9]))
    n_head, n_head_kv, head_dim = rng.choice(HEADS)
    dtype = rng.choice(["f16", "bf16"])
    if op == "copy":
        return dict(op=op, n_pairs=_log_int(rng, 1, max(2, (1 << 16) // page)), n_head_kv=n_head_kv,
                    head_dim=head_dim, page_size=page, dtype=dtype, bounds=rng.random() < 0.5,
                    part=rng.random() < 0.5)
    chunk = _log_int(rng, 1, 4096)
    n_seq = _log_int(rng, 1, max(1, min(64, 8192 // chunk)))
    # no more pairs of rows and positions than the largest listed case has
    most = max(1, min(65536, (1 << 28) * 64 // (n_seq * chunk * n_head) - chunk))
    past = 0 if rng.random() < 0.2 else _log_int(rng, 1, most)
    return dict(op=op, n_seq=n_seq, chunk=chunk, same=rng.random() < 0.4, n_head=n_head, n_head_kv=n_head_kv,
                head_dim=head_dim, page_size=page, dtype=dtype, max_past=past, mask=rng.random() < 0.3,
                window=rng.choice([0, 0, 0, _log_int(rng, 1, past + chunk)]))


def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """(cached tokens before, new tokens) per sequence: part of the case, the
    same for every seed."""
    r = random.Random("%s lens" % sorted((k, v) for k, v in case.items() if k != "name"))
    if case["same"]:
        new = [case["chunk"]] * case["n_seq"]
    else:  # decodes, chunks, idle sequences
        new = [r.choice([0, 1, 1, r.randint(1, case["chunk"])]) for _ in range(case["n_seq"])]
        new[r.randrange(len(new))] = case["chunk"]
    past = [r.randint(case["max_past"] // 4, case["max_past"]) for _ in new]
    past[r.randrange(len(past))] = case["max_past"]
    return past, new


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _tables(blocks, width, gen):
    """Shuffled pages for sequences of these block counts; -1 where a row ends."""
    total = sum(blocks)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(blocks), width), -1, dtype=torch.int32)
    live = torch.arange(width)[None, :] < torch.tensor(blocks)[:, None]
    table = table.cuda()
    table[live.cuda()] = order
    return table


def _prepare_prefill(case, s, gen):
    dev = dict(device="cuda")
    ps, n_seq, H, D = case["page_size"], case["n_seq"], case["n_head_kv"], case["head_dim"]
    past, new = _lens(case)
    lens = [a + b for a, b in zip(past, new)]
    blocks = [_ceil(n, ps) for n in lens]
    s["max_blocks"] = max(1, max(blocks))
    n_pages = sum(blocks) + 3
    s["table"] = _tables(blocks, s["max_blocks"], gen)
    owned = torch.zeros((n_pages, ps), dtype=torch.bool, **dev)
    pos = torch.arange(s["max_blocks"] * ps, **dev).view(s["max_blocks"], ps)
    live = pos[None] < torch.tensor(lens, **dev)[:, None, None]
    row = s["table"].long().clamp(min=0)
    owned[row[live.any(2)]] = live[live.any(2)]
    s["k"], s["v"] = (torch.empty((n_pages, ps, H, D), dtype=DTYPES[case["dtype"]], **dev) for _ in range(2))
    for x in (s["k"], s["v"]):
        x.normal_(generator=gen)
        x.masked_fill_(~owned[:, :, None, None], float("nan"))
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, **dev)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, **dev)
    s["max_new"] = max(new)
    rows = cu[-1] + 3  # a few rows of padding
    s["q"] = (torch.randn((rows, case["n_head"], D), generator=gen, **dev) * 1.5).to(DTYPES[case["dtype"]])
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = D ** -0.5
    s["mask_rows"] = None
    if case["mask"]:
        width = s["max_blocks"] * ps
        m = torch.randn((n_seq, width), generator=gen, **dev)
        off = torch.rand((n_seq, width), generator=gen, **dev)
        m = m.masked_fill(off < 0.3, float("-inf")).masked_fill(off > 0.95, -65504.0)
        longest = max(range(n_seq), key=lens.__getitem__)
        if n_seq > 1:
            m[(longest + 1) % n_seq] = float("-inf")  # a sequence with nothing to attend to
        m[longest, 0] = 0.0
        s["mask_rows"] = m.to(torch.float16)


def _prepare_fork(case, s, gen):
    dev = dict(device="cuda")
    ps, n, beams = case["page_size"], case["n_seq"], case["beams"]
    r = random.Random("%s fork" % sorted((k, v) for k, v in case.items() if k != "name"))
    width = _ceil(case["max_len"], ps) + 1
    lens, blocks, share = [], [], []  # share: blocks that a row has in common with the first of its beams
    for i in range(n):
        if i % beams == 0:
            lens.append(r.randint(case["max_len"] // 3, case["max_len"]))
        else:
            lens.append(lens[i - i % beams])
        full = lens[i] // ps
        share.append(0 if i % beams == 0 else r.randint(full // 2, full))
        blocks.append(_ceil(lens[i], ps))
    total = sum(b - c for b, c in zip(blocks, share))
    s["n_pages"] = total + n + 64
    table = _tables(blocks, width, gen)
    # pages that rows do not share: a fresh numbering of the whole pool
    order = torch.randperm(s["n_pages"], generator=gen, **dev).to(torch.int32)
    b, c = torch.tensor(blocks, **dev)[:, None], torch.tensor(share, **dev)[:, None]
    col = torch.arange(width, **dev)[None, :]
    mine = (col < b) & (col >= c)
    table[mine] = order[:total]
    first = torch.arange(n, **dev) // beams * beams
    s["table"] = torch.where(col < c, table[first], table)
    s["free_pages"] = torch.full((s["n_pages"],), -1, dtype=torch.int32, **dev)
    s["free_pages"][: n + 64] = order[total:]
    s["n_free"] = torch.tensor([n + 64], dtype=torch.int32, **dev)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, **dev)
    src, keep = [], []
    for i in range(n):
        p, at = r.random(), i - i % beams
        if p >= case["change"]:
            src.append(i)
            keep.append(lens[i])
        elif beams > 1:  # another beam of the same request survives in this place
            src.append(at + r.randrange(beams))
            keep.append(lens[at])
        elif p < case["change"] / 3:  # the request is over
            src.append(-1)
            keep.append(0)
        elif p < case["change"] * 2 / 3:  # draft tokens are taken back
            src.append(i)
            keep.append(max(0, lens[i] - r.randint(1, 8)))
        else:  # a new request with a prompt that another one has
            j = r.randrange(n)
            src.append(j)
            keep.append(r.randint(0, lens[j]))
    s["src"] = torch.tensor(src, dtype=torch.int32, **dev)
    # (rows that survive: a seed's own numbers of tokens taken back)
    less = torch.randint(0, 2, (n,), generator=gen, **dev).to(torch.int32)
    s["keep"] = (torch.tensor(keep, dtype=torch.int32, **dev) - less).clamp(min=0)
    s["table_out"] = torch.empty_like(s["table"])
    s["seq_lens_out"] = torch.empty_like(s["seq_lens"])
    s["n_free_out"] = torch.empty_like(s["n_free"])


def _prepare_copy(case, s, gen):
    dev = dict(device="cuda")
    ps, n, H, D = case["page_size"], case["n_pairs"], case["n_head_kv"], case["head_dim"]
    n_pages = 2 * n + 1
    s["k"], s["v"] = (torch.empty((n_pages, ps, H, D), dtype=DTYPES[case["dtype"]], **dev) for _ in range(2))
    s["k"].normal_(generator=gen)
    s["v"].normal_(generator=gen)
    s["lo"] = s["hi"] = None
    if case["bounds"]:
        s["lo"], s["hi"] = s["k"].amin(1), s["k"].amax(1)
    order = torch.randperm(n_pages, generator=gen, **dev).to(torch.int32)
    rows = torch.randint(0, ps, (n,), generator=gen, **dev).to(torch.int32)
    # a fork's list: a place per sequence, -1 where nothing is copied
    on = torch.ones(n + 2, dtype=torch.bool, **dev)
    on[0] = on[n // 2 + 1] = False
    s["src"], s["dst"] = (torch.full((n + 2,), -1, dtype=torch.int32, **dev) for _ in range(2))
    s["src"][on], s["dst"][on] = order[:n], order[n:2 * n]
    s["rows"] = None
    if case["part"]:
        s["rows"] = torch.zeros(n + 2, dtype=torch.int32, **dev)
        s["rows"][on] = rows


def _prepare_logprobs(case, s, gen):
    dev = dict(device="cuda")
    rows, vocab = case["n_rows"], case["n_vocab"]
    # logits of a language model: a wide middle and a few likely tokens
    x = torch.randn((rows, vocab), generator=gen, **dev) * 2.5
    likely = torch.randint(0, vocab, (rows, 8), generator=gen, **dev)
    x.scatter_add_(1, likely, torch.rand((rows, 8), generator=gen, **dev) * 12)
    t = torch.randint(0, vocab, (rows,), generator=gen, **dev)
    s["tokens"] = torch.where(torch.rand(rows, generator=gen, **dev) < 0.7, likely[:, 0], t).to(torch.int32)
    if case["banned"]:  # tokens that a grammar rules out
        for at in range(0, rows, 64):
            off = torch.rand((min(64, rows - at), vocab), generator=gen, **dev) < case["banned"]
            off.scatter_(1, s["tokens"][at:at + 64, None].long(), False)
            x[at:at + 64].masked_fill_(off, float("-inf"))
    s["logits"] = x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case)
    {"prefill": _prepare_prefill, "fork": _prepare_fork, "copy": _prepare_copy,
     "logprobs": _prepare_logprobs}[case["op"]](case, s, gen)
    return s


# ---------------------------------------------------------------- own calls

def _package():
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(here, "llama-cpp-ascend310b4-addon_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b200_decode

    return b200_decode


def _run_own(s):
    B = _package()
    if s["op"] == "fork":
        if "workspace" not in s:
            size = B.paged_fork_workspace_size(s["n_seq"], s["table"].shape[1], s["n_pages"])
            s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        f = B.paged_fork(s["src"], s["keep"], s["seq_lens"], s["table"], s["free_pages"], s["n_free"], s["page_size"],
                         table_out=s["table_out"], seq_lens_out=s["seq_lens_out"], n_free_out=s["n_free_out"],
                         workspace=s["workspace"])
        return dict(table=f.block_table, seq_lens=f.seq_lens, n_free=f.n_free, free_pages=s["free_pages"],
                    copy_src=f.copy_src, copy_dst=f.copy_dst, copy_rows=f.copy_rows)
    if s["op"] == "logprobs":
        r = B.token_logprobs(s["logits"], s["tokens"], s["k"])
        out = dict(logprob=r.logprob, entropy=r.entropy)
        if s["k"]:
            out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
        return out
    if "cache" not in s:  # the handle a program keeps for its cache
        s["cache"] = B.PagedKV(s["k"], s["v"], k_lo=s.get("lo"), k_hi=s.get("hi"))
    if s["op"] == "copy":
        B.paged_copy(s["cache"], s["src"], s["dst"], rows=s["rows"])
        return _copied(s)
    if "workspace" not in s:
        size = B.paged_prefill_workspace_size(s["head_dim"], s["q"].shape[0], s["n_seq"], s["n_head"], s["n_head_kv"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return B.paged_prefill(s["cache"], s["q"], s["table"], s["seq_lens"], s["cu"], s["scale"], mask=s["mask_rows"],
                           window=s["window"], out=s["out"], workspace=s["workspace"])


def _copied(s):
    out = dict(k=s["k"], v=s["v"])
    if s["lo"] is not None:
        out.update(lo=s["lo"], hi=s["hi"])
    return out


# -------------------------------------------------------------- plain forms

def _plain_prefill(s):
    n_seq, H, D, ps = s["n_seq"], s["n_head_kv"], s["head_dim"], s["page_size"]
    dev = s["q"].device
    G = s["n_head"] // H
    cu, lens = s["cu"].long(), s["seq_lens"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["max_new"], device=dev)
    row = cu[:-1, None] + i  # [n_seq, max_new]
    real = i < new[:, None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)]
    page = s["table"].long().clamp(min=0)
    p = torch.arange(s["max_blocks"] * ps, device=dev)
    owned = p < lens[:, None]
    at = (lens - new)[:, None] + i  # the rows' positions
    live = owned[:, None, :] & (p <= at[..., None])
    if s["window"]:
        live &= p > (at - s["window"])[..., None]
    bias = None
    if s["mask_rows"] is not None:
        bias = s["mask_rows"][:, None, : p.numel()].float()
        owned = owned & (bias[:, 0] != float("-inf"))
        live &= bias != float("-inf")
        # relative to the row's largest entry: a row of lowest values keeps the scores' own bits
        bias = bias - torch.where(live, bias, float("-inf")).amax(-1, keepdim=True).clamp(min=-65504.0)
    out = torch.zeros((s["q"].shape[0], H, G, D), dtype=s["q"].dtype, device=dev)
    for h in range(H):  # one KV head at a time: the scores of all would not fit
        k, v = (torch.where(owned[..., None], s[x][page, :, h].flatten(1, 2).float(), 0.0) for x in "kv")
        w = q[:, :, h * G:(h + 1) * G].float().flatten(1, 2) @ k.transpose(1, 2)  # [n_seq, max_new * G, tokens]
        w = w.unflatten(1, (-1, G)).mul_(s["scale"])
        if bias is not None:
            w += torch.where(live, bias, 0.0)[:, :, None]
        w.masked_fill_(~live[:, :, None], float("-inf"))
        w -= w.amax(-1, keepdim=True).clamp(min=-3e38)
        w.exp_()
        total = w.sum(-1, keepdim=True)
        o = (w.flatten(1, 2) @ v).unflatten(1, (-1, G)) / torch.where(total > 0, total, 1.0)
        out[row[real], h] = o[real].to(out.dtype)
    return out.flatten(1, 2)


def _plain_fork(s):
    ps, n, n_pages = s["page_size"], s["n_seq"], s["n_pages"]
    dev = s["table"].device
    width = s["table"].shape[1]
    lens, src = s["seq_lens"].long(), s["src"].long()
    k = torch.where(src >= 0, torch.minimum(s["keep"].long(), lens[src.clamp(min=0)]), 0).clamp(min=0)
    col = torch.arange(width, device=dev)[None, :]
    old_b, new_b = (lens + ps - 1) // ps, (k + ps - 1) // ps
    old_live, new_live = col < old_b[:, None], col < new_b[:, None]
    old = torch.where(old_live, s["table"].long(), n_pages)
    new = torch.where(new_live, s["table"].long()[src.clamp(min=0)], n_pages)
    one = torch.ones_like(new)
    held = torch.zeros(n_pages + 1, dtype=torch.int64, device=dev)
    held.scatter_add_(0, new.reshape(-1), one.reshape(-1))
    # pages that nobody holds any more, in ascending order
    was = torch.zeros_like(held).scatter_add_(0, old.reshape(-1), one.reshape(-1))
    freed = ((was > 0) & (held == 0))[:n_pages]
    n0 = s["n_free"].long()
    at = torch.where(freed, n0 + freed.cumsum(0) - 1, n_pages)
    stack = torch.cat([s["free_pages"], s["free_pages"].new_zeros(1)])
    stack.scatter_(0, at, torch.arange(n_pages, device=dev).int())
    pool = n0 + freed.sum()
    # rows whose last page is not full need it alone
    tail = k % ps
    page = torch.where(tail > 0, new.gather(1, (new_b - 1).clamp(min=0)[:, None])[:, 0], n_pages)
    tails = torch.zeros(n_pages + 1, dtype=torch.int64, device=dev).scatter_add_(0, page, torch.ones_like(page))
    low = torch.full((n_pages + 1,), n, dtype=torch.int64, device=dev)
    row = torch.arange(n, device=dev)
    low.scatter_reduce_(0, page, row, "amin")
    need = (tail > 0) & ~((held[page] == tails[page]) & (low[page] == row))
    rank = need.cumsum(0) - 1
    got = need & (rank < pool)
    fresh = stack[(pool - 1 - rank).clamp(0, n_pages)].long()
    lost = need & ~got  # no page left: the row ends with its last full block
    k = torch.where(lost, k - tail, k)
    last = col == (new_b - 1)[:, None]
    new = torch.where(last & got[:, None], fresh[:, None], new)
    new = torch.where(new_live & ~(last & lost[:, None]), new, -1)
    return dict(table=new.int(), seq_lens=k.int(), n_free=(pool - got.sum()).int(), free_pages=stack[:n_pages],
                copy_src=torch.where(got, page, -1).int(), copy_dst=torch.where(got, fresh, -1).int(),
                copy_rows=torch.where(got, tail, 0).int())


def _plain_copy(s):
    ps, last = s["page_size"], s["k"].shape[0] - 1
    src, dst = s["src"].long(), s["dst"].long()
    on = src >= 0
    # (an entry of nothing writes what another place already holds)
    src, dst = torch.where(on, src, last), torch.where(on, dst, last)
    rows = torch.full_like(src, ps) if s["rows"] is None else s["rows"].long()
    takes = (torch.arange(ps, device=src.device) < rows[:, None]) & on[:, None]
    for x in ("k", "v"):
        s[x][dst] = torch.where(takes[..., None, None], s[x][src], s[x][dst])
    if s["lo"] is not None:
        some = (takes.any(1))[:, None, None]
        for x in ("lo", "hi"):
            s[x][dst] = torch.where(some, s[x][src], s[x][dst])
    return _copied(s)


def _plain_logprobs(s):
    x = s["logits"].float()
    t = s["tokens"].long()[:, None]
    top = x.amax(1, keepdim=True)
    d = x - top
    w = torch.exp(d)
    z = w.double().sum(1, keepdim=True)
    w *= torch.where(d == float("-inf"), 0.0, d)
    mean = w.double().sum(1, keepdim=True) / z
    lse = torch.log(z)
    out = dict(logprob=(d.gather(1, t).double() - lse)[:, 0].float(), entropy=(lse - mean)[:, 0].float())
    if s["k"]:
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        out.update(top_ids=i[:, : s["k"]].int(), top_logprobs=((v[:, : s["k"]] - top).double() - lse).float())
    return out


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "prefill":
        return _plain_prefill(state)
    if state["op"] == "fork":
        return _plain_fork(state)
    if state["op"] == "copy":
        return _plain_copy(state)
    return _plain_logprobs(state)


# -------------------------------------------------------------------- work

def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "f32" else 2
        cells = case["n_rows"] * case["n_vocab"]
        return dict(bytes=cells * size + case["n_rows"] * (12 + 8 * case["k"]), flops=6 * cells)
    if case["op"] == "fork":
        # a third of the rows' pages change hands; every entry is read and written once
        entries = case["n_seq"] * (_ceil(case["max_len"], case["page_size"]) + 1)
        return dict(bytes=4 * 2 * entries + 28 * case["n_seq"], flops=10 * entries)
    if case["op"] == "copy":
        row = case["n_head_kv"] * case["head_dim"] * 2
        rows = case["n_pairs"] * (case["page_size"] - 1) // 2 if case["part"] else case["n_pairs"] * case["page_size"]
        rows += case["n_pairs"] if case["bounds"] else 0
        return dict(bytes=rows * row * 4 + 12 * case["n_pairs"], flops=0)
    past, new = _lens(case)
    w = case["window"] or 1 << 40
    pairs, seen = 0, 0
    for a, n in zip(past, new):
        full = max(0, min(n, w - a))  # rows that see everything before them
        pairs += full * a + full * (full + 1) // 2 + (n - full) * w
        seen += a + n - max(0, a + 1 - w) if n else 0
    H, D = case["n_head"], case["head_dim"]
    return dict(bytes=seen * (case["n_head_kv"] * D * 4 + (2 if case["mask"] else 0)) + sum(new) * H * D * 4
                + sum(_ceil(a + n, case["page_size"]) for a, n in zip(past, new)) * 4, flops=4 * pairs * H * D)


# ------------------------------------------------------------------- exact

def _exact_prefill(s):
    past, new = _lens({k: s[k] for k in ("op", "n_seq", "chunk", "same", "n_head", "n_head_kv", "head_dim",
                                         "page_size", "dtype", "max_past", "mask", "window")})
    H, D, ps = s["n_head_kv"], s["head_dim"], s["page_size"]
    G = s["n_head"] // H
    if work(s)["flops"] > 12e12:
        return None
    dev = s["q"].device
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    start = 0
    for i, (a, n) in enumerate(zip(past, new)):
        for lo in range(0, n, 512):
            hi = min(n, lo + 512)
            pos = torch.arange(a + hi, device=dev)
            if s["mask_rows"] is not None:
                pos = pos[s["mask_rows"][i, pos] != float("-inf")]
            page = s["table"][i, pos // ps].long()
            at = torch.arange(a + lo, a + hi, device=dev)
            seen = pos[None, :] <= at[:, None]
            if s["window"]:
                seen &= at[:, None] - pos[None, :] < s["window"]
            for h in range(H):
                q = s["q"][start + lo:start + hi, h * G:(h + 1) * G].double()
                x = (q @ s["k"][page, pos % ps, h].double().T) * s["scale"]  # [rows, G, tokens]
                if s["mask_rows"] is not None:
                    x += s["mask_rows"][i, pos].double()
                x = torch.where(seen[:, None, :], x, -float("inf"))
                any_ = seen.any(1)
                x = torch.softmax(x[any_], -1) @ s["v"][page, pos % ps, h].double()
                rows = torch.arange(start + lo, start + hi, device=dev)[any_]
                out[rows, h * G:(h + 1) * G] = x
        start += n
    return out


def _exact_fork(s):
    ps = s["page_size"]
    old, lens = s["table"].tolist(), s["seq_lens"].tolist()
    src, keep, stack, top = s["src"].tolist(), s["keep"].tolist(), s["free_pages"].tolist(), int(s["n_free"][0])
    width = s["table"].shape[1]
    got = [max(0, min(keep[i], lens[j])) if j >= 0 else 0 for i, j in enumerate(src)]
    new = [old[max(j, 0)][: _ceil(g, ps)] for j, g in zip(src, got)]
    holders = {}
    for i, row in enumerate(new):
        for b, p in enumerate(row):
            holders.setdefault(p, []).append((i, (b + 1) * ps > got[i]))
    for p in sorted({p for row, n in zip(old, lens) for p in row[: _ceil(n, ps)] if p not in holders}):
        stack[top] = p
        top += 1
    copies = []
    for i, row in enumerate(new):
        copies.append((-1, -1, 0))
        if got[i] % ps == 0:
            continue
        mine = holders[row[-1]]
        if all(part for _, part in mine) and mine[0][0] == i:
            continue
        if top == 0:
            row.pop()
            got[i] -= got[i] % ps
            continue
        top -= 1
        copies[-1] = (row[-1], stack[top], got[i] % ps)
        row[-1] = stack[top]
    dev = s["table"].device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(table=i32([row + [-1] * (width - len(row)) for row in new]), seq_lens=i32(got), n_free=i32([top]),
                free_pages=i32(stack), copy_src=i32([c[0] for c in copies]), copy_dst=i32([c[1] for c in copies]),
                copy_rows=i32([c[2] for c in copies]))


def _exact_logprobs(s):
    n = s["n_rows"]
    dev = s["logits"].device
    out = dict(logprob=torch.empty(n, dtype=torch.float64, device=dev),
               entropy=torch.empty(n, dtype=torch.float64, device=dev))
    if s["k"]:
        out.update(top_ids=torch.empty((n, s["k"]), dtype=torch.int32, device=dev),
                   top_logprobs=torch.empty((n, s["k"]), dtype=torch.float64, device=dev))
    for at in range(0, n, 64):
        x = s["logits"][at:at + 64].double()
        y = torch.log_softmax(x, 1)
        rows = slice(at, at + x.shape[0])
        out["logprob"][rows] = y[torch.arange(x.shape[0], device=dev), s["tokens"][rows].long()]
        out["entropy"][rows] = -torch.nan_to_num(y.exp() * y, nan=0.0).sum(1)
        if s["k"]:
            i = (-x).argsort(dim=1, stable=True)[:, : s["k"]]
            out["top_ids"][rows] = i.int()
            out["top_logprobs"][rows] = y.gather(1, i)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefill":
        return _exact_prefill(s)
    if case["op"] == "fork":
        return _exact_fork(s)
    if case["op"] == "copy":
        return None  # nothing is computed
    return _exact_logprobs(s)
