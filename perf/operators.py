"""Cases of the paged key-value cache operators: paged_plan, paged_store,
paged_select and paged_attn (b200_decode.py), each beside its plain form in
elementary torch operations and its definition in 64 bits.

A case is one call as a serving loop makes it: a batch of sequences whose
cached tokens live in fixed-size pages, found through a block table.  Pages
are handed out in shuffled order, every slot that no cached token owns holds
NaN (a recycled page is never cleared), and the lengths of a batch are ragged.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, KV heads, head dim) of the shapes this repository runs.
HEADS = [(12, 2, 128), (64, 8, 128), (24, 2, 64), (8, 2, 64), (16, 4, 256), (32, 8, 128), (4, 4, 256), (8, 8, 64)]
# One workspace serves every call of a stream; a serving loop allocates it once.
WORKSPACE_BYTES = 64 << 20


def listed():
    return [
        # One decode step of a small batch: one token per sequence, a few of them open a page.
        dict(name="plan_decode_64", op="plan", n_seq=64, page_size=16, max_len=4096, chunk=1, release=False),
        # A scheduler step of a busy server: decodes, prompt chunks, idle rows and finished requests.
        dict(name="plan_mixed_1024", op="plan", n_seq=1024, page_size=16, max_len=8192, chunk=512, release=True),
        # The K and V rows of one decode step, with the page bounds that block selection reads.
        dict(name="store_decode_64", op="store", n_seq=64, n_head_kv=8, head_dim=128, page_size=16, dtype="f16",
             max_len=2048, chunk=1),
        # A prompt of 4 sequences going into the cache of one layer.
        dict(name="store_prompt_8k", op="store", n_seq=4, n_head_kv=8, head_dim=128, page_size=64, dtype="bf16",
             max_len=4096, chunk=2048),
        # Which 128 of up to 2048 pages each KV head reads, 16 sequences.
        dict(name="select_16x32k", op="select", n_seq=16, n_head=64, n_head_kv=8, head_dim=128, page_size=16,
             dtype="f16", min_len=16384, max_len=32768, k_blocks=128),
        # One very long sequence: 8192 pages scored for one token.
        dict(name="select_1x128k", op="select", n_seq=1, n_head=12, n_head_kv=2, head_dim=128, page_size=16,
             dtype="bf16", min_len=131000, max_len=131072, k_blocks=256),
        # A chat that has just begun: latency only.
        dict(name="attn_1x37", op="attn", n_seq=1, n_head=12, n_head_kv=2, head_dim=128, page_size=16, dtype="f16",
             min_len=37, max_len=37, mask=False, k_blocks=0),
        # One sequence at the benchmark's context.
        dict(name="attn_1x4160", op="attn", n_seq=1, n_head=64, n_head_kv=8, head_dim=128, page_size=16, dtype="f16",
             min_len=4160, max_len=4160, mask=False, k_blocks=0),
        # An ordinary serving batch, lengths from nothing to 8192.
        dict(name="attn_48_ragged", op="attn", n_seq=48, n_head=64, n_head_kv=8, head_dim=128, page_size=16,
             dtype="f16", min_len=0, max_len=8192, mask=False, k_blocks=0),
        # Small heads, an odd page size, bf16 and a mask (shared prompts with parts switched off).
        dict(name="attn_33_d64_mask", op="attn", n_seq=33, n_head=24, n_head_kv=2, head_dim=64, page_size=24,
             dtype="bf16", min_len=1, max_len=5000, mask=True, k_blocks=0),
        # Long documents: the largest cache.
        dict(name="attn_8x128k", op="attn", n_seq=8, n_head=64, n_head_kv=8, head_dim=128, page_size=64, dtype="f16",
             min_len=32768, max_len=131072, mask=False, k_blocks=0),
        # Attention over the selected pages only.
        dict(name="attn_16x32k_sel128", op="attn", n_seq=16, n_head=64, n_head_kv=8, head_dim=128, page_size=16,
             dtype="f16", min_len=16384, max_len=32768, mask=False, k_blocks=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "select", "attn", "attn"])
    page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 128])
    if op == "plan":
        return dict(op=op, n_seq=_log_int(rng, 1, 2000), page_size=page, max_len=_log_int(rng, 16, 8192),
                    chunk=_log_int(rng, 1, 512), release=rng.random() < 0.5)
    n_head, n_head_kv, head_dim = rng.choice(HEADS)
    dtype = rng.choice(["f16", "bf16"])
    if op == "store":
        chunk = _log_int(rng, 1, 2048)
        n_seq = _log_int(rng, 1, min(1024, 8192 // chunk))
        return dict(op=op, n_seq=n_seq, n_head_kv=n_head_kv, head_dim=head_dim, page_size=page, dtype=dtype,
                    max_len=_log_int(rng, 1, min(2048, (1 << 17) // n_seq)), chunk=chunk)
    n_seq = _log_int(rng, 1, 64)
    if op == "select":  # enough blocks for a choice: at least 16, at most half of them taken
        max_len = _log_int(rng, 16 * page, min(131072, max(16 * page, (1 << 19) // n_seq)))
        if max_len > 16384 * page:
            page = 16
        blocks = (max_len + page - 1) // page
        return dict(op=op, n_seq=n_seq, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page_size=page,
                    dtype=dtype, min_len=rng.choice([0, 1, max_len // 2, max_len]), max_len=max_len,
                    k_blocks=_log_int(rng, 4, min(blocks // 2, 512)))
    max_len = _log_int(rng, 1, min(131072, (1 << 18) // n_seq))
    min_len = rng.choice([0, 1, max_len // 2, max_len])
    blocks = (max_len + page - 1) // page
    k_blocks = _log_int(rng, 1, min(blocks + 2, 512)) if rng.random() < 0.3 else 0
    return dict(op=op, n_seq=n_seq, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page_size=page, dtype=dtype,
                min_len=min_len, max_len=max_len, mask=rng.random() < 0.3, k_blocks=k_blocks)


def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """Cached tokens per sequence: part of the case, the same for every seed."""
    r = random.Random("%s lens" % sorted((k, v) for k, v in case.items() if k != "name"))
    if case["op"] in ("plan", "store"):
        return [r.randint(0, case["max_len"]) for _ in range(case["n_seq"])]
    lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["n_seq"])]
    lens[r.randrange(len(lens))] = case["max_len"]
    return lens


def _new_lens(case):
    """Tokens each sequence appends in this step; -1 gives its pages back."""
    r = random.Random("%s new" % sorted((k, v) for k, v in case.items() if k != "name"))
    if case["op"] == "store":
        return [case["chunk"]] * case["n_seq"]
    out = []
    for _ in range(case["n_seq"]):
        p = r.random()
        if case["chunk"] == 1 or p < 0.8:
            out.append(1)
        elif p < 0.9:
            out.append(r.randint(1, case["chunk"]))
        elif p < 0.95 or not case["release"]:
            out.append(0)
        else:
            out.append(-1)
    return out


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


def _cache(case, lens, table, n_pages, gen):
    """K and V pages [n_pages, page, heads, dim] of normal values; NaN in every
    slot that no cached token owns.  One page more is allocated behind them."""
    shape = (n_pages + 1, case["page_size"], case["n_head_kv"], case["head_dim"])
    owned = torch.zeros(shape[:2], dtype=torch.bool, device="cuda")
    width = table.shape[1]
    pos = torch.arange(width * case["page_size"], device="cuda").view(width, case["page_size"])
    for i, n in enumerate(lens):
        b = _ceil(n, case["page_size"])
        owned[table[i, :b].long()] = pos[:b] < n
    out = []
    for _ in range(2):
        x = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda")
        x.normal_(generator=gen)
        x.masked_fill_(~owned[:, :, None, None], float("nan"))
        out.append(x)
    return out


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case)
    ps, n_seq = case["page_size"], case["n_seq"]
    lens = _lens(case)
    dev = dict(device="cuda")
    if case["op"] == "plan":
        new = _new_lens(case)
        blocks = [_ceil(n, ps) for n in lens]
        s["max_blocks"] = _ceil(case["max_len"] + case["chunk"], ps)
        need = sum(_ceil(n + max(a, 0), ps) - b for n, a, b in zip(lens, new, blocks))
        s["n_pages"] = sum(blocks) + need + 64
        s["table"] = _tables(blocks, s["max_blocks"], gen)
        perm = torch.randperm(need + 64, generator=gen, **dev).to(torch.int32) + sum(blocks)
        s["free_pages"] = torch.full((s["n_pages"],), -1, dtype=torch.int32, **dev)
        s["free_pages"][: need + 64] = perm
        s["n_free"] = torch.tensor([need + 64], dtype=torch.int32, **dev)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, **dev)
        s["new_lens"] = torch.tensor(new, dtype=torch.int32, **dev)
        s["max_tokens"] = sum(max(a, 0) for a in new) + 8  # a few rows of padding
        s["seq_lens_out"] = torch.empty_like(s["seq_lens"])
        s["n_free_out"] = torch.empty_like(s["n_free"])
        return s
    H, D = case["n_head_kv"], case["head_dim"]
    if case["op"] == "store":
        after = [n + case["chunk"] for n in lens]
        blocks = [_ceil(n, ps) for n in after]
        s["n_pages"] = sum(blocks)
        table = _tables(blocks, max(blocks), gen)
        k, v = _cache(case, lens, table, s["n_pages"], gen)
        s["k_all"], s["v_all"] = k, v
        # A page's bounds cover the rows it holds; an unused page's are whatever the last owner left.
        s["lo_all"] = torch.nan_to_num(k.float(), nan=float("inf")).amin(1).clamp(max=60000.0).to(k.dtype)
        s["hi_all"] = torch.nan_to_num(k.float(), nan=-float("inf")).amax(1).clamp(min=-60000.0).to(k.dtype)
        tokens = n_seq * case["chunk"]
        pos = (torch.tensor(lens, **dev)[:, None] + torch.arange(case["chunk"], **dev)[None, :])
        page = table.gather(1, pos // ps).long()
        slots = (page * ps + pos % ps).reshape(-1)
        s["slots"] = torch.cat([slots, torch.full((3,), -1, dtype=torch.int64, **dev)])  # padding rows
        s["new_k"] = torch.randn((tokens + 3, H, D), generator=gen, **dev)
        s["new_v"] = torch.randn((tokens + 3, H, D), generator=gen, **dev)
        return s
    blocks = [_ceil(n, ps) for n in lens]
    s["max_blocks"] = max(1, max(blocks))
    n_pages = sum(blocks) + 3
    s["table"] = _tables(blocks, s["max_blocks"], gen)
    k, v = _cache(case, lens, s["table"], n_pages, gen)
    s["k"], s["v"] = k[:n_pages], v[:n_pages]
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, **dev)
    s["q"] = torch.randn((n_seq, case["n_head"], D), generator=gen, **dev) * 1.5
    s["scale"] = D ** -0.5
    s["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, **dev)
    if case["op"] == "select":
        s["lo"], s["hi"] = torch.zeros_like(k[:n_pages, 0]), torch.zeros_like(k[:n_pages, 0])
        for at in range(0, n_pages, 4096):
            part = k[at:min(n_pages, at + 4096)].float()
            rows = slice(at, at + part.shape[0])
            s["lo"][rows] = torch.nan_to_num(part, nan=60000.0).amin(1).to(k.dtype)
            s["hi"][rows] = torch.nan_to_num(part, nan=-60000.0).amax(1).to(k.dtype)
        return s
    s["mask_rows"] = None
    if case["mask"]:
        width = s["max_blocks"] * ps
        m = torch.randn((n_seq, width), generator=gen, **dev)
        off = torch.rand((n_seq, width), generator=gen, **dev)
        m = m.masked_fill(off < 0.3, float("-inf")).masked_fill(off > 0.95, -65504.0)
        longest = max(range(n_seq), key=lens.__getitem__)
        m[(longest + 1) % n_seq] = float("-inf")  # a row with nothing to attend to
        m[longest, 0] = 0.0
        s["mask_rows"] = m.to(torch.float16)
    s["sel"] = None
    if case["k_blocks"]:
        # Each KV head's own pages: a random choice that always has the newest block, ascending.
        kb = case["k_blocks"]
        rank = torch.rand((n_seq, H, s["max_blocks"]), generator=gen, **dev)
        b = torch.tensor(blocks, **dev)[:, None, None]
        at = torch.arange(s["max_blocks"], **dev)
        rank = torch.where(at < b, rank, 2.0).masked_fill(at == b - 1, -1.0)
        kk = min(kb, s["max_blocks"])
        got = rank.argsort(-1)[..., :kk]
        got = torch.where(got < b, got, s["max_blocks"]).sort(-1).values
        got = torch.where(got < b, got, -1).to(torch.int32)
        s["sel"] = torch.full((n_seq, H, kb), -1, dtype=torch.int32, **dev)
        s["sel"][..., :kk] = got
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
    if s["op"] == "plan":
        p = B.paged_plan(s["new_lens"], s["seq_lens"], s["table"], s["free_pages"], s["n_free"], s["page_size"],
                         s["max_tokens"], seq_lens_out=s["seq_lens_out"], n_free_out=s["n_free_out"])
        return dict(slots=p.slots, positions=p.positions, cu=p.cu, seq_lens=p.seq_lens, n_free=p.n_free,
                    table=s["table"], free_pages=s["free_pages"])
    if "cache" not in s:  # the handle a program keeps for its cache
        if s["op"] == "store":
            n = s["n_pages"]
            s["cache"] = B.PagedKV(s["k_all"][:n], s["v_all"][:n], k_lo=s["lo_all"][:n], k_hi=s["hi_all"][:n])
        else:
            s["cache"] = B.PagedKV(s["k"], s["v"], k_lo=s.get("lo"), k_hi=s.get("hi"))
    if s["op"] == "store":
        B.paged_store(s["cache"], s["new_k"], s["new_v"], s["slots"])
        n = s["n_pages"]
        return dict(k=s["k_all"][:n], v=s["v_all"][:n], lo=s["lo_all"][:n], hi=s["hi_all"][:n])
    if s["op"] == "select":
        return B.paged_select(s["cache"], s["q"], s["table"], s["seq_lens"], s["k_blocks"], workspace=s["workspace"])
    return B.paged_attn(s["cache"], s["q"], s["table"], s["seq_lens"], s["scale"], mask=s["mask_rows"], sel=s["sel"],
                        workspace=s["workspace"])


# -------------------------------------------------------------- plain forms

def _plain_plan(s):
    ps, width, T = s["page_size"], s["max_blocks"], s["max_tokens"]
    old, new = s["seq_lens"].long(), s["new_lens"].long()
    rel, add = new < 0, new.clamp(min=0)
    old_b, end_b = (old + ps - 1) // ps, (old + add + ps - 1) // ps
    cu = torch.cat([add.new_zeros(1), add.cumsum(0)])
    fits = ~rel & (cu[1:] <= T) & (end_b <= width)
    need = torch.where(fits, end_b - old_b, 0)
    freed = torch.where(rel, old_b, 0)
    n0 = s["n_free"].long()
    pool = n0 + freed.sum()
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= pool))
    got = torch.where(ok, need, 0)
    # push the released pages, then pop from the top
    col = torch.arange(width, device=old.device)[None, :]
    at = torch.where(rel[:, None] & (col < old_b[:, None]), n0 + (freed.cumsum(0) - freed)[:, None] + col,
                     s["n_pages"])
    stack = torch.cat([s["free_pages"], s["free_pages"].new_zeros(1)])
    stack.scatter_(0, at.reshape(-1), s["table"].reshape(-1))
    pop = pool - 1 - ((upto - need)[:, None] + col - old_b[:, None])
    fresh = ok[:, None] & (col >= old_b[:, None]) & (col < end_b[:, None])
    table = torch.where(fresh, stack[pop.clamp(0, s["n_pages"])], s["table"])
    t = torch.arange(T, device=old.device)
    i = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = i < old.numel()
    i = i.clamp(max=old.numel() - 1)
    live &= ok[i]
    pos = old[i] + t - cu[i]
    page = table[i, (pos // ps).clamp(0, width - 1)].long()
    slots = torch.where(live, page * ps + pos % ps, -1)
    lens = torch.where(rel, 0, torch.where(ok, old + add, old))
    return dict(slots=slots, positions=torch.where(live, pos, -1).int(), cu=cu.clamp(max=T).int(), seq_lens=lens.int(),
                n_free=(pool - got.sum()).int(), table=table, free_pages=stack[: s["n_pages"]])


def _plain_store(s):
    ps, n = s["page_size"], s["n_pages"]
    slots = torch.where(s["slots"] >= 0, s["slots"], n * ps)  # padding goes to the page behind the cache
    page, off = slots // ps, slots % ps
    k = s["new_k"].to(s["k_all"].dtype)
    s["k_all"][page, off] = k
    s["v_all"][page, off] = s["new_v"].to(s["v_all"].dtype)
    # bounds: a page whose first row arrives starts afresh, the others widen
    first = torch.where(off == 0, page, n)
    lo, hi = s["lo_all"].float(), s["hi_all"].float()
    lo[first], hi[first] = float("inf"), float("-inf")
    lo.index_reduce_(0, page, k.float(), "amin")
    hi.index_reduce_(0, page, k.float(), "amax")
    s["lo_all"][:n] = lo[:n].to(k.dtype)
    s["hi_all"][:n] = hi[:n].to(k.dtype)
    return dict(k=s["k_all"][:n], v=s["v_all"][:n], lo=s["lo_all"][:n], hi=s["hi_all"][:n])


def _plain_select(s):
    n_seq, H, D, kb = s["n_seq"], s["n_head_kv"], s["head_dim"], s["k_blocks"]
    width = s["max_blocks"]
    page = s["table"].long().clamp(min=0)
    q = s["q"].double().view(n_seq, H, -1, D)
    # 64 bits: two pages whose scores nearly agree must not change places
    hi = s["hi"][page].permute(0, 2, 3, 1).double()
    lo = s["lo"][page].permute(0, 2, 3, 1).double()
    score = (q.clamp(min=0) @ hi + q.clamp(max=0) @ lo).amax(2)  # [n_seq, H, width]
    b = ((s["seq_lens"].long() + s["page_size"] - 1) // s["page_size"])[:, None, None]
    at = torch.arange(width, device=q.device)
    score = torch.where(at < b, score, float("-inf")).masked_fill(at == b - 1, float("inf"))
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :kb]
    order = torch.where(order < b, order, width).sort(-1).values
    sel = torch.full((n_seq, H, kb), -1, dtype=torch.int32, device=q.device)
    sel[..., : order.shape[-1]] = torch.where(order < b, order, -1).int()
    return sel


def _plain_attn(s):
    n_seq, H, D, ps = s["n_seq"], s["n_head_kv"], s["head_dim"], s["page_size"]
    dev = s["q"].device
    q = s["q"].view(n_seq, H, -1, D)
    if s["sel"] is None:
        block = torch.arange(s["max_blocks"], device=dev).expand(n_seq, 1, -1)
        page = s["table"].long().clamp(min=0)
        k = s["k"][page].flatten(1, 2).transpose(1, 2).float()  # [n_seq, H, tokens, D]
        v = s["v"][page].flatten(1, 2).transpose(1, 2).float()
    else:
        block = s["sel"].long()  # [n_seq, H, k_blocks]
        row = torch.arange(n_seq, device=dev)[:, None, None]
        head = torch.arange(H, device=dev)[None, :, None]
        page = s["table"][row, block.clamp(min=0)].long().clamp(min=0)
        k = s["k"][page, :, head].flatten(2, 3).float()
        v = s["v"][page, :, head].flatten(2, 3).float()
    pos = (block[..., None] * ps + torch.arange(ps, device=dev)).flatten(2)  # [n_seq, 1 or H, tokens]
    live = (pos >= 0) & (pos < s["seq_lens"].long()[:, None, None]) & (block >= 0).repeat_interleave(ps, dim=2)
    bias = torch.zeros((), device=dev)
    if s["mask_rows"] is not None:
        row = torch.arange(n_seq, device=dev)[:, None, None]
        bias = s["mask_rows"][row, pos.clamp(0, s["mask_rows"].shape[1] - 1)].float()
        live = live & (bias != float("-inf"))
        # relative to the row's largest entry: a row of lowest values keeps the scores' own bits
        bias = bias - torch.where(live, bias, float("-inf")).amax(-1, keepdim=True).clamp(min=-65504.0)
        bias = torch.where(live, bias, 0.0)[:, :, None, :]
    k = torch.where(live[..., None], k, 0.0)
    v = torch.where(live[..., None], v, 0.0)
    x = (q @ k.transpose(-1, -2)) * s["scale"] + bias
    x = torch.where(live[:, :, None, :], x, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    return out.reshape(n_seq, -1, D)


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "plan":
        return _plain_plan(state)
    if state["op"] == "store":
        return _plain_store(state)
    if state["op"] == "select":
        return _plain_select(state)
    return _plain_attn(state)


# -------------------------------------------------------------------- work

def work(case):
    ps, n_seq, lens = case["page_size"], case["n_seq"], _lens(case)
    if case["op"] == "plan":
        new = _new_lens(case)
        tokens = sum(max(a, 0) for a in new)
        opened = sum(_ceil(n + max(a, 0), ps) - _ceil(n, ps) for n, a in zip(lens, new))
        back = sum(_ceil(n, ps) for n, a in zip(lens, new) if a < 0)
        # lengths in and out, token starts; slot and position per token; a page read and written per block
        return dict(bytes=4 * 4 * n_seq + 12 * tokens + 8 * (opened + back), flops=10 * (tokens + n_seq))
    H, D = case["n_head_kv"], case["head_dim"]
    if case["op"] == "store":
        tokens = n_seq * case["chunk"]
        rows = sum(_ceil(n + case["chunk"], ps) - n // ps for n in lens)  # pages touched
        part = sum(1 for n in lens if n % ps)  # pages already begun: their bounds are read too
        return dict(bytes=tokens * (H * D * (8 + 4) + 8) + (rows + part) * H * D * 4, flops=2 * tokens * H * D)
    blocks = [_ceil(n, ps) for n in lens]
    fixed = 4 * n_seq * case["n_head"] * D + 4 * n_seq
    if case["op"] == "select":
        return dict(bytes=sum(blocks) * (H * D * 4 + 4) + fixed + 4 * n_seq * H * case["k_blocks"],
                    flops=2 * sum(blocks) * case["n_head"] * D)
    fixed *= 2  # queries and outputs
    if case["k_blocks"]:
        tokens = sum(n - max(0, b - case["k_blocks"]) * ps for n, b in zip(lens, blocks))
        fixed += sum(min(b, case["k_blocks"]) for b in blocks) * H * 4
    else:
        tokens = sum(lens)
    fixed += sum(min(b, case["k_blocks"] or b) for b in blocks) * 4
    return dict(bytes=tokens * (H * D * 4 + (2 if case["mask"] else 0)) + fixed, flops=4 * tokens * case["n_head"] * D)


# ------------------------------------------------------------------- exact

def _exact_plan(s):
    ps, T, width, n_pages = s["page_size"], s["max_tokens"], s["max_blocks"], s["n_pages"]
    old, new = s["seq_lens"].tolist(), s["new_lens"].tolist()
    table, stack = s["table"].tolist(), s["free_pages"].tolist()
    top, lens, started = int(s["n_free"][0]), list(old), [0]
    for i, n in enumerate(old):
        if new[i] < 0:
            for b in range(_ceil(n, ps)):
                stack[top] = table[i][b]
                top += 1
            lens[i] = 0
        started.append(started[-1] + max(new[i], 0))
    slots, positions, asked, pool = [-1] * T, [-1] * T, 0, top
    for i, n in enumerate(old):
        if new[i] <= 0 or started[i + 1] > T or _ceil(n + new[i], ps) > width:
            continue
        need = _ceil(n + new[i], ps) - _ceil(n, ps)
        asked += need
        if need and asked > pool:
            continue
        for b in range(_ceil(n, ps), _ceil(n + new[i], ps)):
            top -= 1
            table[i][b] = stack[top]
        for j in range(new[i]):
            slots[started[i] + j] = table[i][(n + j) // ps] * ps + (n + j) % ps
            positions[started[i] + j] = n + j
        lens[i] = n + new[i]
    dev = s["table"].device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(slots=torch.tensor(slots, dtype=torch.int64, device=dev), positions=i32(positions),
                cu=i32([min(c, T) for c in started]), seq_lens=i32(lens), n_free=i32([top]), table=i32(table),
                free_pages=i32(stack))


def _exact_store(s):
    n, ps = s["n_pages"], s["page_size"]
    dtype = s["k_all"].dtype
    k, v = s["k_all"][:n].double(), s["v_all"][:n].double()
    lo, hi = s["lo_all"][:n].double(), s["hi_all"][:n].double()
    slots = s["slots"].tolist()
    pages = {}
    for t, at in enumerate(slots):
        if at >= 0:
            pages.setdefault(at // ps, []).append((t, at % ps))
    for p, rows in pages.items():
        t, off = [r[0] for r in rows], [r[1] for r in rows]
        new = s["new_k"][t].to(dtype).double()
        k[p, off] = new
        v[p, off] = s["new_v"][t].to(dtype).double()
        a, b = new.min(0).values, new.max(0).values
        lo[p] = a if 0 in off else torch.minimum(a, lo[p])
        hi[p] = b if 0 in off else torch.maximum(b, hi[p])
    return dict(k=k, v=v, lo=lo, hi=hi)


def _exact_select(s):
    H, kb, ps = s["n_head_kv"], s["k_blocks"], s["page_size"]
    out = torch.full((s["n_seq"], H, kb), -1, dtype=torch.int32)
    group = s["n_head"] // H
    for i, n in enumerate(s["seq_lens"].tolist()):
        b = _ceil(n, ps)
        if not b:
            continue
        pages = s["table"][i, :b].long()
        lo, hi = s["lo"][pages].double(), s["hi"][pages].double()
        q = s["q"][i].double()
        for h in range(H):
            best = torch.stack([torch.maximum(lo[:, h] * q[h * group + j], hi[:, h] * q[h * group + j]).sum(-1)
                                for j in range(group)]).max(0).values.tolist()
            older = sorted(range(b - 1), key=lambda x: (-best[x], x))[: kb - 1]
            chosen = sorted(older + [b - 1])
            out[i, h, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out.to(s["q"].device)


def _exact_attn(s):
    H, D, ps = s["n_head_kv"], s["head_dim"], s["page_size"]
    group = s["n_head"] // H
    out = torch.zeros((s["n_seq"], s["n_head"], D), dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(s["seq_lens"].tolist()):
        for h in range(H):
            if s["sel"] is None:
                blocks = torch.arange(_ceil(n, ps), device=out.device)
            else:
                blocks = s["sel"][i, h].long()
                blocks = blocks[blocks >= 0]
            pos = (blocks[:, None] * ps + torch.arange(ps, device=out.device)).reshape(-1)
            pos = pos[pos < n]
            if s["mask_rows"] is not None:
                pos = pos[s["mask_rows"][i, pos] != float("-inf")]
            if not pos.numel():
                continue
            page = s["table"][i, pos // ps].long()
            k, v = s["k"][page, pos % ps, h].double(), s["v"][page, pos % ps, h].double()
            x = k @ s["q"][i, h * group:(h + 1) * group].double().T * s["scale"]
            if s["mask_rows"] is not None:
                x = x + s["mask_rows"][i, pos].double()[:, None]
            out[i, h * group:(h + 1) * group] = torch.softmax(x, 0).T @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "select":
        return _exact_select(s)
    return _exact_attn(s)
