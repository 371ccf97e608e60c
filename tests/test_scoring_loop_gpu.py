"""A beam search over the paged cache with every operator that it takes: plan,
store, chunk attention, log probabilities, fork and copy, drafts that are taken
back, and requests that end.  Each attention output is checked against 64 bits over
the cache as it is, and after every step the cache against what the tokens of each
beam stored, bit for bit."""
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_ref as R
from chunk_ref import chunk_ref, logprobs_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def B():
    import b200_decode

    return b200_decode


@pytest.mark.parametrize("dtype,ps,hq,hkv,d", [("f16", 16, 8, 2, 128), ("bf16", 5, 6, 2, 64)])
def test_beam_search(dtype, ps, hq, hkv, d):
    bw, t = B(), R.DTYPES[dtype]
    g = torch.Generator("cuda").manual_seed(d)
    layers, vocab, width, beams, requests = 2, 211, 96, 3, 2
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    emb, wq = rand(vocab, width), [rand(width, hq * d) / 10 for _ in range(layers)]
    wk, wv = ([rand(width, hkv * d) / 10 for _ in range(layers)] for _ in range(2))
    wo, head = [rand(hq * d, width) / 30 for _ in range(layers)], rand(width, vocab) / 5
    n, max_blocks = beams * requests, 40
    n_pages = n * max_blocks
    caches = []
    for _ in range(layers):
        kv = [torch.full((n_pages, ps, hkv, d), float("nan"), dtype=t, device="cuda") for _ in range(2)]
        caches.append(bw.PagedKV(*kv, *(torch.zeros((n_pages, hkv, d), dtype=t, device="cuda") for _ in range(2))))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, table = i32([0] * n), torch.full((n, max_blocks), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.randperm(n_pages, device="cuda", generator=g).int(), i32([n_pages])
    stored = [[] for _ in range(n)]  # per row and token: its K and V in every layer

    def step(tokens):
        """tokens[s]: what row s appends; the logits of every new token."""
        new = [len(x) for x in tokens]
        plan = bw.paged_plan(i32(new), lens, table, free, n_free, ps, sum(new) + 2)
        cu, at_lens = plan.cu.cpu().numpy(), plan.seq_lens.cpu().numpy()
        x = emb[[tok for row in tokens for tok in row]]
        x = torch.cat([x, torch.zeros((2, width), device="cuda")])
        kept = [[] for _ in range(sum(new))]
        for layer, cache in enumerate(caches):
            q, k, v = x @ wq[layer], x @ wk[layer], x @ wv[layer]
            q[:-2] += plan.positions[:-2, None] / 50.0  # a position's mark
            bw.paged_store(cache, k, v, plan.slots)
            q = q.to(t).unflatten(1, (hq, d))
            out = torch.zeros_like(q)
            bw.paged_prefill(cache, q, table, lens, plan.cu, d ** -0.5, out=out)
            c = dict(k=cache.k.double().cpu().numpy(), v=cache.v.double().cpu().numpy(), table=table.cpu().numpy(),
                     lens=at_lens)
            want, tol = chunk_ref(c, q, cu, ps, d ** -0.5)
            assert ((out.double() - want).abs()[:-2] <= tol[:-2]).all()
            for i in range(sum(new)):
                kept[i].append((k[i].to(t).cpu(), v[i].to(t).cpu()))
            x = x + out.float().flatten(1) @ wo[layer]
        for s in range(n):
            stored[s] += kept[cu[s]:cu[s + 1]]
        return x[:-2] @ head

    def branch(src, keep):
        """Rows become prefixes of rows; the pages that cannot be shared are copied."""
        f = bw.paged_fork(i32(src), i32(keep), lens, table, free, n_free, ps)
        for cache in caches:
            bw.paged_copy(cache, f.copy_src, f.copy_dst, f.copy_rows)
        stored[:] = [list(stored[j][:m]) if j >= 0 else [] for j, m in zip(src, keep)]

    def check():
        tab, m = table.cpu(), lens.tolist()
        assert m == [len(x) for x in stored]
        for layer, cache in enumerate(caches):
            for s in range(n):
                if m[s]:
                    pos = torch.arange(m[s])
                    page = tab[s, pos // ps].long()
                    for part, have in enumerate((cache.k, cache.v)):
                        rows = have.cpu()[page, pos % ps].flatten(1)
                        assert torch.equal(rows, torch.stack([x[layer][part] for x in stored[s]]))
        held = {int(p) for s in range(n) for p in tab[s, : R.ceil_div(m[s], ps)]}
        spare = free.cpu()[: int(n_free)].tolist()
        assert not held & set(spare) and len(held) + len(set(spare)) == n_pages

    prompts = [list(range(3, 40)), list(range(60, 73))]
    logits = step([prompts[0], [], [], prompts[1], [], []])
    check()
    ends = [len(prompts[0]) - 1, sum(map(len, prompts)) - 1]
    r = bw.token_logprobs(logits[ends], None, beams)
    branch([0] * beams + [beams] * beams, [len(prompts[0])] * beams + [len(prompts[1])] * beams)
    check()
    score = r.top_logprobs.double().cpu()
    tokens = r.top_ids.flatten().tolist()
    for turn in range(6):
        # two drafts behind every beam's token; only the token itself is kept
        logits = step([[tok, 5, 9] for tok in tokens])
        check()
        r = bw.token_logprobs(logits, i32([5, 9, -1] * n), beams)
        want = logprobs_ref(logits.double(), i32([5, 9, -1] * n), beams)
        assert torch.equal(r.top_ids, want[2])
        # half a unit of f32 for each of a few dozen roundings of values below 32
        assert (r.logprob.double() - want[0]).abs().max() < 48 * 32 * 2.0 ** -24
        assert (r.entropy.double() - want[1]).abs().max() < 48 * 32 * 2.0 ** -24
        now = score.flatten()[:, None] + r.top_logprobs[::3].double().cpu()  # [rows, beams]
        src, tokens, score = [], [], []
        for q in range(requests):
            best = now[q * beams:(q + 1) * beams].flatten().topk(beams)
            src += [q * beams + int(i) // beams for i in best.indices]
            tokens += [int(r.top_ids[3 * (q * beams + int(i) // beams), int(i) % beams]) for i in best.indices]
            score.append(best.values)
        score = torch.stack(score)
        branch(src, [len(stored[j]) - 2 for j in src])
        check()
    branch([-1] * n, [0] * n)
    check()
    assert int(n_free) == n_pages and B().device_status(reset=True) == 0


def calls(seed):
    """One call of every operator on seeded inputs, as a function, and the tensors that it leaves."""
    bw = B()
    r = np.random.default_rng(seed)
    c = R.make_cache(r, [300, 77, 0], 16, 2, 128, "f16")
    dk, dv = R.to_device(c, "f16")
    cache = bw.PagedKV(dk, dv)
    i32 = lambda v: torch.from_numpy(np.asarray(v, np.int32)).cuda()  # noqa: E731
    q = torch.from_numpy(r.standard_normal((210, 8, 128)).astype(np.float32)).cuda().half()
    table, lens, cu = i32(c["table"]), i32(c["lens"]), i32([0, 200, 205, 210])
    logits = torch.from_numpy(r.standard_normal((40, 5000)).astype(np.float32)).cuda()
    free, n_free = i32(r.permutation(60)), i32([40])
    out = torch.zeros_like(q)
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in
          (bw.paged_prefill_workspace_size(128, 210, 3, 8, 2), bw.paged_fork_workspace_size(3, table.shape[1], 60))]
    new = torch.zeros_like(table)
    src, keep, tokens = i32([0, 0, 1]), i32([290, 33, 70]), i32(r.integers(0, 5000, 40))
    left = torch.empty_like(lens), torch.empty_like(n_free)

    def run():
        bw.paged_prefill(cache, q, table, lens, cu, 0.1, out=out, workspace=ws[0])
        f = bw.paged_fork(src, keep, lens, table, free, n_free, 16, table_out=new, seq_lens_out=left[0],
                          n_free_out=left[1], workspace=ws[1])
        p = bw.token_logprobs(logits, tokens, 7)
        return [out, new, left[0], left[1], f.copy_src, f.copy_dst, f.copy_rows, p.logprob, p.entropy, p.top_ids,
                p.top_logprobs]

    return run


def test_two_streams_at_once():
    """Two programs' calls beside one another, each with workspaces of its own."""
    runs = [calls(1), calls(2)]
    alone = []
    for run in runs:
        alone.append([x.clone() for x in run()])
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, run in zip(streams, runs):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    last = run()
                got.append(last)
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert B().device_status(reset=True) == 0


FIRST = """
import sys
sys.path[:0] = %r
import torch
import test_scoring_loop_gpu as t
run = t.calls(3)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(got, want))
assert t.B().device_status() == 0
print("captured")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.join(os.path.dirname(here), "llama-cpp-ascend310b4-addon_b200")]
    p = subprocess.run([sys.executable, "-c", FIRST % paths], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]
