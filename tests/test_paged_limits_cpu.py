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


RANGE_TEST = r'''
// PaRange (csrc/paged_range.cuh) on host threads: one per CUDA thread, the warp
// and block functions built from barriers.
#include <algorithm>
#include <barrier>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
struct Dim { unsigned x; };
static thread_local Dim threadIdx, blockIdx;
static Dim gridDim;

template <int W>
struct Cta {
    std::barrier<> all{32 * W};
    std::vector<std::unique_ptr<std::barrier<>>> warp;
    int lanes[W][32];
    Cta() { for (int w = 0; w < W; ++w) warp.push_back(std::make_unique<std::barrier<>>(32)); }
};
constexpr int W = 4;
static Cta<W>* cta;
static int lane_id() { return threadIdx.x & 31; }
static int warp_id() { return threadIdx.x >> 5; }
static int from_lane(int v, int src) {
    cta->lanes[warp_id()][lane_id()] = v;
    cta->warp[warp_id()]->arrive_and_wait();
    const int r = cta->lanes[warp_id()][src];
    cta->warp[warp_id()]->arrive_and_wait();
    return r;
}
static int __shfl_up_sync(unsigned, int v, int o) { return from_lane(v, lane_id() >= o ? lane_id() - o : lane_id()); }
static int __shfl_sync(unsigned, int v, int src) { return from_lane(v, src & 31); }
static unsigned __ballot_sync(unsigned, bool p) {
    unsigned r = 0;
    cta->lanes[warp_id()][lane_id()] = p;
    cta->warp[warp_id()]->arrive_and_wait();
    for (int i = 0; i < 32; ++i) r |= (unsigned)(cta->lanes[warp_id()][i] != 0) << i;
    cta->warp[warp_id()]->arrive_and_wait();
    return r;
}
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }
static void __syncthreads() { cta->all.arrive_and_wait(); }
#include "paged_range.cuh"

struct Found { int cb, ce, fb, fe, seq0, base0, per_cta; };

// The ranges of every warp; units(s) is `first` when a thread asks for the first
// time and `later` after that.
static std::vector<Found> ranges(const std::vector<int>& first, const std::vector<int>& later, int segs, int ctas) {
    const int n = (int)first.size();
    std::vector<Found> out(ctas * W);
    gridDim.x = ctas;
    for (int b = 0; b < ctas; ++b) {
        Cta<W> c;
        cta = &c;
        b200::PaRangeShared<W> sh;
        memset(&sh, 0x7f, sizeof sh);  // shared memory holds anything
        std::vector<std::thread> t;
        for (int i = 0; i < 32 * W; ++i)
            t.emplace_back([&, i] {
                threadIdx.x = i;
                blockIdx.x = b;
                std::vector<char> seen(n, 0);
                auto units = [&](int s) {
                    if (s < 0 || s >= n) { printf("sequence %d of %d\n", s, n); exit(9); }
                    const int u = seen[s] ? later[s] : first[s];
                    seen[s] = 1;
                    return u;
                };
                const b200::PaRange<W> r(sh, n, segs, units);
                if ((i & 31) == 0) out[b * W + i / 32] = {r.cb, r.ce, r.fb, r.fe, r.seq0, r.base0, r.per_cta};
            });
        for (auto& x : t) x.join();
    }
    return out;
}

int main() {
    srand(5);
    for (int n : {1, 7, 128, 129, 200, 400})
        for (int kind = 0; kind < 4; ++kind) {
            const int segs = 1 + rand() % 3, ctas = 1 + rand() % 5;
            std::vector<int> len(n), other(n);
            for (auto& v : len) v = kind == 1 ? rand() % 2 : kind == 2 ? (rand() % 50 == 0) * 1000 : rand() % 40;
            if (kind == 3) len[rand() % n] = 5000;
            for (auto& v : other) v = rand() % 3 ? 0 : rand() % 60;
            // lengths that stay: the ranges cover every unit in order, each begins where it says
            std::vector<int> start(n + 1, 0);
            for (int s = 0; s < n; ++s) start[s + 1] = start[s] + len[s] * segs;
            int at = 0;
            for (const Found& f : ranges(len, len, segs, ctas)) {
                if (f.fb >= f.fe) continue;
                if (f.fb != at || f.fb < f.cb || f.fe > f.ce) return 1;
                at = f.fe;
                if (f.seq0 < 0 || f.seq0 >= n || f.base0 != start[f.seq0] || f.fb < start[f.seq0] || f.fb >= start[f.seq0 + 1])
                    return 2;
            }
            if (at != start[n]) return 3;
            // lengths that change while the ranges are found: nothing outside the batch
            for (const Found& f : ranges(len, other, segs, ctas)) {
                if (f.fb >= f.fe) continue;
                if (f.seq0 < 0 || f.seq0 >= n || f.base0 < 0 || f.base0 > f.fb) {
                    printf("%d sequences, kind %d: warp at unit %d starts in sequence %d, unit %d\n", n, kind, f.fb, f.seq0,
                           f.base0);
                    return 4;
                }
            }
        }
    // the pieces of a segment lie within the grid, whatever length it claims
    for (int grid : {1, 7, 148})
        for (int per : {1, 13, 4000})
            for (int i = 0; i < 2000; ++i) {
                const int from = rand() % (grid * per), nu = 1 + (i % 2 ? rand() % (1 << 27) : rand() % per);
                const int c0 = from / per, k = b200::pa_pieces(from, nu, per, grid);
                if (k < 1 || c0 + k > grid) return 5;
                const long long last = (long long)from + nu - 1;
                if (last < (long long)grid * per && k != (int)(last / per) - c0 + 1) return 6;
            }
    return 0;
}
'''


def test_work_ranges_on_the_host(tmp_path):
    """The split of a batch's units over warps: complete and in order for any
    lengths, and inside the batch even where the lengths change meanwhile."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "ranges.cpp", tmp_path / "ranges"
    src.write_text(RANGE_TEST)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc = os.path.join(root, "llama-cpp-ascend310b4-addon_b200", "csrc")
    r = subprocess.run([gxx, "-std=c++20", "-O1", "-pthread", "-I" + csrc, str(src), "-o", str(exe)], capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stdout)


@no_device
@pytest.mark.parametrize("n_seq,q_stride,out,meets", [
    (2, 512, 0, True), (2, 512, 16, True), (2, 512, -16, True), (2, 512, 4096 - 16, True), (2, 512, -4096 + 16, True),
    (2, 512, 4096, False), (2, 512, -4096, False), (1, 512, 2048, False), (1, 512, 2032, True), (1, 0, 2048, False),
    (1, 0, -2048, False), (1, 0, 16, True),
    # rows of a wider matrix: out behind the last row, in a gap of three rows, or past that
    (3, 2048, 2 * 8192 + 2048, False), (3, 2048, 2 * 8192 + 2032, True), (1, 2048, 2048, False), (3, 2048, 2048, False),
    (3, 2048, 2064, True),
    (3, 2048, -6144, False), (3, 2048, -6144 + 16, True), (2, 4096, 2048, False), (2, 4096, 2032, True),
    (2, 4096, 16384 - 4096, False), (2, 4096, 16384 - 4080, True)])
def test_attn_refuses_an_output_that_meets_the_queries(n_seq, q_stride, out, meets):
    """Rows of 4 heads x 128 f32, 2048 bytes; `out` bytes from the first query."""
    bw = B()
    kv = bw._PagedKVStruct(bw.TYPE_F16, 128, 2, 16, 8, PTR, PTR, 16 * 512, 512, 256, 16 * 512, 512, 256, None, None)
    at = 1 << 20
    rc = bw.lib().b200_paged_attn(C.byref(kv), at, q_stride, n_seq, 4, PTR, 4, 4, PTR, None, 0, None, 0, 1.0, at + out, PTR,
                                  1 << 30, None)
    assert (rc == bw.EINVAL) == meets
