"""How attention over the paged 8-bit cache divides its work
(fyodor_amd/csrc/kv8_shares.h), on the host: every share that is joined is
launched exactly once, and a tile's shares are its steps, for batches of any
lengths, drafts, windows and workspaces."""
import ctypes
import subprocess

import numpy as np
import pytest

from fyodor_amd.build import CSRC, hipcc

SOURCE = r"""
#include <vector>
#include "kv8_shares.h"
using namespace fy;

// What is wrong with how a call is divided: 1 a share that is launched but once too often or not at all, 2 more
// shares than the workspace has places for, 4 shares that are not the tile's steps, 8 more items than workgroups.
extern "C" int divide(const int *starts, const int *lengths, int requests, int count, int max_tokens, int max_length,
    int heads, int kv_heads, int width, int page_tokens, int table_stride, int window, double part, int *form)
{
    Kv8Attention a = {};
    a.cache.pages = 1 << 20;
    a.cache.page_tokens = page_tokens;
    a.cache.kv_heads = kv_heads;
    a.cache.width = width;
    a.count = count;
    a.starts = starts;
    a.lengths = lengths;
    a.table_stride = table_stride;
    a.requests = requests;
    a.max_tokens = max_tokens;
    a.max_length = max_length;
    a.heads = heads;
    a.window = window;
    const Plan whole = plan_of(a, nullptr, SIZE_MAX);
    double bytes = 0;
    for (const Split *s : {&whole.few, &whole.wide})
        if (s->most > 1) bytes += (double)s->most * share_bytes(a, *s);
    const Plan p = plan_of(a, nullptr, (size_t)(bytes * part));
    *form = (p.any_few && p.few.packed ? 1 : 0) | (p.any_few && p.few.most > 1 ? 2 : 0) | (p.any_wide && p.wide.most > 1 ? 4 : 0);
    int wrong = 0;
    long items = 0;
    for (int r = 0; r < requests; ++r) {
        const Request q = request_of(a, r);
        if (q.rows <= 0) continue;
        const bool few = p.any_few && q.rows <= p.most_rows;
        const Split &split = few ? p.few : p.wide;
        const int tile_rows = few ? kRows : kWideRows, tiles = (q.rows + tile_rows - 1) / tile_rows;
        std::vector<int> launched(tiles * (kMostSplits + 1), 0);
        const bool packed = few && split.packed;
        if (packed) {
            const Items n = items_of(a, split, q, p.most_rows);
            items += (long)n.tiles * n.shares;
            for (int left = 0; left < n.tiles * n.shares; ++left) {
                const Item at = item_at(n.tiles, left);
                if (at.tile >= tiles || at.share > kMostSplits) wrong |= 1;
                else ++launched[at.tile * (kMostSplits + 1) + at.share];
            }
        }
        for (int tile = 0; tile < tiles; ++tile) {
            const Range g = range_of(a, q, tile, tile_rows, split.most, split.least);
            if (g.active > split.most) wrong |= 2;
            for (int sp = 0; packed && sp < g.active; ++sp) wrong |= launched[tile * (kMostSplits + 1) + sp] != 1;
            int at = g.begin;
            for (int sp = 0; sp < g.active && g.end > g.begin; ++sp) {
                if (g.from(sp) != at || g.until(sp) <= at) wrong |= 4;
                at = g.until(sp);
            }
            if (at != g.end) wrong |= 4;
        }
    }
    if (p.any_few && p.few.packed && items > (long)((p.few.tile + kRows - 1) / kRows) * requests * p.few.most) wrong |= 8;
    return wrong;
}
"""


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    out = tmp_path_factory.mktemp("shares")
    (out / "shares.hip").write_text(SOURCE)
    subprocess.run([hipcc(), "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-fPIC", "-shared", f"-I{CSRC}",
                    str(out / "shares.hip"), "-o", str(out / "shares.so")], check=True, capture_output=True)
    call = ctypes.CDLL(str(out / "shares.so")).divide
    call.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_int] * 10 + [ctypes.c_double, ctypes.c_void_p]

    def run(lengths, counts, heads, kv_heads, width, page_tokens, window, max_length, max_tokens=None, part=1.0):
        lengths = np.ascontiguousarray(lengths, np.int32)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        form = ctypes.c_int()
        wrong = call(starts.ctypes.data, lengths.ctypes.data, len(lengths), int(starts[-1]),
                     int(max_tokens or max(counts)), int(max_length), heads, kv_heads, width, page_tokens,
                     int(lengths.max()) // page_tokens + 2, window, part, ctypes.byref(form))
        return wrong, form.value
    return run


@pytest.mark.parametrize("requests,tokens,heads,kv_heads,width,window", [
    (21, 9, 32, 8, 128, 8192), (20, 5, 32, 8, 128, 6144), (63, 5, 32, 8, 128, 8192), (31, 10, 20, 4, 128, 8192),
    (21, 5, 32, 8, 128, 12288), (64, 1, 32, 8, 128, 8192), (16, 17, 32, 32, 64, 8192), (40, 33, 6, 6, 64, 0),
])
@pytest.mark.parametrize("part", [1.0, 0.6, 0.4])
def test_drafts_of_many_requests(divide, requests, tokens, heads, kv_heads, width, window, part):
    """Every position of a step of 64 for the first new token, in requests longer than the window and than expected."""
    packed = False
    for first in range(20000, 20064):
        for expected in (32768, 14000):
            lengths = first + tokens + 64 * np.arange(requests) % 4096
            wrong, form = divide(lengths, [tokens] * requests, heads, kv_heads, width, 64, window, expected, part=part)
            assert wrong == 0, (first, expected)
            packed |= bool(form & 1)
    assert packed or part < 1


@pytest.mark.parametrize("seed", range(4))
def test_batches_of_any_kind(divide, seed):
    rng = np.random.default_rng(seed)
    log = lambda low, high: int(round(np.exp(rng.uniform(np.log(low), np.log(high)))))
    forms = set()
    for _ in range(4000):
        heads, kv_heads, width = [(32, 8, 128), (32, 4, 64), (16, 8, 256), (32, 32, 128), (8, 1, 512), (20, 4, 128),
                                  (6, 2, 64), (70, 1, 64), (8, 8, 64)][rng.integers(9)]
        requests, tokens = log(1, 64), [1, log(2, 40), log(2, 700)][rng.integers(3)]
        counts = rng.integers(0, tokens + 1, requests)
        counts[rng.integers(requests)] = tokens
        longest = log(tokens, 60000)
        lengths = np.maximum(rng.integers(0, longest + 1, requests), counts)
        window = [0, 0, log(1, 1000), log(1000, 20000)][rng.integers(4)]
        args = (lengths, counts, heads, kv_heads, width, int(rng.choice([16, 32, 64, 128])), window,
                max(1, [longest, longest // 3, 3 * longest][rng.integers(3)]))
        for part in (1.0, rng.uniform(0, 1)):
            wrong, form = divide(*args, part=part)
            forms.add(form)
            assert wrong == 0, args
    assert {0, 1, 2, 4} <= {f & b for f in forms for b in (0, 1, 2, 4)}
