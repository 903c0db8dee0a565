"""Calls of the serving operators (include/fyodor_hip_serving.h) at the ends of what they allow, on an MI355X against
the statements in serving_check.py."""
import numpy as np
import pytest

from serving_check import F32_HALF, Pages, angles_of, attention_bound
from test_gpu_serving import (DeviceCache, DevicePages, Server, check_attention, dev, env,   # noqa: F401 (fixtures)
                              make_attention, run_attention, run_store)

pytestmark = pytest.mark.gpu


# ---- steps that do not fit --------------------------------------------------

@pytest.mark.parametrize("requests", [3, 1027])
def test_rows_cut_off(env, dev, requests):
    """Rows past max_tokens are the step's last ones; the others keep position lengths - counts + j and their slots,
    whether a request brings more than fits by itself or the ones before it took the room."""
    table = np.full((requests, 4), -1, np.int32)
    table[:3] = np.arange(12).reshape(3, 4)
    none = [0] * (requests - 3)
    for counts, room, want in (([5, 6, 9], 8, [35, 36, 37, 38, 39, 24, 25, 26]),
                               ([30, 1, 1], 4, [10, 11, 12, 13]),
                               ([0, 6, 2], 7, [24, 25, 26, 27, 28, 29, 7]),
                               ([40, 2**31 - 1, 2**31 - 1], 3, [0, 1, 2])):
        state = Pages(requests, 4, 20, 16, np.arange(20))
        state.table[:], state.held[:3], state.free_count[0] = table, [3, 2, 1], 8
        lengths = [40, 30, 9] + none
        device = DevicePages(env, dev, state, room)
        device.step(lengths, counts + none)
        starts = dev.get(device.starts, np.empty(requests + 1, np.int32))
        assert np.array_equal(starts[:4], np.minimum(np.cumsum([0] + counts), 2**31 - 1))
        assert np.all(starts[3:] == starts[3])
        positions, slots = (dev.get(p, np.empty(room + 1, np.int32)) for p in (device.positions, device.slots))
        assert positions.tolist() == want + [-7]
        request = np.repeat([0, 1, 2], np.minimum(counts, 50))[:room]
        assert np.array_equal(slots[:-1], table[request, np.array(want) // 16] * 16 + np.array(want) % 16)
        assert slots[-1] == -7
        # What the statement of the page step gives.
        device.check(*state.step(lengths, counts + none, room))


@pytest.mark.parametrize("max_tokens", [7, 48])
def test_steps_cut_off(env, dev, max_tokens):
    """Page step, store and attention agree on the positions of a step's rows when not all of them fit: no row sees
    one that comes later or was never stored."""
    server = Server(env, dev, max_tokens=max_tokens)
    for lengths, counts in [([40, 30, 0, 0, 0], [40, 30, 0, 0, 0]), ([5, 20, 3, 0, 0], [5, 20, 3, 0, 0]),
                            ([300, 21, 4, 9, 0], [300, 1, 1, 9, 0]), ([6, 28, 11, 16, 12], [1, 7, 7, 7, 12])]:
        server.inputs(lengths, counts)
        server.launch()
        env[0].sync(env[2])
        server.check(lengths, counts)


# ---- the cache: elements that are not finite ---------------------------------

@pytest.mark.parametrize("page_tokens,width,heads,rotated,shift", [(16, 64, 2, 64, 0), (64, 128, 2, 20, 0),
                                                                   (128, 512, 0, 0, 0), (32, 256, 0, 0, 4)])
def test_loads_of_what_is_not_finite(env, dev, page_tokens, width, heads, rotated, shift):
    """A head's rows of a page with an infinite or NaN element read as NaN, all of them, from a long run and from a
    single token, and still after a finite token; other heads read as stored."""
    rt, kern, stream = env
    rng = np.random.default_rng(width)
    kv_heads = 4
    cache = DeviceCache(env, dev, 3, page_tokens, kv_heads, width, rng)
    frequencies, _ = kern.rope_frequencies(max(rotated, 2), 10000.0)

    def read(slots):
        n = kv_heads * width
        rows = dev.put(np.zeros((len(slots), 2 * n), np.float32))
        kern.kv8_load(cache.arg, dev.put(np.array(slots, np.int32)), len(slots), rows, 2 * n, rows + 4 * n, 2 * n, stream)
        rt.sync(stream)
        return dev.get(rows, np.empty((len(slots), 2, kv_heads, width), np.float32))

    def store(slots, bad):
        """Rows into these slots; bad: the values at element `width - 3` of the last row's K and V heads 0, 1, ..."""
        x = rng.standard_normal((len(slots), heads + 2 * kv_heads, width)).astype(np.float32)
        for h, b in enumerate(bad):
            x[-1, heads + h, width - 3] = x[-1, heads + kv_heads + h, width - 3] = b
        angles = angles_of(np.array(slots) % page_tokens, frequencies, 1.0).astype(np.float32)
        with np.errstate(invalid="ignore"):
            run_store(env, dev, cache, slots, x, heads, rotated, False, angles, shift)
        cache.check()

    def check(slots, bad):
        got = read(slots)
        assert np.all(np.isnan(got[:, :, bad]))
        fine = [h for h in range(kv_heads) if h not in bad]
        for kind, c in enumerate((cache.k, cache.v)):
            page, t = np.array(slots) // page_tokens, np.array(slots) % page_tokens
            want = c.codes[page, :, t].astype(np.float32) * c.scales[page][..., None]
            assert np.array_equal(got[:, kind, fine], want[:, fine])

    # A run from a page's first slot on, a token more, a finite one after it.
    run = list(range(page_tokens, page_tokens + page_tokens - 3))
    store(run, [np.inf, -np.inf, np.nan])
    check(run, [0, 1, 2])
    store([run[-1] + 1], [])
    check(run + [run[-1] + 1], [0, 1, 2])
    # A page that was fine; then infinity after NaN and NaN after infinity.
    run = list(range(2 * page_tokens, 2 * page_tokens + 5))
    store(run, [])
    check(run, [])
    store([run[-1] + 1], [np.inf, np.nan, -np.inf])
    store([run[-1] + 2], [np.nan, np.inf, -np.inf])
    run += [run[-1] + 1, run[-1] + 2]
    check(run, [0, 1, 2])
    # A whole page, and anew.
    store(list(range(page_tokens)), [-np.inf, np.inf, np.nan])
    check(list(range(page_tokens)), [0, 1, 2])
    store([0], [])
    check([0], [])


# ---- the cache: pages whose rows have gaps ------------------------------------

@pytest.mark.parametrize("page_tokens,kv_heads,width,pages,rotated", [
    (16, 2, 64, 9, 32), (32, 8, 64, 60, 64), (64, 1, 128, 5, 0), (128, 2, 256, 4, 256), (128, 8, 128, 12, 128),
    (64, 2, 512, 3, 30)])
def test_store_with_gaps(env, dev, page_tokens, kv_heads, width, pages, rotated):
    """Pages of which some positions are not stored, as rows that are left out or without rows at all: their runs share
    the page's scale, which grows from run to run."""
    rng = np.random.default_rng(pages)
    cache = DeviceCache(env, dev, pages, page_tokens, kv_heads, width, rng)
    frequencies, _ = env[1].rope_frequencies(max(rotated, 2), 10000.0)
    for kept, rows_of_others in ((0.5, True), (0.8, False), (0.05, True), (0.95, False)):
        slots, sizes = [], []
        for page in rng.permutation(pages):
            positions = np.arange(page_tokens)
            keep = rng.random(page_tokens) < kept
            if rng.random() < 0.5:
                keep[0] = True
            here = page * page_tokens + positions
            here = np.where(keep, here, rng.choice([-1, pages * page_tokens, -2**31])) if rows_of_others else here[keep]
            slots += here.tolist()
            sizes += (1 + np.arange(len(here)) * rng.choice([0, 0.3, -0.9 / page_tokens])).tolist()
            if rng.random() < 0.3:
                slots += [-1] * 5
                sizes += [1.0] * 5
        x = rng.standard_normal((len(slots), 2 * kv_heads, width)) * np.array(sizes)[:, None, None]
        angles = angles_of(np.array(slots) % page_tokens, frequencies, 1.0).astype(np.float32)
        run_store(env, dev, cache, np.array(slots, np.int64).astype(np.int32), x.astype(np.float32), 0, rotated, True,
                  angles)
        cache.check()


def test_store_with_far_gaps(env, dev):
    """Two rows of a page with 127 left out between them, and single positions of a page in turn."""
    rng = np.random.default_rng(5)
    cache = DeviceCache(env, dev, 3, 128, 2, 64, rng)
    for slots in ([0] + [-1] * 127 + [127] + [-1] * 127 + [128] + [-1] * 40 + [200], list(range(256, 384, 2)),
                  [-1] * 300 + [383] + [-1] * 300):
        x = rng.standard_normal((len(slots), 4, 64)).astype(np.float32)
        x *= (1 + np.arange(len(slots), dtype=np.float32))[:, None, None]
        run_store(env, dev, cache, slots, x, 0, 0, False, np.zeros((len(slots), 32, 2), np.float32))
        cache.check()


# ---- attention: work split over the positions ------------------------------

def dense_attention(cache, table, q, first, counts, window, scale):
    """Attention in 64 bits of requests that share the pages of `table` (one row of it), request r's counts[r] rows
    from position first[r] on: (out, bound)."""
    rows, heads, width = q.shape
    kv_heads, page_tokens = cache.kv_heads, cache.page_tokens
    position = np.concatenate([f + np.arange(n) for f, n in zip(first, counts)])
    t = np.arange(position.max() + 1)
    seen = t <= position[:, None]
    if window:
        seen &= t > position[:, None] - window
    out, bound = np.empty(q.shape), np.empty((rows, heads))
    for h in range(kv_heads):
        k, v = (c.values()[table[t // page_tokens], h, t % page_tokens] for c in (cache.k, cache.v))
        top = np.where(seen, np.abs(v).max(1), 0).max(1)
        for g in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
            x = q[:rows, g].astype(np.float64)
            weight = np.where(seen, np.abs(x) @ np.abs(k).T, 0).max(1) * abs(scale)
            s = np.where(seen, x @ k.T * scale, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            out[:, g] = e @ v / e.sum(1, keepdims=True)
            bound[:, g] = attention_bound(weight, top, width, int(t[-1]) + 1)
    return out, bound


@pytest.mark.parametrize("requests,tokens,heads,kv_heads,width,window,at", [
    (21, 9, 32, 8, 128, 8192, 43), (63, 5, 32, 8, 128, 8192, 0), (20, 5, 32, 8, 128, 6144, 44),
    (31, 10, 20, 4, 128, 8192, 33),
])
def test_drafts_under_a_long_window(env, dev, requests, tokens, heads, kv_heads, width, window, at):
    """Drafts of many requests whose tiles have unequal numbers of steps, so of shares: the first new token at
    positions `at`, at + 1, .. of a step of 64. Scratch holds NaN: a share that nobody wrote shows."""
    first = window + 64 * 3 + at + np.arange(requests)
    counts = [tokens] * requests
    lengths = first + tokens
    cache, _, _, table = make_attention(env, dev, [int(lengths.max())], [1], heads, kv_heads, width, 64, 31)
    rng = np.random.default_rng(32)
    q = rng.standard_normal((requests * tokens, heads, width)).astype(np.float32)
    starts = (tokens * np.arange(requests + 1)).astype(np.int32)
    want, bound = dense_attention(cache, table[0], q, first, counts, window, width ** -0.5)
    size = env[1].kv8_attention_bytes(cache.arg, len(q), requests, tokens, 32768, heads, window)
    for workspace in (size, size // 2 & ~15, 0):
        got = run_attention(env, dev, cache, q, starts, lengths, np.repeat(table, requests, 0), window=window,
                            longest=32768, workspace=workspace)
        off = np.abs(got - want).max(2)
        assert np.all(off <= bound), (workspace, np.argwhere(~(off <= bound))[:5].tolist())


# ---- attention: scores at the ends of fp32 ----------------------------------

SCORE_BATCHES = [([300], [1]), ([80], [80]), ([300, 80, 9], [1, 80, 4]), ([9000], [1])]


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (2, 1, 512)])
@pytest.mark.parametrize("lengths,counts", SCORE_BATCHES)
@pytest.mark.parametrize("size", [1e7, 3e8, 1e20, 1e33])
def test_far_scores(env, dev, heads, kv_heads, width, lengths, counts, size):
    """Scores of `size`, where fp32 has no fractions left: one position takes a row (all but those whose best two
    scores fp32 does not tell apart)."""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 64, 33, spread=0.1)
    q *= np.float32(size ** 0.5)
    cache.k.scales[table[table >= 0][table[table >= 0] < cache.pages]] *= np.float32(size ** 0.5)
    cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    scale, clear = np.float32(width ** -0.5), 0
    for r, n in enumerate(lengths):
        t = np.arange(n)
        page = table[r, t // 64]
        for h in range(heads):
            k, v = (c.values()[page, h * kv_heads // heads, t % 64] for c in (cache.k, cache.v))
            for row in range(starts[r], starts[r + 1]):
                last = n - (starts[r + 1] - row) + 1
                x = q[row, h].astype(np.float64)
                s = k[:last] @ x * scale
                top = np.abs(v[:last]).max()
                assert np.all(np.abs(got[row, h]) <= top * (1 + 2.0 ** -16))
                # Off by this much each (attention_bound's part of the scores), another position weighs e^-50.
                off = (np.abs(k[:last]) @ np.abs(x)).max() * scale * (2.0 ** -22 + (width / 16 + 12) * F32_HALF)
                order = np.argsort(s)
                if last == 1 or s[order[-1]] - s[order[-2]] > 2 * off + 50:
                    clear += 1
                    assert np.abs(got[row, h] - v[order[-1]]).max() <= attention_bound(0, top, width, n), (row, h)
    assert clear > heads * sum(counts) // 2


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (2, 1, 512)])
@pytest.mark.parametrize("lengths,counts", SCORE_BATCHES)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_beyond_fp32(env, dev, heads, kv_heads, width, lengths, counts, sign):
    """Scores of about 1e42, of either sign or all of one: no answer in fp32, and none that looks like one. What sees
    nothing still gives zeros."""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 64, 34, spread=0.1)
    used = table[table >= 0][table[table >= 0] < cache.pages]
    q *= np.float32(1e21)
    cache.k.scales[used] *= np.float32(1e21)
    cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    assert np.all(np.isnan(got[:starts[-1]]))
    # All scores far above, or far below.
    q = np.abs(q)
    cache.k.codes[:] = sign * np.maximum(np.abs(cache.k.codes), 1)
    cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    assert np.all(np.isnan(got[:starts[-1]]))
    table[:] = -1
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    assert np.all(got[:starts[-1]] == 0)


def test_some_scores_below_fp32(env, dev):
    """A position whose score is below fp32's range weighs nothing beside others."""
    for heads, kv_heads, width in ((8, 2, 64), (4, 2, 256)):
        for tokens in (1, 40):
            lengths = [200]
            cache, q, starts, table = make_attention(env, dev, lengths, [tokens], heads, kv_heads, width, 64, 35)
            q = np.abs(q)
            far = table[0, 1]
            cache.k.codes[far] = -np.maximum(np.abs(cache.k.codes[far]), 1)
            cache.k.scales[far] = 1e38
            cache.put()
            got = run_attention(env, dev, cache, q, starts, lengths, table)
            hole = table.copy()
            hole[0, 1] = -1
            check_attention(cache, q, got, starts, lengths, hole)


@pytest.mark.parametrize("heads,kv_heads,width,counts", [(4, 2, 64, [1, 1, 1]), (2, 1, 128, [20, 1, 2]),
                                                        (2, 2, 256, [1, 70, 3]), (2, 1, 512, [1, 2, 1])])
@pytest.mark.parametrize("workspace", [None, 0])
def test_small_and_large_values(env, dev, heads, kv_heads, width, counts, workspace):
    """Equal scores over many positions whose values are as small as a page's scale can be (which a head of zeros
    stores, too), alone and before larger values, and over the largest ones."""
    lengths = [70000, 40000, 3]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 128, 36, spread=0.0)
    q[:] = 0
    small, large = 2.0 ** -100, 2.0 ** 120
    codes = cache.v.codes.copy()
    for base, tail in ((small, small), (large, large), (small, 1 / 90), (small, 2.0 ** 15)):
        cache.v.codes[:] = codes
        for r, n in enumerate(lengths):
            need = -(-n // 128)
            few = 2 * need // 3
            cache.v.scales[table[r, :few]], cache.v.scales[table[r, few:need]] = base, tail
            if tail != base:
                cache.v.codes[table[r, :few]] = 0
        cache.put()
        got = run_attention(env, dev, cache, q, starts, lengths, table, workspace=workspace)
        values = cache.v.values()
        for r, n in enumerate(lengths):
            t = np.arange(n)
            for h in range(kv_heads):
                v = values[table[r, t // 128], h, t % 128]
                total, top = np.cumsum(v, 0), np.abs(v).max()
                bound = attention_bound(0, top, width, n)   # all scores are 0 exactly
                for row in range(starts[r], starts[r + 1]):
                    last = n - (starts[r + 1] - row) + 1
                    want = total[last - 1] / last
                    assert np.abs(want).max() > 2 * bound
                    off = np.abs(got[row, h * heads // kv_heads:(h + 1) * heads // kv_heads] - want)
                    assert np.all(off <= bound), (base, tail, row)
