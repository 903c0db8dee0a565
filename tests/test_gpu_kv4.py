"""The 4-bit paged cache and log probabilities (include/fyodor_hip_kv4.h, include/fyodor_hip_logprobs.h) on an MI355X
against their statements in kv4_check.py, at the sizes and data where they can go wrong. Codes, steps, ids and ranks
are exact; rotated rows are one rounding from 64 bits; attention stays in the bound that attention_bound derives, log
probabilities in the one that logprobs derives."""
import ctypes
import time

import numpy as np
import pytest

from fyodor_amd.hip import Graph, Kernels, Kv4, Runtime
from kv4_check import Cache4, held, logprobs, store
from serving_check import Dev, F32_HALF, Pages, angles_of, attention, attention_bound, rotate
from test_gpu_serving import STEPS, DevicePages

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    rt, kern = Runtime(), Kernels()
    stream = rt.stream()
    yield rt, kern, stream
    rt.sync(stream)


@pytest.fixture()
def dev(env):
    d = Dev(env[0])
    yield d
    env[0].sync(env[2])
    d.close()


class DeviceCache4:
    def __init__(self, env, dev, pages, page_tokens, kv_heads, width, rng):
        self.env, self.dev = env, dev
        self.k, self.v = (Cache4(pages, page_tokens, kv_heads, width, rng, kind) for kind in "kv")
        self.pages, self.page_tokens, self.kv_heads, self.width = pages, page_tokens, kv_heads, width
        self.put()

    def put(self):
        """The statement's codes and steps on the device."""
        self.at = [self.dev.put(x) for x in (self.k.packed(), self.v.packed(), self.k.packed_steps(),
                                             self.v.packed_steps())]
        self.arg = Kv4(*self.at, self.pages, self.page_tokens, self.kv_heads, self.width)

    def check(self):
        """Every bit of the cache, what no row was stored in among them."""
        for c, codes, steps in ((self.k, self.at[0], self.at[2]), (self.v, self.at[1], self.at[3])):
            got = c.unpack_steps(self.dev.get(steps, np.empty(c.steps.size, np.float16)))
            same = (got.view(np.uint16) == c.steps.view(np.uint16)) | (np.isnan(got) & np.isnan(c.steps))
            assert np.all(same), (c.kind, np.argwhere(~same)[:3])
            got = c.unpack(self.dev.get(codes, np.empty(c.codes.size // 2, np.uint8)))
            bad = np.argwhere(got != c.codes)
            assert not len(bad), (c.kind, bad[:3], got[tuple(bad[0])], c.codes[tuple(bad[0])])


def run_store(env, dev, cache, slots, x, heads, rotated, halves, angles, shift=0, pad=0):
    """Rows x [count][heads + 2 kv_heads][width] through the store, into the statement too; the rotated q rows."""
    rt, kern, stream = env
    count, width, kvh = len(slots), cache.width, cache.kv_heads
    n = (heads + 2 * kvh) * width
    rows = np.zeros((count, n + pad), np.float32)
    rows[:, :n] = x.reshape(count, n)
    src = dev.put(rows, shift)
    q_out = dev.put(np.full((count, heads * width + pad), 9.0, np.float32), shift) if heads and rotated else 0
    kern.kv4_store(cache.arg, dev.put(np.asarray(slots, np.int32)), count, src + 4 * heads * width, n + pad,
                   src + 4 * (heads + kvh) * width, n + pad, dev.put(angles) if rotated else 0, rotated, int(halves),
                   src if q_out else 0, n + pad, q_out, heads * width + pad, heads, stream)
    rt.sync(stream)
    k = x[:, heads:heads + kvh]
    if rotated:
        with np.errstate(all="ignore"):
            k = rotate(k, angles, halves).astype(np.float32)
    store(cache.k, cache.v, slots, k, x[:, heads + kvh:])
    assert np.array_equal(dev.get(src, rows), rows, equal_nan=True)
    return dev.get(q_out, np.empty((count, heads * width + pad), np.float32)) if q_out else None


@pytest.mark.parametrize("page_tokens,kv_heads,width,heads,rotated,halves,shift,pad", [
    (16, 2, 64, 4, 64, False, 0, 0), (32, 1, 64, 0, 0, False, 0, 0), (64, 3, 128, 3, 64, True, 0, 0),
    (128, 8, 128, 8, 128, False, 0, 4), (64, 2, 256, 2, 64, True, 4, 1), (16, 1, 512, 2, 512, True, 0, 0),
    (32, 2, 128, 4, 38, False, 0, 0), (32, 2, 128, 4, 38, True, 8, 2), (128, 1, 512, 0, 128, False, 0, 0),
    (16, 5, 64, 5, 20, True, 0, 0), (16, 7, 64, 7, 16, True, 0, 0),
])
def test_store(env, dev, page_tokens, kv_heads, width, heads, rotated, halves, shift, pad):
    """Prompts, tokens one by one, positions written again, rows in any order, rows that go nowhere."""
    rng = np.random.default_rng(page_tokens + width)
    pages = 7
    cache = DeviceCache4(env, dev, pages, page_tokens, kv_heads, width, rng)
    order = rng.permutation(pages)
    slot = lambda request, p: int(order[3 * request + p // page_tokens]) * page_tokens + p % page_tokens
    frequencies, _ = env[1].rope_frequencies(max(rotated, 2), 10000.0)

    def step(rows, size=1.0):
        """rows: (request, position) or the slot of a row that goes nowhere."""
        slots = [r if isinstance(r, int) else slot(*r) for r in rows]
        x = (size * rng.standard_normal((len(rows), heads + 2 * kv_heads, width))).astype(np.float32)
        angles = angles_of(np.array([0 if isinstance(r, int) else r[1] for r in rows]), frequencies,
                           1.0).astype(np.float32)
        got = run_store(env, dev, cache, slots, x, heads, rotated, halves, angles, shift, pad)
        if got is not None:
            want = rotate(x[:, :heads], angles, halves).reshape(len(rows), -1)
            assert np.all(np.abs(got[:, :want.shape[1]] - want) <= np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -149)
            assert np.all(got[:, want.shape[1]:] == 9.0)
        cache.check()

    n0, n1 = 2 * page_tokens + 5, page_tokens - 1
    step([-1] + [(0, p) for p in range(n0)] + [pages * page_tokens, 2**31 - 1, -2**31] + [(1, p) for p in range(n1)])
    step([(0, n0), (1, n1)], 0.2)
    step([(1, n1 + 1)], 50.0)
    step([(1, 3), (0, 9), (0, 8), (1, 2)])
    back = [(0, p) for p in range(17)]
    rng.shuffle(back)
    step(back, 1e-3)
    step([(0, p) for p in range(5, 29)])


@pytest.mark.parametrize("width,rotated,halves,shift,pad", [(64, 64, False, 0, 0), (128, 64, True, 0, 4),
                                                            (256, 38, True, 4, 1), (512, 512, False, 8, 0)])
def test_store_in_place(env, dev, width, rotated, halves, shift, pad):
    """q rotated where it is, beside the k and v of the same rows, which stay; rows that go nowhere are rotated too."""
    rt, kern, stream = env
    rng = np.random.default_rng(width)
    heads, kv_heads, count = 5, 2, 90
    cache = DeviceCache4(env, dev, 4, 32, kv_heads, width, rng)
    n = (heads + 2 * kv_heads) * width
    rows = rng.standard_normal((count, n + pad)).astype(np.float32)
    x = rows[:, :n].reshape(count, -1, width)
    slots = rng.permutation(4 * 32)[:count].astype(np.int32)
    slots[[3, 50, count - 1]] = -1
    angles = angles_of(np.arange(count), env[1].rope_frequencies(rotated, 10000.0)[0], 1.0).astype(np.float32)
    src = dev.put(rows, shift)
    kern.kv4_store(cache.arg, dev.put(slots), count, src + 4 * heads * width, n + pad, src + 4 * (heads + kv_heads) * width,
                   n + pad, dev.put(angles), rotated, int(halves), src, n + pad, src, n + pad, heads, stream)
    rt.sync(stream)
    got = dev.get(src, rows)
    assert np.array_equal(got[:, heads * width:], rows[:, heads * width:])
    want = rotate(x[:, :heads], angles, halves).reshape(count, -1)
    assert np.all(np.abs(got[:, :heads * width] - want) <= np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -149)
    store(cache.k, cache.v, slots, rotate(x[:, heads:heads + kv_heads], angles, halves).astype(np.float32),
          x[:, heads + kv_heads:])
    cache.check()


def test_store_values(env, dev):
    """Extremes that tie, quotients next to and on borders, steps at both ends, blocks of zeros, what is not finite."""
    rng = np.random.default_rng(3)
    cache = DeviceCache4(env, dev, 4, 32, 2, 64, rng)
    x = rng.standard_normal((24, 4, 64)).astype(np.float32)
    x[0, :, 5], x[0, :, 3] = 4, -4                         # the negative one
    x[1] = np.arange(64, dtype=np.float32) / 4 - 8          # quotients on every border
    x[1, 1:] = -x[1, 1:]
    x[2] = np.nextafter(x[1], np.float32(9))
    x[3] = np.nextafter(x[1], np.float32(-9))
    x[4] = 0
    x[5, :, :32] = -0.0
    x[6] *= np.float32(2.0 ** -20)                          # steps below fp16's normal numbers
    x[7] *= np.float32(2.0 ** -22)
    x[8] *= np.float32(1e-40)
    x[9] *= np.float32(20000)
    x[10] *= np.float32(3e37)
    x[11, 1, 3] = np.inf
    x[12, 2, 60] = -np.inf
    x[13, 3, 0] = np.nan
    x[14, 0] = np.nan
    for i in range(15, 20):                                  # largest magnitudes on borders of the step's rounding
        x[i, :, 7] = 8 * (128 + 0.5 * (i - 14)) / 256
        x[i] = np.clip(x[i], -x[i, :, 7:8], x[i, :, 7:8])
    x[20, :, 40] = 65280
    x[21, :, 40] = 65408
    x[22, :, 40] = -65407.99
    slots = rng.permutation(4 * 32)[:24]
    run_store(env, dev, cache, slots, x, 0, 0, False, None)
    cache.check()
    # Stored anew the marks are gone.
    run_store(env, dev, cache, slots[11:15], np.clip(x[:4], -9, 9), 0, 0, False, None)
    cache.check()


def run_load(env, dev, cache, slots, shift=0, pad=0, together=False):
    rt, kern, stream = env
    count, n = len(slots), cache.kv_heads * cache.width
    both = np.full((2, count, n + pad), 3.5, np.float32)
    if together:   # k | v in common rows
        both = np.full((1, count, 2 * n + pad), 3.5, np.float32)
    at = dev.put(both, shift)
    stride = both.shape[2]
    to_v = at + 4 * n if together else at + 4 * count * stride
    kern.kv4_load(cache.arg, dev.put(np.asarray(slots, np.int32)), count, at, stride, to_v, stride, stream)
    rt.sync(stream)
    got = dev.get(at, both)
    assert np.all(got[..., (2 if together else 1) * n:] == 3.5)
    return (got[0, :, :n], got[0, :, n:2 * n]) if together else (got[0, :, :n], got[1, :, :n])


@pytest.mark.parametrize("page_tokens,kv_heads,width,shift,pad,together", [
    (16, 2, 64, 0, 0, False), (64, 3, 128, 0, 4, True), (128, 1, 256, 4, 0, False), (32, 2, 512, 0, 3, True),
    (16, 5, 64, 8, 1, False), (64, 8, 128, 0, 0, False),
])
def test_load(env, dev, page_tokens, kv_heads, width, shift, pad, together):
    rng = np.random.default_rng(width)
    cache = DeviceCache4(env, dev, 9, page_tokens, kv_heads, width, rng)
    total = 9 * page_tokens
    x = rng.standard_normal((60, 2 * kv_heads, width)).astype(np.float32)
    x[7, 0, 5], x[9, 2 * kv_heads - 1, 6] = np.inf, np.nan
    slots = rng.permutation(total)[:60]
    run_store(env, dev, cache, slots, x, 0, 0, False, None)
    keys, values = held(cache.k, cache.v)
    asked = np.concatenate([slots, [-1, total, slots[3], slots[3], -2**31, 2**31 - 1]])
    k, v = run_load(env, dev, cache, asked, shift, pad, together)
    for got, want in ((k, keys), (v, values)):
        for i, s in enumerate(asked):
            row = np.full(kv_heads * width, 3.5) if not 0 <= s < total else want[s // page_tokens, :, s % page_tokens]
            assert np.array_equal(got[i].astype(np.float64), row.ravel(), equal_nan=True), i


# ---- attention ------------------------------------------------------------

def make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, seed, spread=True):
    """A cache with rows in every position that a request holds, garbage in all others, and a batch."""
    rng = np.random.default_rng(seed)
    need = [-(-max(n, 0) // page_tokens) for n in lengths]
    pages, stride = sum(need) + 3, max(max(need), 1) + 1
    order = rng.permutation(pages)
    table, taken = np.full((len(lengths), stride), -1, np.int32), 0
    cache = DeviceCache4(env, dev, pages, page_tokens, kv_heads, width, rng)
    size = np.exp(0.5 * rng.standard_normal((kv_heads, 1, width))) if spread else 1.0
    for r, n in enumerate(need):
        table[r, :n] = order[taken:taken + n]
        taken += n
        if n:
            p = np.arange(lengths[r])
            at = (table[r, p // page_tokens], slice(None), p % page_tokens)
            for c in (cache.k, cache.v):
                x = rng.standard_normal((len(p), kv_heads, 1, width)) * size
                # Codes and steps as rows of this kind have them.
                d = np.abs(x.reshape(len(p), kv_heads, -1, 32)).max(3) / 8 * rng.choice([-1, 1], (1, kv_heads, width // 32))
                d = (d.astype(np.float16).view(np.uint16) & 0xFFF8).view(np.float16)   # 8 bits
                c.steps[at] = d
                c.codes[at] = np.clip(np.rint(x[:, :, 0] / np.repeat(d.astype(float), 32, 2)) + 8, 0, 15)
    cache.put()
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rng.standard_normal((int(starts[-1]) + 2, heads, width)).astype(np.float32)
    return cache, q, starts, table


def run_attention(env, dev, cache, q, starts, lengths, table, window=0, scale=None, workspace=None, longest=None,
                  most=None, count=None, q_pad=0, out_pad=0, shift=0):
    rt, kern, stream = env
    rows, heads, width = q.shape
    count = rows if count is None else count
    n = heads * width
    scale = width ** -0.5 if scale is None else scale
    counts = np.diff(starts.astype(np.int64))
    most = max(1, int(counts.max())) if most is None else most
    longest = max(1, int(np.max(lengths))) if longest is None else longest
    wide = np.zeros((rows, n + q_pad), np.float32)
    wide[:, :n] = q.reshape(rows, n)
    out = np.full((rows, n + out_pad), 0.25, np.float32)
    po = dev.put(out, shift)
    size = kern.kv4_attention_bytes(cache.arg, count, len(lengths), most, longest, heads, window)
    size = size if workspace is None else min(workspace, size)
    # Whatever the scratch held before.
    scratch = dev.put(np.full(size, 0xFF, np.uint8)) if size else 0
    kern.kv4_attention(cache.arg, dev.put(wide, shift), n + q_pad, po, n + out_pad, count, dev.put(starts),
                       dev.put(np.asarray(lengths, np.int32)), dev.put(table), table.shape[1], len(lengths), most,
                       longest, heads, window, scale, scratch, size, stream)
    rt.sync(stream)
    got = dev.get(po, out)
    assert np.all(got[:, n:] == 0.25)
    return got[:, :n].reshape(rows, heads, width)


def check_attention(cache, q, got, starts, lengths, table, window=0, scale=None, count=None):
    rows, heads, width = q.shape
    count = rows if count is None else count
    scale = width ** -0.5 if scale is None else scale
    keys, values = held(cache.k, cache.v)
    want, weight, top = attention(q, np.full(q.shape, 0.25), keys, values, starts, lengths, table, cache.pages,
                                  cache.page_tokens, window, np.float32(scale), count)
    bound = attention_bound(weight, top, width, max(1, int(np.max(lengths))))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.where(np.isnan(want), 0, np.abs(got - want)).max(2)
    bound = np.where(np.isnan(want).any(2), 0, bound)
    assert np.all(off <= bound), (off / np.maximum(bound, 1e-30)).max()


SHAPES = [(4, 2, 64), (8, 1, 64), (32, 8, 128), (5, 5, 128), (6, 2, 256), (16, 1, 128), (4, 2, 512), (20, 4, 128),
          (24, 1, 64)]


@pytest.mark.parametrize("heads,kv_heads,width", SHAPES)
@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128])
def test_attention_decode(env, dev, heads, kv_heads, width, page_tokens):
    """One token per request, lengths around pages' and tiles' ends, one request without a token and one without
    positions."""
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 40]
    counts = [1] * 13 + [0]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, 1)
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)
    assert np.all(got[12] == 0) and np.all(got[13:] == 0.25)


@pytest.mark.parametrize("heads,kv_heads,width", SHAPES)
@pytest.mark.parametrize("window", [0, 70])
def test_attention_runs(env, dev, heads, kv_heads, width, window):
    """Prompts from position 0 and later, drafts and single tokens in one batch, rows before the first position."""
    lengths, counts = [33, 200, 90, 77, 130, 10], [33, 70, 5, 0, 1, 14]
    for page_tokens in (16, 64):
        cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, 2)
        got = run_attention(env, dev, cache, q, starts, lengths, table, window=window)
        check_attention(cache, q, got, starts, lengths, table, window=window)
        # Request 5's first four rows stand before position 0.
        assert np.all(got[starts[5]:starts[5] + 4] == 0)


@pytest.mark.parametrize("heads,kv_heads,width", [(80, 1, 64), (129, 1, 128), (144, 2, 128), (72, 1, 256), (96, 1, 512)])
@pytest.mark.parametrize("lengths,counts", [([300, 41, 90], [1, 1, 1]), ([300, 41, 90], [2, 0, 7]), ([150], [3])])
def test_attention_wide_groups(env, dev, heads, kv_heads, width, lengths, counts):
    """Groups of more heads than a call of few rows takes."""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 32, 9)
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)


@pytest.mark.parametrize("heads,kv_heads,width,page_tokens,length,tokens,window", [
    (8, 2, 128, 64, 9000, 1, 0), (8, 2, 128, 16, 9001, 3, 0), (4, 4, 64, 128, 5000, 1, 1000),
    (16, 1, 64, 32, 6000, 9, 0), (8, 8, 128, 64, 2500, 300, 0), (4, 2, 256, 32, 1500, 130, 500),
    (2, 1, 512, 64, 3001, 2, 0), (8, 2, 128, 32, 700, 700, 0), (4, 1, 64, 16, 1030, 515, 100),
    (8, 2, 128, 128, 1, 1, 0),
])
def test_attention_long(env, dev, heads, kv_heads, width, page_tokens, length, tokens, window):
    """Long caches, split work with its workspace, with less and with none, and the same bits twice."""
    cache, q, starts, table = make_attention(env, dev, [length], [tokens], heads, kv_heads, width, page_tokens, 3)
    first = run_attention(env, dev, cache, q, starts, [length], table, window=window)
    check_attention(cache, q, first, starts, [length], table, window=window)
    again = run_attention(env, dev, cache, q, starts, [length], table, window=window)
    assert np.array_equal(first, again)
    for workspace in (0, 16, 20000):
        got = run_attention(env, dev, cache, q, starts, [length], table, window=window, workspace=workspace)
        check_attention(cache, q, got, starts, [length], table, window=window)
    # A wrong guess of the longest request changes the split at most.
    for longest in (1, 100000):
        got = run_attention(env, dev, cache, q, starts, [length], table, window=window, longest=longest)
        check_attention(cache, q, got, starts, [length], table, window=window)


@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 128), (4, 4, 64), (2, 1, 256)])
@pytest.mark.parametrize("lengths,counts", [([150, 400, 60], [1, 2, 1]), ([150, 400, 60], [100, 33, 1]),
                                            ([60, 400, 60], [1, 300, 1])])
def test_attention_holes(env, dev, page_tokens, heads, kv_heads, width, lengths, counts):
    """Positions whose page is missing or no page are not there; a request with none left gives zeros. (What the
    missing pages' stand-in holds is garbage.)"""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, 4)
    table[0, 0], table[1, 2], table[1, 1], table[2, :] = -1, 2**31 - 1, -2**31, cache.pages
    if not (table == 0).any():
        for c in (cache.k, cache.v):
            c.steps[0] = np.float16(np.nan)
        cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)
    assert np.all(got[starts[2]:starts[3]] == 0)


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (4, 2, 512), (16, 1, 128)])
@pytest.mark.parametrize("page_tokens", [16, 128])
@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_attention_window_unstored(env, dev, heads, kv_heads, width, page_tokens, tokens):
    """Positions before every row's window were never stored (a program that goes on from a window's worth of
    positions): what memory holds there, NaN and infinity among it, does not matter."""
    lengths, counts, window = [300, 171], [tokens, 1], 75
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, 8)
    for r in range(2):
        for p in range(lengths[r] - counts[r] - window + 1):
            at = (table[r, p // page_tokens], slice(None), p % page_tokens)
            cache.k.steps[at] = np.float16(np.nan)
            cache.v.steps[at] = np.float16(np.nan if p % 2 else np.inf)
    cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table, window=window)
    check_attention(cache, q, got, starts, lengths, table, window=window)
    assert np.all(np.isfinite(got))


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (4, 2, 512)])
@pytest.mark.parametrize("tokens", [1, 4, 80])
def test_attention_values(env, dev, heads, kv_heads, width, tokens):
    """Magnitudes at the ends: tiny and huge queries, scores far apart, a zero query, NaN and infinity in one head,
    small and large steps, a position that reads as NaN seen by some of the rows only."""
    lengths, counts = [300, 300], [tokens, 1]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 32, 5)
    q[:, 1] = 0
    q[:, 2] *= 40        # one position takes everything
    q[0, 3, 7] = np.nan
    q[1, 0] *= 1e-30
    q[-3, 1] *= 1e-38
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)
    q[0, 3, 7] = np.inf
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    assert np.all(np.isnan(got[0, 3]))
    q[0, 3, 7] = 1
    # Steps of whole pages at both ends of fp16.
    for up, down in ((2.0 ** 11, 2.0 ** -19), (2.0 ** -22, 1)):
        cache.v.steps[table[0, :5]] = (cache.v.steps[table[0, :5]].astype(float) * up).astype(np.float16)
        cache.v.steps[table[0, 5:9]] = (cache.v.steps[table[0, 5:9]].astype(float) * down).astype(np.float16)
        cache.put()
        got = run_attention(env, dev, cache, q, starts, lengths, table)
        check_attention(cache, q, got, starts, lengths, table)
    # A position that reads as NaN, as the store marks it.
    for r, p in ((0, 290), (1, 299)):
        cache.k.steps[table[r, p // 32], 0, p % 32] = np.float16(np.nan)
        cache.v.steps[table[r, p // 32], 0, p % 32] = 0
    cache.put()
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)
    group = heads // kv_heads
    sees = np.arange(300 - tokens, 300) >= 290
    assert np.all(np.isnan(got[:tokens][sees][:, :group])) and np.all(np.isfinite(got[:tokens][~sees]))
    assert np.all(np.isnan(got[tokens, :group])) and np.all(np.isfinite(got[:, group:]))


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (2, 1, 512)])
@pytest.mark.parametrize("lengths,counts", [([200, 70], [1, 1]), ([260, 70], [90, 1])])
@pytest.mark.parametrize("size", [1e8, 1e20, 1e33])
def test_attention_far_scores(env, dev, heads, kv_heads, width, lengths, counts, size):
    """Scores far beyond what fp16 and the exponential hold: the largest takes everything."""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 16, 6)
    q *= np.float32(size)
    got = run_attention(env, dev, cache, q, starts, lengths, table, scale=1.0)
    keys, values = held(cache.k, cache.v)
    assert np.all(np.isfinite(got))
    for r in range(2):
        for row in range(starts[r], starts[r + 1]):
            p = lengths[r] - counts[r] + row - starts[r]
            t = np.arange(p + 1)
            page = table[r, t // 16]
            for h in range(heads):
                s = keys[page, h // (heads // kv_heads), t % 16] @ q[row, h].astype(np.float64)
                order = np.argsort(s)
                # Scores closer than their own error could weigh anything.
                if len(s) > 1 and s[order[-1]] - s[order[-2]] < 1e-4 * np.abs(s).max():
                    continue
                want = values[page[order[-1]], h // (heads // kv_heads), order[-1] % 16]
                # Weights are within a few steps of 2^15 and their own inverse.
                assert np.all(np.abs(got[row, h] - want) <= np.abs(want) * 64 * F32_HALF + 1e-30)


def test_attention_scores_beyond_fp32(env, dev):
    """Nothing but scores that fp32 does not hold: NaN, never zeros."""
    cache, q, starts, table = make_attention(env, dev, [40, 40], [1, 30], 4, 2, 64, 16, 6)
    for c in (cache.k,):
        c.codes[:], c.steps[:] = 7, np.float16(8)
    cache.put()
    for sign in (1, -1):
        q[:] = sign * 1e38
        got = run_attention(env, dev, cache, q, starts, [40, 40], table, scale=1.0)
        assert np.all(np.isnan(got[:31]))


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 3]])
@pytest.mark.parametrize("q_pad,out_pad,shift", [(4, 8, 0), (1, 3, 0), (0, 0, 4), (5, 0, 12)])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 128), (4, 2, 64), (2, 2, 512)])
def test_attention_strides(env, dev, counts, q_pad, out_pad, shift, heads, kv_heads, width):
    lengths = [100, 70, 33]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 32, 6)
    got = run_attention(env, dev, cache, q, starts, lengths, table, q_pad=q_pad, out_pad=out_pad, shift=shift)
    check_attention(cache, q, got, starts, lengths, table)


@pytest.mark.parametrize("counts,window", [([150, 1, 37], 0), ([150, 1, 37], 90)])
@pytest.mark.parametrize("q_pad,out_pad,shift", [(4, 8, 0), (1, 3, 0), (0, 0, 4), (5, 0, 12)])
@pytest.mark.parametrize("heads,kv_heads,width", [(6, 2, 256), (3, 1, 256), (12, 4, 64), (10, 2, 128)])
def test_attention_prompt_strides(env, dev, counts, window, q_pad, out_pad, shift, heads, kv_heads, width):
    """Prompts whose rows end inside a tile, at any stride and alignment, holes among their pages."""
    lengths = [250, 70, 133]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 16, 10)
    table[0, 3], table[2, 5] = -1, 2**30
    got = run_attention(env, dev, cache, q, starts, lengths, table, window=window, q_pad=q_pad, out_pad=out_pad, shift=shift)
    check_attention(cache, q, got, starts, lengths, table, window=window)


@pytest.mark.parametrize("workspace", [None, 0])
@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 64), (8, 2, 128), (4, 2, 256)])
def test_attention_prompt_rows(env, dev, heads, kv_heads, width, workspace):
    """Prompts in wide tiles, whole and in shares: a wavefront's lanes hand their rows to each other, so every row and
    element of many runs of the same call has the same bits, at a stride that stores whole pieces and at one that does not."""
    lengths, counts = [900, 165], [101, 165]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 32, 21)
    first = run_attention(env, dev, cache, q, starts, lengths, table, workspace=workspace)
    check_attention(cache, q, first, starts, lengths, table)
    for i in range(12):
        got = run_attention(env, dev, cache, q, starts, lengths, table, workspace=workspace, out_pad=i % 2)
        assert np.array_equal(first, got), i


def test_attention_rows_cut_off(env, dev):
    """starts past `count`, negative and out of order: no row outside is read or written."""
    lengths = [50, 60, 70, 80]
    cache, q, _, table = make_attention(env, dev, lengths, [5, 5, 5, 5], 4, 2, 64, 16, 7)
    starts = np.array([-3, 4, 2, 30, 2**31 - 1], np.int32)
    got = run_attention(env, dev, cache, q, starts, lengths, table, most=10, count=10)
    assert np.all(got[10:] == 0.25) and np.all(np.isfinite(got))
    keys, values = held(cache.k, cache.v)
    want, weight, top = attention(q, np.full(q.shape, 0.25), keys, values, np.array([-3, 4]), lengths[:1], table,
                                  cache.pages, 16, 0, np.float32(0.125), 10)
    assert np.all(np.abs(got[:2] - want[:2]).max(2) <= attention_bound(weight, top, 64, 80)[:2])
    starts = np.array([2**31 - 1, -2**31, -2**31, 2**31 - 1, -2**31], np.int32)
    for most in (1, 22):
        got = run_attention(env, dev, cache, q, starts, [50, 60, -80, 80], table, most=most, count=22)
        assert np.all(got[most:] == 0.25)
        assert np.all(got[:most] == 0)   # request 2: rows from 0 on, before its first position


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 128), (4, 4, 64), (6, 2, 256), (4, 2, 512), (40, 1, 64),
                                                  (70, 1, 64)])
def test_attention_many_requests(env, dev, heads, kv_heads, width):
    """A batch of 150 requests, most with one token, prompts among them (the 1st, 64th, 65th and last too), some with
    nothing."""
    rng = np.random.default_rng(12)
    lengths, counts = rng.integers(1, 60, 150), np.ones(150, int)
    for r, n in ((0, 40), (63, 150), (64, 17), (70, 90), (128, 33), (149, 130)):
        counts[r], lengths[r] = n, n + int(rng.integers(0, 40))
    counts[[1, 65, 100]] = 0
    cache, q, starts, table = make_attention(env, dev, lengths.tolist(), counts.tolist(), heads, kv_heads, width, 32, 13)
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 128), (8, 2, 64), (2, 2, 256), (4, 1, 512)])
def test_attention_mixed_split(env, dev, heads, kv_heads, width):
    """A prompt, a single token and drafts over long caches in one batch: work split with its workspace, with parts of
    it and with none; the same bits twice."""
    lengths, counts = [3000, 1500, 40, 2200], [100, 1, 30, 3]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 64, 14)
    size = env[1].kv4_attention_bytes(cache.arg, len(q), 4, 100, 3000, heads, 0)
    first = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, first, starts, lengths, table)
    assert np.array_equal(first, run_attention(env, dev, cache, q, starts, lengths, table))
    for workspace in (size // 2 & ~15, size // 5 & ~15, 0):
        got = run_attention(env, dev, cache, q, starts, lengths, table, workspace=workspace)
        check_attention(cache, q, got, starts, lengths, table)


@pytest.mark.parametrize("heads,kv_heads,width,tokens", [(8, 8, 64, [1]), (32, 4, 64, [3, 1, 0, 2]), (8, 8, 128, [1]),
                                                        (8, 8, 64, [40, 1, 90, 1])])
def test_attention_ragged_split(env, dev, heads, kv_heads, width, tokens):
    """Many requests of very unequal lengths, as a batch that expects long ones splits them; with less workspace."""
    rng = np.random.default_rng(15)
    n = 64 if tokens[0] == 3 else 40
    lengths = rng.integers(1, 3000, n)
    lengths[[3, 7]] = 0, 1
    counts = np.where(np.arange(n) < 2 * len(tokens), np.resize(tokens, n), 1)
    counts = np.minimum(counts, np.maximum(lengths, 1))
    cache, q, starts, table = make_attention(env, dev, lengths.tolist(), counts.tolist(), heads, kv_heads, width, 32, 16)
    size = env[1].kv4_attention_bytes(cache.arg, len(q), n, int(counts.max()), 9000, heads, 0)
    for workspace in (size, size // 2 & ~15):
        got = run_attention(env, dev, cache, q, starts, lengths, table, longest=9000, workspace=workspace)
        check_attention(cache, q, got, starts, lengths, table)


@pytest.mark.parametrize("heads,kv_heads,width", [(8, 2, 128), (4, 2, 64), (4, 2, 256), (2, 1, 512)])
@pytest.mark.parametrize("counts", [[1, 1], [150, 3]])
def test_attention_common_rows(env, dev, heads, kv_heads, width, counts):
    """q and out as columns of the same rows, with others between them that stay."""
    rt, kern, stream = env
    lengths = [300, 171]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, heads, kv_heads, width, 32, 17)
    n, gap, rows = heads * width, 8, len(q)
    both = np.full((rows, 2 * n + gap), 0.25, np.float32)
    both[:, n + gap:] = q.reshape(rows, n)
    at = dev.put(both)
    size = kern.kv4_attention_bytes(cache.arg, rows, 2, max(counts), 300, heads, 0)
    scratch = dev.put(np.full(max(size, 16), 0xFF, np.uint8))
    kern.kv4_attention(cache.arg, at + 4 * (n + gap), 2 * n + gap, at, 2 * n + gap, rows, dev.put(starts),
                       dev.put(np.array(lengths, np.int32)), dev.put(table), table.shape[1], 2, max(counts), 300, heads, 0,
                       width ** -0.5, scratch, size, stream)
    rt.sync(stream)
    got = dev.get(at, both)
    assert np.array_equal(got[:, n:], both[:, n:])
    check_attention(cache, q, got[:, :n].reshape(rows, heads, width), starts, lengths, table)


def test_attention_scales(env, dev):
    """A scale of 0, a negative one and a large one."""
    lengths, counts = [100, 64], [20, 1]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, 4, 2, 64, 16, 8)
    for scale in (0.0, -0.125, 3.0):
        got = run_attention(env, dev, cache, q, starts, lengths, table, scale=scale)
        check_attention(cache, q, got, starts, lengths, table, scale=scale)


@pytest.mark.parametrize("tokens", [3, 150])
def test_far_pages(env, dev, tokens):
    """Pages past 2^32 bytes into the code arrays: attention, a store and a load."""
    rt, kern, stream = env
    pages, page_tokens, kv_heads, width = 70000, 128, 8, 128    # 4.6 GB each
    lengths, counts = [300], [tokens]
    small, q, starts, table = make_attention(env, dev, lengths, counts, 16, kv_heads, width, page_tokens, 9)
    codes, steps = kern.kv4_bytes(pages, page_tokens, kv_heads, width)
    at = [rt.malloc(n) for n in (codes, codes, steps, steps)]
    dev.ptrs += at
    far = np.array([[69999, 3, 66999, -1]], np.int32)
    for (c, codes_at, steps_at) in ((small.k, at[0], at[2]), (small.v, at[1], at[3])):
        packed = [x.reshape(c.codes.shape[0], -1) for x in (c.packed(), c.packed_steps())]
        for j in range(3):
            for x, to in zip(packed, (codes_at, steps_at)):
                rt.upload(to + int(far[0, j]) * x[0].nbytes, x[table[0, j]])
    big = DeviceCache4.__new__(DeviceCache4)
    big.arg = Kv4(*at, pages, page_tokens, kv_heads, width)
    big.kv_heads, big.width = kv_heads, width
    got = run_attention(env, dev, big, q, starts, lengths, far)
    check_attention(small, q, got, starts, lengths, table)
    x = np.random.default_rng(1).standard_normal((1, 2 * kv_heads, width)).astype(np.float32)
    slot, n = np.array([69999 * page_tokens + 77], np.int32), kv_heads * width
    src = dev.put(x)
    kern.kv4_store(big.arg, dev.put(slot), 1, src, 2 * n, src + 4 * n, 2 * n, 0, 0, 0, 0, 0, 0, 0, 0, stream)
    k, v = run_load(env, dev, big, slot)
    store(small.k, small.v, [77], x[:, :kv_heads], x[:, kv_heads:])
    keys, values = held(small.k, small.v)
    assert np.array_equal(k[0], keys[0, :, 77].ravel()) and np.array_equal(v[0], values[0, :, 77].ravel())


# ---- log probabilities ----------------------------------------------------

def run_logprobs(env, dev, x, mask, scale, tokens, top, pad=0, shift=0, workspace=None, stream=None, ranks=True,
                 entropies=True):
    rt, kern, default = env
    stream = default if stream is None else stream
    rows, n = x.shape
    wide = np.full((rows, n + pad), np.nan, np.float32)
    wide[:, :n] = x
    out = [np.full(rows + 1, -7, np.float32), np.full(rows + 1, -7, np.int32), np.full(rows + 1, -7, np.float32),
           np.full(rows * top + 1, -7, np.int32), np.full(rows * top + 1, -7, np.float32)]
    at = [dev.put(o) for o in out]
    size = kern.logprobs_bytes(n, rows, top)
    size = size if workspace is None else min(workspace, size)
    scratch = dev.put(np.full(size, 0xFF, np.uint8)) if size else 0
    kern.logprobs(dev.put(wide, shift), n + pad, n, rows, dev.put(mask) if mask is not None else 0, scale,
                  dev.put(np.asarray(tokens, np.int32)) if tokens is not None else 0, at[0], at[1] if ranks else 0,
                  at[2] if entropies else 0, top, at[3], at[4], scratch, size, stream)
    rt.sync(stream)
    got = [dev.get(p, o) for p, o in zip(at, out)]
    assert all(g[-1] == -7 for g in got)
    return [g[:-1] for g in got[:3]] + [g[:-1].reshape(rows, top) for g in got[3:]]


def check_logprobs(got, x, mask, scale, tokens, top):
    lp, ranks, entropy, ids, top_lp, off = logprobs(x, mask, scale, tokens, top)
    assert np.array_equal(got[1], ranks) and np.array_equal(got[3], ids)
    for g, want, more in ((got[0], lp, off[0]), (got[2], entropy, off[1]), (got[4], top_lp, off[0][:, None])):
        # (Beyond fp32 the rounding is minus infinity: 2 x 3e38.)
        with np.errstate(over="ignore"):
            rounded = want.astype(np.float32)
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isneginf(g), np.isneginf(rounded))
        fine = np.isfinite(rounded)
        with np.errstate(invalid="ignore"):
            late = np.abs(g - want) > more + np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -149
        assert not np.any(late & fine), np.abs(g - want)[late & fine][:5]


def logits_of(rows, n, seed, rounded=False):
    rng = np.random.default_rng(seed)
    x = (2.5 * rng.standard_normal((rows, n))).astype(np.float32)
    x[np.arange(rows)[:, None], rng.integers(0, n, (rows, 6))] += np.float32(7)
    if rounded:   # to 8 bits: ties
        x = ((x.view(np.uint32) + 0x8000) & 0xFFFF0000).view(np.float32)
    mask = rng.integers(0, 2**32, (n + 31) // 32, dtype=np.uint32) & rng.integers(0, 2**32, (n + 31) // 32, dtype=np.uint32)
    mask &= rng.integers(0, 2**32, (n + 31) // 32, dtype=np.uint32)
    tokens = np.where(rng.random(rows) < 0.5, x.argmax(1), rng.integers(0, n, rows))
    return x, mask, tokens


@pytest.mark.parametrize("rows,n,top,scale,rounded,pad,shift", [
    (1, 1, 1, 1.0, False, 0, 0), (3, 2, 2, 1.0, False, 0, 0), (1, 5, 64, 0.7, False, 0, 0), (2, 63, 20, 1.0, True, 1, 4),
    (5, 64, 64, 1.0, False, 0, 0), (4, 1000, 5, 1.25, True, 3, 8), (7, 1023, 64, 1.0, True, 0, 0),
    (1, 4096, 20, 1.0, False, 0, 0), (3, 4097, 33, 0.5, False, 0, 12), (2, 8191, 1, 3.0, True, 2, 0),
    (64, 32000, 20, 1.0, False, 0, 0), (1, 32000, 5, 1.0, True, 0, 0), (9, 50257, 64, 1.0, True, 0, 0),
    (300, 1537, 8, 1.0, False, 0, 4), (2, 262144, 20, 0.8, False, 0, 0), (1, 262147, 64, 1.0, True, 1, 4),
    (1500, 700, 3, 1.0, False, 0, 0), (40, 20011, 0, 1.0, False, 0, 0),
])
@pytest.mark.parametrize("masks", [False, True])
def test_logprobs(env, dev, rows, n, top, scale, rounded, pad, shift, masks):
    x, mask, tokens = logits_of(rows, n, n + rows, rounded)
    mask = mask if masks else None
    tokens[rows // 2] = [-1, n, 2**31 - 1, -2**31][rows % 4]
    first = run_logprobs(env, dev, x, mask, scale, tokens, top, pad, shift)
    check_logprobs(first, x, mask, scale, tokens, top)
    again = run_logprobs(env, dev, x, mask, scale, tokens, top, pad, shift)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(first, again))
    for workspace in (0, env[1].logprobs_bytes(n, rows, top) // 3 & ~15):
        got = run_logprobs(env, dev, x, mask, scale, tokens, top, pad, shift, workspace=workspace)
        check_logprobs(got, x, mask, scale, tokens, top)


@pytest.mark.parametrize("n", [40, 3001, 40000])
@pytest.mark.parametrize("rows", [1, 24])
def test_logprobs_rows(env, dev, rows, n):
    """Rows that are all the same, sorted either way, zeros of both signs, minus infinity, one token, NaN and infinity,
    masked or not, magnitudes at the ends."""
    x, mask, tokens = logits_of(24, n, 5)
    keep = 1 - (mask[np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32) & 1)
    off, on = np.flatnonzero(keep == 0)[0], np.flatnonzero(keep)
    x[0] = 3.5
    x[1] = np.sort(x[1])
    x[2] = np.sort(x[2])[::-1]
    x[3] = np.where(np.arange(n) % 3, 0.0, -0.0)
    x[4, ::2] = -np.inf
    x[5] = -np.inf
    x[6] = -np.inf
    x[6, on[-1]] = 2.0
    x[7, on[3]] = np.nan
    x[8, on[4]] = np.inf
    x[9, off], x[10, off] = np.nan, np.inf
    x[11] *= np.float32(1e30)
    x[12] = np.where(np.arange(n) % 2, np.float32(3e38), np.float32(-3e38))
    x[13] *= np.float32(1e-30)
    x[14] = np.where(keep, -np.inf, x[14])       # nothing but masked entries
    x[15, on[2]] = 200.0                          # one token takes everything
    x[16] = np.sort(x[16])
    x[16, 1:] = x[16, :-1]
    x[17, :n // 2] = 5.0                          # many of the largest
    x[18] = np.tile(np.array([1, 2, 3, 4], np.float32), n // 4 + 1)[:n]
    tokens[4], tokens[6], tokens[17], tokens[0] = 0, on[0], n // 2 - 1, n - 1
    tokens[9], tokens[11] = off, x[11].argmax()
    pick = np.arange(24) if rows == 24 else None
    for top in (5, 64):
        for m in (None, mask):
            for part in ([pick] if rows == 24 else [[i] for i in range(0, 19, 1)]):
                got = run_logprobs(env, dev, x[part], m, 1.0, tokens[part], top)
                check_logprobs(got, x[part], m, 1.0, tokens[part], top)


@pytest.mark.parametrize("rows,n,top", [(6, 3001, 20), (3, 40000, 64), (1100, 2500, 5)])
@pytest.mark.parametrize("exponent", [-20, -11, 7, 20])
@pytest.mark.parametrize("spread", [0.01, 1.0, 40.0])
def test_logprobs_scales(env, dev, rows, n, top, exponent, spread):
    """The scales that the header allows, to both ends, on logits that they bring to nearly equal ones, to ordinary ones
    and to a few likely ones; logits of the ends of fp32 and ordinary ones under the same scale."""
    scale = 2.0 ** exponent * (1 if abs(exponent) == 20 else 1.1)
    x, mask, tokens = logits_of(rows, n, exponent + 40)
    x *= np.float32(spread / scale)
    x[rows // 2] = 2.5 * np.random.default_rng(1).standard_normal(n)
    x[rows - 1] = np.where(np.arange(n) % 3, np.float32(3e38), np.float32(-3e38))
    for m in (None, mask):
        got = run_logprobs(env, dev, x, m, scale, tokens, top)
        check_logprobs(got, x, m, scale, tokens, top)


@pytest.mark.parametrize("n,shift", [(32000, 0), (128257, 8), (262147, 4)])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_logprobs_equal(env, dev, n, shift, top):
    """Rows in which more groups of logits reach the bound than are listed: zeros (a batch's padding), few values,
    equal ones above or below the others, in the last tokens only, after larger ones that are few or many."""
    rng = np.random.default_rng(n)
    x, mask, tokens = logits_of(9, n, 7)
    x[0] = 0
    x[1] = np.where(np.arange(n) % 2, np.float32(-1), np.float32(0))
    x[2] = rng.integers(0, 3, n)
    x[3] = np.minimum(x[3], 0)
    x[4] = np.where(np.arange(n) < n - 30, np.float32(1), np.float32(2))
    x[5] = 0
    x[5, rng.permutation(n)[:7]] = 3
    x[6] = 0
    x[6, rng.permutation(n)[:700]] = rng.permutation(700) + 1
    x[7] = np.where(np.arange(n) < n // 2, -np.inf, np.float32(-3e38))
    x[8] = np.where(np.arange(n) // 16 % 64 < 9, np.float32(5), x[8] - 40)   # in the same groups of every set
    tokens[:4] = n - 1, 1, n // 2, 0
    for m in (None, mask):
        for workspace in (None, 0):
            got = run_logprobs(env, dev, x, m, 1.0, tokens, top, shift=shift, workspace=workspace)
            check_logprobs(got, x, m, 1.0, tokens, top)


@pytest.mark.parametrize("shift,workspace", [(0, None), (4, None), (0, 0)])
def test_logprobs_longest_row(env, dev, shift, workspace):
    """2^24 logits: whole numbers in a known order (ranks to the last one, exact counts), and all equal."""
    n, top = 1 << 24, 64
    order = (np.arange(n) * 0x9E3779B1 + 12345) % n            # the rank of each id (an odd factor: each once)
    first = np.empty(n, np.int64)
    first[order] = np.arange(n)
    x = np.stack([(-order).astype(np.float32), np.full(n, 2.5, np.float32)])
    for token in (int(first[-1]), int(first[0]), n - 1):
        tokens = [token, token]
        lp, ranks, entropy, ids, top_lp = run_logprobs(env, dev, x, None, 2.0 ** -20, tokens, top, shift=shift,
                                                       workspace=workspace)
        assert ranks.tolist() == [order[token], token]
        assert np.array_equal(ids[0], first[:top]) and np.array_equal(ids[1], np.arange(top))
        w = np.arange(n) * 2.0 ** -20
        p = np.exp(-w)
        lse, p = np.log(p.sum()), p / p.sum()
        # As in kv4_check.logprobs.
        chain = n / 256 + 64 + 16
        each = (p * (3 * w + 4 + chain)).sum() * F32_HALF + n * 2.0 ** -126
        assert abs(lp[0] - (-w[order[token]] - lse)) <= each + abs(lp[0]) * F32_HALF * (1 + 1e-6)
        assert abs(entropy[0] - (lse + (p * w).sum())) <= each + (p * w * (3 * w + 8 + chain)).sum() * F32_HALF + (
            p * w).sum() * each + abs(entropy[0]) * F32_HALF * (1 + 1e-6)
        # Nothing but the maximum, which is counted: the logarithm, rounded once.
        assert lp[1] == np.float32(-24 * np.log(2)) and entropy[1] == np.float32(24 * np.log(2))
        assert np.all(top_lp[1] == np.float32(-24 * np.log(2)))


def test_logprobs_padding_costs_little(env, dev):
    """Rows of zeros that pad a batch are no slower than rows of logits, but for the choice among equal ones (17 times
    as slow with every group gone through)."""
    rt, kern, stream = env
    rows, n, top = 64, 128256, 20
    x = logits_of(rows, n, 3)[0]
    size = kern.logprobs_bytes(n, rows, top)
    scratch, ids, lp = dev.put(np.zeros(size, np.uint8)), dev.put(np.zeros(rows * top, np.int32)), dev.put(
        np.zeros(rows * top, np.float32))

    def best(x):
        at, least = dev.put(x), np.inf
        for _ in range(6):
            rt.sync(stream)
            begin = time.perf_counter()
            for _ in range(50):
                kern.logprobs(at, n, n, rows, 0, 1.0, 0, 0, 0, 0, top, ids, lp, scratch, size, stream)
            rt.sync(stream)
            least = min(least, time.perf_counter() - begin)
        return least

    whole = best(x)
    x[rows // 2:] = 0
    assert best(x) < 5 * whole


def test_logprobs_parts(env, dev):
    """Some of the results only; rank 0 is the greedy choice."""
    rt, kern, stream = env
    x, mask, tokens = logits_of(5, 3000, 8)
    lp, ranks, entropy, ids, top_lp = run_logprobs(env, dev, x, mask, 1.0, tokens, 4)
    for a in (dict(ranks=False), dict(entropies=False), dict(ranks=False, entropies=False)):
        got = run_logprobs(env, dev, x, mask, 1.0, tokens, 0, **a)
        assert np.array_equal(got[0], lp)
        assert np.array_equal(got[1], ranks if a.get("ranks", True) else np.full(5, -7))
        assert np.array_equal(got[2], entropy if a.get("entropies", True) else np.full(5, -7))
    got = run_logprobs(env, dev, x, mask, 1.0, None, 4)
    assert np.array_equal(got[3], ids) and np.array_equal(got[0], np.full(5, -7)) and np.array_equal(got[2], entropy)
    best = dev.put(np.zeros(5, np.uint32))
    kern.lib.nya_hip_greedy.argtypes = [ctypes.c_size_t] * 6
    assert kern.lib.nya_hip_greedy(dev.put(x), 3000, 5, dev.put(mask), best, stream) == 0
    rt.sync(stream)
    assert np.array_equal(dev.get(best, np.zeros(5, np.uint32)), ids[:, 0].astype(np.uint32))


# ---- a step as it is used -------------------------------------------------

class Server4:
    """One layer of a server and its answers: requests that come, decode, take drafts back and finish."""

    def __init__(self, env, dev, heads=8, kv_heads=2, width=64, page_tokens=16, requests=5, max_tokens=160, pages=60,
                 vocabulary=5003, top=6):
        self.env, self.dev = env, dev
        rt, kern, _ = env
        self.rng = np.random.default_rng(11)
        self.heads, self.kv_heads, self.width, self.max_tokens = heads, kv_heads, width, max_tokens
        self.requests, self.vocabulary, self.top = requests, vocabulary, top
        self.cache = DeviceCache4(env, dev, pages, page_tokens, kv_heads, width, self.rng)
        self.state = Pages(requests, 20, pages, page_tokens, self.rng.permutation(pages))
        self.pages = DevicePages(env, dev, self.state, max_tokens)
        self.rotated = 32
        self.frequencies, _ = kern.rope_frequencies(self.rotated, 10000.0)
        self.f = dev.put(self.frequencies)
        n = (heads + 2 * kv_heads) * width
        self.x = np.zeros((max_tokens, n), np.float32)
        self.px = dev.put(self.x)
        self.pa = dev.put(np.zeros((max_tokens, self.rotated // 2, 2), np.float32))
        self.pq = dev.put(np.zeros((max_tokens, heads * width), np.float32))
        self.out = np.full((max_tokens, heads * width), 0.25, np.float32)
        self.po = dev.put(self.out)
        self.logits = np.zeros((requests, vocabulary), np.float32)
        self.tokens = np.zeros(requests, np.int32)
        self.pl, self.pt = dev.put(self.logits), dev.put(self.tokens)
        self.answers = [np.zeros(requests, np.float32), np.zeros(requests, np.int32), np.zeros(requests, np.float32),
                        np.zeros((requests, top), np.int32), np.zeros((requests, top), np.float32)]
        self.pans = [dev.put(a) for a in self.answers]
        self.size = kern.kv4_attention_bytes(self.cache.arg, max_tokens, requests, max_tokens, 320, heads, 0)
        self.size = max(self.size, kern.logprobs_bytes(vocabulary, requests, top), 16)
        self.scratch = dev.put(np.full(self.size, 0xFF, np.uint8))

    def launch(self, stream=None):
        rt, kern, default = self.env
        stream = default if stream is None else stream
        p, n, h, kvh, w = self.pages, self.x.shape[1], self.heads, self.kv_heads, self.width
        p.launch(stream)
        kern.rope_angles(p.positions, self.max_tokens, self.f, self.rotated, 1.0, self.pa, stream)
        kern.kv4_store(self.cache.arg, p.slots, self.max_tokens, self.px + 4 * h * w, n, self.px + 4 * (h + kvh) * w, n,
                       self.pa, self.rotated, 1, self.px, n, self.pq, h * w, h, stream)
        kern.kv4_attention(self.cache.arg, self.pq, h * w, self.po, h * w, self.max_tokens, p.starts, p.lengths,
                           p.table, p.stride, len(self.state.held), self.max_tokens, 320, h, 0, w ** -0.5, self.scratch,
                           self.size, stream)
        # One workspace for all of a stream's calls.
        kern.logprobs(self.pl, self.vocabulary, self.vocabulary, self.requests, 0, 1.25, self.pt, *self.pans[:3],
                      self.top, *self.pans[3:], self.scratch, self.size, stream)

    def inputs(self, lengths, counts):
        rt = self.env[0]
        self.x = self.rng.standard_normal(self.x.shape).astype(np.float32)
        self.logits, _, tokens = logits_of(self.requests, self.vocabulary, int(self.rng.integers(1 << 30)))
        self.tokens = np.where(np.asarray(counts) > 0, tokens, -1).astype(np.int32)
        for to, x in ((self.px, self.x), (self.po, self.out), (self.pl, self.logits), (self.pt, self.tokens),
                      (self.pages.lengths, np.asarray(lengths, np.int32)),
                      (self.pages.counts, np.asarray(counts, np.int32))):
            rt.upload(to, x)

    def check(self, lengths, counts):
        h, kvh, w = self.heads, self.kv_heads, self.width
        starts, positions, slots = self.state.step(lengths, counts, self.max_tokens)
        self.pages.check(starts, positions, slots)
        x = self.x.reshape(self.max_tokens, -1, w)
        angles = angles_of(positions, self.frequencies, 1.0).astype(np.float32)
        q, k = (rotate(x[:, a:b], angles, True).astype(np.float32) for a, b in ((0, h), (h, h + kvh)))
        store(self.cache.k, self.cache.v, slots, k, x[:, h + kvh:])
        self.cache.check()
        got = self.dev.get(self.po, self.out).reshape(q.shape)
        check_attention(self.cache, q, got, starts, lengths, self.state.table)
        check_logprobs([self.dev.get(p, a) for p, a in zip(self.pans, self.answers)], self.logits, None, 1.25,
                       self.tokens, self.top)


# Every position that a row sees was stored.
STORED = STEPS[:-1] + [([34, 166, 50, 60, 8], [1, 60, 1, 60, 1])]


def test_serving_steps(env, dev):
    server = Server4(env, dev)
    for lengths, counts in STORED:
        server.inputs(lengths, counts)
        server.launch()
        env[0].sync(env[2])
        server.check(lengths, counts)


def test_serving_steps_captured(env, dev):
    """The whole step captured once and replayed for every step, with eager work between, on another stream."""
    rt, kern, stream = env
    server, other = Server4(env, dev), rt.stream()
    graph = Graph(rt, other, [lambda: server.launch(other)])
    eager = Server4(env, dev)
    for lengths, counts in STORED:
        server.inputs(lengths, counts)
        graph.launch()
        eager.inputs(lengths, counts)
        eager.launch()
        rt.sync(stream)
        rt.sync(other)
        server.check(lengths, counts)
        eager.check(lengths, counts)
    graph.close()


def test_two_calls_at_once(env, dev):
    """Attention and log probabilities on two streams with workspaces of their own."""
    rt, kern, stream = env
    other = rt.stream()
    calls, answers = [], []
    for seed, s in ((21, stream), (22, other)):
        lengths = [4000]
        cache, q, starts, table = make_attention(env, dev, lengths, [1], 8, 2, 128, 64, seed)
        size = kern.kv4_attention_bytes(cache.arg, 1, 1, 1, 4000, 8, 0)
        out = dev.put(np.zeros(q.shape, np.float32))
        args = (cache.arg, dev.put(q), 1024, out, 1024, 1, dev.put(starts), dev.put(np.array(lengths, np.int32)),
                dev.put(table), table.shape[1], 1, 1, 4000, 8, 0, 128 ** -0.5, dev.put(np.zeros(max(size, 16), np.uint8)),
                size, s)
        calls.append((cache, q, starts, table, lengths, out, args))
        x, _, tokens = logits_of(3, 40000, seed)
        size = kern.logprobs_bytes(40000, 3, 5)
        parts = [dev.put(np.zeros(n, np.float32)) for n in (3, 3, 3, 15, 15)]
        answers.append((x, tokens, parts, (dev.put(x), 40000, 40000, 3, 0, 1.0, dev.put(tokens.astype(np.int32)),
                                           *parts[:3], 5, *parts[3:], dev.put(np.zeros(max(size, 16), np.uint8)), size,
                                           s)))
    for _ in range(20):
        for c, a in zip(calls, answers):
            kern.kv4_attention(*c[-1])
            kern.logprobs(*a[-1])
    rt.sync(stream)
    rt.sync(other)
    for (cache, q, starts, table, lengths, out, _), (x, tokens, parts, _) in zip(calls, answers):
        got = dev.get(out, q)
        check_attention(cache, q[:1], got[:1], starts, lengths, table)
        got = [dev.get(p, np.empty(n, t)) for p, n, t in zip(parts, (3, 3, 3, 15, 15), "fifif")]
        check_logprobs(got[:3] + [g.reshape(3, 5) for g in got[3:]], x, None, 1.0, tokens, 5)
