"""The serving operators (include/fyodor_hip_serving.h) on an MI355X against
their statements in serving_check.py, at the sizes and data where they can go
wrong. Whole numbers (tables, slots, codes) and scales are exact; rotated rows
are one rounding from 64 bits; attention stays in the bound that
attention_bound derives."""
import numpy as np
import pytest

from fyodor_amd.hip import Graph, Kernels, Kv8, Runtime
from serving_check import Cache, Dev, F32_HALF, Pages, angles_of, attention, attention_bound, rotate

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


# ---- pages ----------------------------------------------------------------

class DevicePages:
    """The device side of a Pages statement."""

    def __init__(self, env, dev, state, max_tokens):
        self.env, self.dev, self.state, self.max_tokens = env, dev, state, max_tokens
        requests, self.stride = state.table.shape
        self.table, self.held = dev.put(state.table), dev.put(state.held)
        self.free_pages, self.free_count = dev.put(state.free_pages), dev.put(state.free_count)
        self.starts = dev.put(np.full(requests + 1, -7, np.int32))
        self.positions, self.slots = (dev.put(np.full(max_tokens + 1, -7, np.int32)) for _ in range(2))
        self.lengths, self.counts = (dev.put(np.zeros(requests, np.int32)) for _ in range(2))

    def step(self, lengths, counts):
        rt, kern, stream = self.env
        rt.upload(self.lengths, np.asarray(lengths, np.int32))
        rt.upload(self.counts, np.asarray(counts, np.int32))
        self.launch(stream)
        rt.sync(stream)

    def launch(self, stream):
        s = self.state
        self.env[1].page_step(self.lengths, self.counts, len(s.held), s.page_tokens, self.table, self.stride, self.held,
                              self.free_pages, s.pages, self.free_count, self.starts, self.positions, self.slots,
                              self.max_tokens, stream)

    def check(self, starts, positions, slots):
        s, get = self.state, self.dev.get
        assert np.array_equal(get(self.free_count, s.free_count), s.free_count)
        assert np.array_equal(get(self.held, s.held), s.held)
        assert np.array_equal(get(self.table, s.table), s.table)
        assert np.array_equal(get(self.free_pages, s.free_pages), s.free_pages)
        assert np.array_equal(get(self.starts, starts), starts)
        for p, want in ((self.positions, positions), (self.slots, slots)):
            got = get(p, np.empty(self.max_tokens + 1, np.int32))
            assert np.array_equal(got[:-1], want) and got[-1] == -7


@pytest.mark.parametrize("requests,size,stride,pages,max_tokens", [
    (1, 16, 1, 1, 1), (1, 128, 5, 5, 640), (5, 32, 9, 30, 77), (64, 64, 20, 700, 300), (64, 16, 300, 9000, 5000),
    (300, 16, 40, 6000, 2049), (1024, 32, 6, 4000, 1200), (1025, 16, 7, 3000, 2500), (2500, 64, 5, 8000, 20000),
])
def test_page_step(env, dev, requests, size, stride, pages, max_tokens):
    rng = np.random.default_rng(requests + size)
    state = Pages(requests, stride, pages, size, rng.permutation(pages))
    device = DevicePages(env, dev, state, max_tokens)
    full = stride * size
    per = max(1, 2 * max_tokens // requests)
    for step in range(7):
        # Growth, shrinking, finished requests, too little memory, lengths
        # beyond the table, nothing at all, more rows than fit.
        lengths = rng.integers(0, full + 1, requests)
        if step == 1:
            lengths[:] = full
        if step == 2:
            lengths[::2] = 0
        if step == 3:
            lengths[-1] = full + 1
            lengths[rng.integers(requests)] = 2**31 - 1
            lengths[rng.integers(requests)] = -5
        if step == 4:
            lengths[:] = 0
        counts = np.minimum(rng.integers(0, per + 1, requests), np.maximum(lengths, 0))
        if step == 5:
            counts[rng.integers(requests)] = -3
            counts[rng.integers(requests)] += 2     # more than it holds
        if step == 6:
            counts[:] = 1
        want = state.step(lengths, counts, max_tokens)
        device.step(lengths, counts)
        device.check(*want)
        # Again: nothing changes.
        if step in (0, 6):
            device.step(lengths, counts)
            device.check(*want)


def test_page_step_skips_bad_pages(env, dev):
    """Entries that are no pages give no slots, and a stack count past its room is cut off."""
    rt = env[0]
    state = Pages(2, 4, 8, 16, np.arange(8))
    state.table[:] = [[3, -9, 99, -1], [7, 2, -1, -1]]
    state.held[:] = [3, 2]
    state.free_count[0] = 0
    device = DevicePages(env, dev, state, 90)
    device.step([48, 20], [48, 20])
    slots = dev.get(device.slots, np.empty(90, np.int32))
    want = np.concatenate([3 * 16 + np.arange(16), np.full(32, -1), 7 * 16 + np.arange(16), 2 * 16 + np.arange(4),
                           np.full(22, -1)])
    assert np.array_equal(slots, want)
    # held and free_count out of range.
    rt.upload(device.held, np.array([50, -2], np.int32))
    rt.upload(device.free_count, np.array([1000, 0], np.int32))
    device.step([64, 0], [1, 0])
    assert np.array_equal(dev.get(device.free_count, state.free_count), [8, 0])


# ---- rotary positions -----------------------------------------------------

@pytest.mark.parametrize("count,rotated,magnitude", [(1, 2, 1.0), (7, 64, 1.0), (33, 128, 1.3), (1000, 512, 0.7),
                                                     (3, 1024, 1.0)])
def test_rope_angles(env, dev, count, rotated, magnitude):
    rt, kern, stream = env
    rng = np.random.default_rng(count)
    positions = rng.integers(0, 1 << rng.integers(1, 31), count).astype(np.int32)
    positions[:3] = [0, 2**31 - 1, 1 << 20][:count]
    frequencies, _ = kern.rope_frequencies(rotated, 500000.0)
    angles = dev.put(np.zeros((count, rotated // 2, 2), np.float32))
    kern.rope_angles(dev.put(positions), count, dev.put(frequencies), rotated, magnitude, angles, stream)
    rt.sync(stream)
    want = angles_of(positions, frequencies, np.float32(magnitude))
    got = dev.get(angles, np.empty_like(want, np.float32))
    # One rounding to fp32; in 64 bits the phase (up to 2^31) is off by 2^31 2^-53 a few times, both here and there.
    assert np.all(np.abs(got - want) <= np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -19 * (positions.max() > 2**24)
                  + 2.0 ** -27 * (positions.max() <= 2**24))


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("count,heads,kv_heads,width,rotated,pad,shift", [
    (1, 1, 0, 2, 2, 0, 0), (3, 4, 2, 64, 64, 0, 0), (5, 32, 8, 128, 128, 0, 0), (2, 16, 8, 256, 64, 4, 0),
    (9, 6, 2, 80, 40, 0, 0), (4, 3, 1, 96, 34, 1, 4), (17, 8, 1, 512, 128, 8, 0), (3, 5, 5, 66, 22, 0, 8),
    (300, 4, 4, 64, 32, 0, 0), (2, 2, 2, 1030, 1024, 2, 0),
])
def test_rope(env, dev, halves, count, heads, kv_heads, width, rotated, pad, shift):
    """Both layouts, parts of a head, odd widths, padded and unaligned rows, in place and elsewhere."""
    rt, kern, stream = env
    rng = np.random.default_rng(width + count)
    frequencies, _ = kern.rope_frequencies(rotated, 10000.0)
    angles = angles_of(rng.integers(0, 5000, count), frequencies, 1.0).astype(np.float32)
    a = dev.put(angles)
    for in_place in (False, True):
        # One row of q | k per token.
        stride = (heads + kv_heads) * width + pad
        x = rng.standard_normal((count, stride), np.float32)
        src = dev.put(x, shift)
        out = src if in_place else dev.put(np.full((count, stride), 7.0, np.float32), shift)
        k = src + 4 * heads * width if kv_heads else 0
        kern.rope(src, stride, out, stride, heads, k, stride, out + 4 * heads * width if kv_heads else 0, stride,
                  kv_heads, width, count, a, rotated, int(halves), stream)
        rt.sync(stream)
        got = dev.get(out, x)
        n = (heads + kv_heads) * width
        want = rotate(x[:, :n].reshape(count, -1, width), angles, halves).reshape(count, -1)
        # One rounding of what 64 bits give.
        assert np.all(np.abs(got[:, :n] - want) <= np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -149)
        assert np.array_equal(got[:, n:], x[:, n:] if in_place else np.full((count, pad), 7.0, np.float32))
        kept = got[:, :n].reshape(count, -1, width)[..., rotated:]
        assert np.array_equal(kept, x[:, :n].reshape(count, -1, width)[..., rotated:])
        if not in_place:
            assert np.array_equal(dev.get(src, x), x)


# ---- the 8-bit cache ------------------------------------------------------

class DeviceCache:
    def __init__(self, env, dev, pages, page_tokens, kv_heads, width, rng):
        self.env, self.dev = env, dev
        self.k, self.v = (Cache(pages, page_tokens, kv_heads, width, rng, kind) for kind in "kv")
        self.pages, self.page_tokens, self.kv_heads, self.width = pages, page_tokens, kv_heads, width
        self.put()

    def put(self):
        """The statement's codes and scales on the device."""
        self.at = [self.dev.put(x) for x in (self.k.packed(), self.v.packed(), self.k.scales, self.v.scales)]
        self.arg = Kv8(*self.at, self.pages, self.page_tokens, self.kv_heads, self.width)

    def check(self):
        for c, codes, scales in ((self.k, self.at[0], self.at[2]), (self.v, self.at[1], self.at[3])):
            got = self.dev.get(scales, c.scales)
            assert np.array_equal(got, c.scales, equal_nan=True)
            got = c.unpack(self.dev.get(codes, np.empty(c.codes.size, np.int8)))
            fine = np.isfinite(c.scales) & c.known
            bad = np.argwhere((got != c.codes) & fine[..., None, None])
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
    kern.kv8_store(cache.arg, dev.put(np.asarray(slots, np.int32)), count, src + 4 * heads * width, n + pad,
                   src + 4 * (heads + kvh) * width, n + pad, dev.put(angles) if rotated else 0, rotated, int(halves),
                   src if q_out else 0, n + pad, q_out, heads * width + pad, heads, stream)
    rt.sync(stream)
    k = x[:, heads:heads + kvh]
    if rotated:
        k = rotate(k, angles, halves).astype(np.float32)
    cache.k.store(slots, k)
    cache.v.store(slots, x[:, heads + kvh:])
    assert np.array_equal(dev.get(src, rows), rows, equal_nan=True)
    return dev.get(q_out, np.empty((count, heads * width + pad), np.float32)) if q_out else None


@pytest.mark.parametrize("page_tokens,kv_heads,width,heads,rotated,halves,shift,pad", [
    (16, 2, 64, 4, 64, False, 0, 0), (32, 1, 64, 0, 0, False, 0, 0), (64, 3, 128, 3, 64, True, 0, 0),
    (128, 8, 128, 8, 128, False, 0, 4), (64, 2, 256, 2, 64, True, 4, 1), (16, 1, 512, 2, 512, True, 0, 0),
    (32, 2, 128, 4, 38, False, 0, 0), (32, 2, 128, 4, 38, True, 8, 2), (128, 1, 512, 0, 128, False, 0, 0),
])
def test_store(env, dev, page_tokens, kv_heads, width, heads, rotated, halves, shift, pad):
    """Prompts, tokens one by one, growing steps, positions written again, several requests in one call."""
    rng = np.random.default_rng(page_tokens + width)
    pages = 12
    cache = DeviceCache(env, dev, pages, page_tokens, kv_heads, width, rng)
    order = rng.permutation(pages)
    slot = lambda request, p: int(order[4 * request + p // page_tokens]) * page_tokens + p % page_tokens
    frequencies, _ = env[1].rope_frequencies(max(rotated, 2), 10000.0)

    def step(rows, size=1.0):
        """rows: (request, position) or None for a row that goes nowhere."""
        slots = [-1 if r is None else slot(*r) for r in rows]
        x = (size * rng.standard_normal((len(rows), heads + 2 * kv_heads, width))).astype(np.float32)
        angles = angles_of(np.array([r[1] if r else 0 for r in rows]), frequencies, 1.0).astype(np.float32)
        got = run_store(env, dev, cache, slots, x, heads, rotated, halves, angles, shift, pad)
        if got is not None:
            want = rotate(x[:, :heads], angles, halves).reshape(len(rows), -1)
            assert np.all(np.abs(got[:, :want.shape[1]] - want) <= np.abs(want) * F32_HALF * (1 + 1e-6) + 2.0 ** -149)
            assert np.all(got[:, want.shape[1]:] == 9.0)
        cache.check()

    # Two prompts, one ending inside a page, with rows that go nowhere around.
    n0, n1 = 2 * page_tokens + 5, page_tokens - 1
    step([None] + [(0, p) for p in range(n0)] + [None, None] + [(1, p) for p in range(n1)] + [None])
    # One token each: small (nothing changes but its codes), then large (the page's codes are rounded again).
    step([(0, n0), (1, n1)], 0.2)
    step([(0, n0 + 1), (1, n1 + 1), (2, 0)], 5.0)
    step([(0, n0 + 2), None, (2, 1)], 40.0)
    # Drafts that cross a page's end, then the rejected ones written again.
    step([(2, p) for p in range(2, page_tokens + 3)])
    step([(2, p) for p in range(page_tokens - 2, page_tokens + 1)], 0.5)
    # A page begun anew by another request's first position.
    step([(1, 0)], 1e-3)


def test_store_values(env, dev):
    """Zeros, subnormals, the largest floats, ties, infinities and NaN, and what a page does after them."""
    rng = np.random.default_rng(3)
    cache = DeviceCache(env, dev, 4, 16, 8, 64, rng)
    angles = np.zeros((16, 32, 2), np.float32)
    x = np.zeros((16, 16, 64), np.float32)
    x[:, 1] = 1e-42 * rng.standard_normal((16, 64))
    x[:, 2] = np.finfo(np.float32).max * rng.uniform(-1, 1, (16, 64))
    x[:, 3] = rng.integers(-254, 255, (16, 64)) / 2       # every half step
    x[0, 3, 0] = 127
    x[:, 4] = rng.standard_normal((16, 64))
    x[3, 4, 5] = np.inf
    x[:, 5] = rng.standard_normal((16, 64))
    x[3, 5, 5] = np.nan
    x[:, 6] = 2.0 ** -99 * rng.standard_normal((16, 64))
    x[:, 7] = rng.standard_normal((16, 64)) * 10.0 ** rng.uniform(-8, 8, (16, 64))
    x[:, 8:] = x[:, :8]
    run_store(env, dev, cache, np.arange(16), x, 0, 0, False, angles)
    cache.check()
    # A finite token into the same page leaves the bad heads bad; anew from the first slot mends them.
    run_store(env, dev, cache, np.array([4]), x[:1], 0, 0, False, angles[:1])
    cache.check()
    assert not np.isfinite(cache.k.scales[0, 4]) and np.isnan(cache.k.scales[0, 5])
    run_store(env, dev, cache, np.array([0]), x[:1], 0, 0, False, angles[:1])
    cache.check()
    assert np.all(np.isfinite(cache.k.scales[0]))
    x[3, 4:6] = x[3, 12:14] = 1
    run_store(env, dev, cache, np.arange(16), x, 0, 0, False, angles)
    cache.check()
    assert cache.k.known[0].all() and np.all(np.isfinite(cache.v.scales[0]))
    x[3, 4, 5], x[3, 5, 5] = np.inf, np.nan
    # NaN and infinity into a page that was fine.
    run_store(env, dev, cache, np.array([1]), x[3:4], 0, 0, False, angles[:1])
    cache.check()
    # Slots outside the cache.
    run_store(env, dev, cache, np.array([64, -1, 2**31 - 1, -2**31, 63]), x[:5], 0, 0, False, angles[:5])
    cache.check()


@pytest.mark.parametrize("n", [257, 1500])
def test_store_many_rows(env, dev, n):
    """Long runs over many pages and single tokens of many requests in one call."""
    rng = np.random.default_rng(n)
    cache = DeviceCache(env, dev, 200, 32, 2, 64, rng)
    order = rng.permutation(200)
    slots = np.concatenate([order[:n // 32 + 1, None] * 32 + np.arange(32)], 1).reshape(-1)[:n]
    single = order[60:160] * 32 + rng.integers(0, 32, 100)
    # Those pages hold something already.
    for c in (cache.k, cache.v):
        c.scales[order[60:160]] = 0.01
    cache.put()
    slots = np.concatenate([single[:50], slots, single[50:], [-1] * 9])
    x = rng.standard_normal((len(slots), 6, 64)).astype(np.float32)
    frequencies, _ = env[1].rope_frequencies(32, 10000.0)
    angles = angles_of(rng.integers(0, 2000, len(slots)), frequencies, 1.0).astype(np.float32)
    run_store(env, dev, cache, slots, x, 2, 32, True, angles)
    cache.check()


@pytest.mark.parametrize("page_tokens,kv_heads,width,shift,pad", [(16, 3, 64, 0, 0), (64, 2, 128, 4, 1),
                                                                  (128, 1, 256, 0, 4), (32, 2, 512, 0, 0)])
def test_load(env, dev, page_tokens, kv_heads, width, shift, pad):
    rt, kern, stream = env
    rng = np.random.default_rng(width)
    cache = DeviceCache(env, dev, 7, page_tokens, kv_heads, width, rng)
    for c in (cache.k, cache.v):
        c.scales[:6] = rng.uniform(1e-3, 2, (6, kv_heads))
    cache.put()
    slots = rng.integers(0, 7 * page_tokens, 50).astype(np.int32)
    slots[[3, 11, 12]] = [-1, 7 * page_tokens, 2**31 - 1]
    n = kv_heads * width
    k = dev.put(np.full((50, 2 * n + pad), 5.0, np.float32), shift)   # one row of k | v
    kern.kv8_load(cache.arg, dev.put(slots), 50, k, 2 * n + pad, k + 4 * n, 2 * n + pad, stream)
    rt.sync(stream)
    got = dev.get(k, np.empty((50, 2 * n + pad), np.float32))
    assert np.all(got[:, 2 * n:] == 5.0) and np.all(got[[3, 11, 12]] == 5.0)
    for c, at in ((cache.k, 0), (cache.v, n)):
        for i, s in enumerate(slots):
            if 0 <= s < 7 * page_tokens:
                page, t = s // page_tokens, s % page_tokens
                with np.errstate(all="ignore"):
                    want = c.codes[page, :, t].astype(np.float32) * c.scales[page][:, None]
                assert np.array_equal(got[i, at:at + n], want.reshape(-1), equal_nan=True)


# ---- attention ------------------------------------------------------------

def make_attention(env, dev, lengths, counts, heads, kv_heads, width, page_tokens, seed, spread=1.0):
    """A cache whose requests hold `lengths` positions in shuffled pages; everything else in it is left as it may be:
    codes of any kind, scales NaN, infinite or huge, table entries of no page."""
    rng = np.random.default_rng(seed)
    need = [-(-max(n, 0) // page_tokens) for n in lengths]
    pages = sum(need) + 3
    cache = DeviceCache(env, dev, pages, page_tokens, kv_heads, width, rng)
    order = rng.permutation(pages)
    table = rng.choice(np.array([-1, -5, pages, 2**31 - 1], np.int32), (len(lengths), max(need + [1]) + 1))
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    for c, s in ((cache.k, 1 / 60), (cache.v, 1 / 90)):
        c.scales[order[:at]] = s * np.exp(spread * rng.standard_normal((at, kv_heads)))
    cache.put()
    rows = sum(max(c, 0) for c in counts)
    q = rng.standard_normal((rows + 2, heads, width)).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(np.maximum(counts, 0))]).astype(np.int32)
    return cache, q, starts, table


def run_attention(env, dev, cache, q, starts, lengths, table, window=0, scale=None, most=None, longest=None,
                  workspace=None, q_pad=0, out_pad=0, shift=0, count=None):
    rt, kern, stream = env
    rows, heads, width = q.shape
    count = rows if count is None else count
    scale = width ** -0.5 if scale is None else scale
    n = heads * width
    wide = np.full((rows, n + q_pad), np.nan, np.float32)
    wide[:, :n] = q.reshape(rows, n)
    out = np.full((rows, n + out_pad), 0.25, np.float32)
    po = dev.put(out, shift)
    most = most or max(1, int(np.diff(starts).max()))
    longest = longest or max(1, int(np.max(lengths)))
    size = kern.kv8_attention_bytes(cache.arg, count, len(lengths), most, longest, heads, window)
    size = size if workspace is None else workspace
    scratch = dev.put(np.full(size, 0xFF, np.uint8)) if size else 0   # NaN
    kern.kv8_attention(cache.arg, dev.put(wide, shift), n + q_pad, po, n + out_pad, count, dev.put(starts),
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
    want, weight, top = attention(q, np.full(q.shape, 0.25), cache.k.values(), cache.v.values(), starts, lengths,
                                  table, cache.pages, cache.page_tokens, window, np.float32(scale), count)
    longest = max(1, int(np.max(lengths)))
    bound = attention_bound(weight, top, width, longest)
    assert np.all(np.isfinite(got) == np.isfinite(want))
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


@pytest.mark.parametrize("heads,kv_heads,width,page_tokens,length,tokens,window", [
    (8, 2, 128, 64, 9000, 1, 0), (8, 2, 128, 16, 9001, 3, 0), (4, 4, 64, 128, 5000, 1, 1000),
    (16, 1, 64, 32, 6000, 9, 0), (8, 8, 128, 64, 2500, 300, 0), (4, 2, 256, 32, 1500, 130, 500),
    (2, 1, 512, 64, 3000, 2, 0), (8, 2, 128, 32, 700, 700, 0), (4, 1, 64, 16, 1030, 515, 100),
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
@pytest.mark.parametrize("lengths,counts", [([150, 400, 60], [1, 2, 1]), ([150, 400, 60], [100, 33, 1])])
def test_attention_holes(env, dev, page_tokens, lengths, counts):
    """Positions whose page is missing or no page are not there; a request with none left gives zeros."""
    cache, q, starts, table = make_attention(env, dev, lengths, counts, 8, 2, 128, page_tokens, 4)
    table[0, 0], table[1, 2], table[1, 1], table[2, :] = -1, 2**31 - 1, -2**31, cache.pages
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    check_attention(cache, q, got, starts, lengths, table)
    assert np.all(got[starts[2]:starts[3]] == 0)


@pytest.mark.parametrize("tokens", [1, 4, 80])
def test_attention_values(env, dev, tokens):
    """Magnitudes at the ends: tiny and huge queries, scores far apart, scales of pages that differ by 2^60, a zero
    query, NaN and infinity in one head, a page that reads as NaN seen by some of the rows only."""
    lengths, counts = [300, 300], [tokens, 1]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, 8, 2, 64, 32, 5)
    q[:, 1] = 0
    q[:, 2] *= 1e-30
    q[:, 3] *= 40        # one position takes everything
    q[0, 4, 7] = np.nan
    q[0, 5, 9] = np.inf
    q[:, 6] *= 1e-38
    got = run_attention(env, dev, cache, q, starts, lengths, table)
    fine = np.ones(q.shape[:2], bool)
    fine[0, 4:6] = False
    assert np.all(np.isnan(got[~fine]))
    clean = np.where(fine[..., None], q, 0)
    check_attention(cache, clean, np.where(fine[..., None], got, run_attention(env, dev, cache, clean, starts, lengths,
                                                                                table)), starts, lengths, table)
    # Steps 2^60 apart, in both orders.
    for c, up in ((cache.v, 2.0 ** 30), (cache.v, 2.0 ** -60)):
        c.scales[table[0, 0:5]] *= np.float32(up)
    cache.put()
    got = run_attention(env, dev, cache, clean, starts, lengths, table)
    check_attention(cache, clean, got, starts, lengths, table)
    # The last page's keys and values read as NaN: rows that see it do, the others do not.
    cache.v.scales[table[0, 9]] = np.nan
    cache.k.scales[table[1, 9]] = np.inf
    cache.put()
    got = run_attention(env, dev, cache, clean, starts, lengths, table)
    sees = np.arange(300 - tokens, 300) >= 9 * 32
    assert np.all(np.isnan(got[:tokens][sees])) and np.all(np.isfinite(got[:tokens][~sees]))
    assert not np.any(np.isfinite(got[tokens]).all(1))


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 3]])
@pytest.mark.parametrize("q_pad,out_pad,shift", [(4, 8, 0), (1, 3, 0), (0, 0, 4), (5, 0, 12)])
def test_attention_strides(env, dev, counts, q_pad, out_pad, shift):
    lengths = [100, 70, 33]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, 8, 2, 128, 32, 6)
    got = run_attention(env, dev, cache, q, starts, lengths, table, q_pad=q_pad, out_pad=out_pad, shift=shift)
    check_attention(cache, q, got, starts, lengths, table)


def test_attention_rows_cut_off(env, dev):
    """starts past `count`, negative and out of order: no row outside is read or written."""
    lengths = [50, 60, 70, 80]
    cache, q, _, table = make_attention(env, dev, lengths, [5, 5, 5, 5], 4, 2, 64, 16, 7)
    starts = np.array([-3, 4, 2, 30, 2**31 - 1], np.int32)
    got = run_attention(env, dev, cache, q, starts, lengths, table, most=10, count=10)
    assert np.all(got[10:] == 0.25) and np.all(np.isfinite(got))
    want, weight, top = attention(q, np.full(q.shape, 0.25), cache.k.values(), cache.v.values(), np.array([-3, 4]),
                                  lengths[:1], table, cache.pages, 16, 0, np.float32(0.125), 10)
    assert np.all(np.abs(got[:2] - want[:2]).max(2) <= attention_bound(weight, top, 64, 80)[:2])


def test_attention_starts_outside(env, dev):
    """starts of the ends of int32: those requests bring nothing, and the rows stay."""
    lengths = [50, 60, 70, 80]
    cache, q, _, table = make_attention(env, dev, lengths, [5, 5, 5, 5], 16, 2, 64, 16, 7)
    starts = np.array([2**31 - 1, -2**31, -2**31, 2**31 - 1, -2**31], np.int32)
    for most in (1, 22):   # requests of a few rows, and wide tiles
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
    size = env[1].kv8_attention_bytes(cache.arg, len(q), 4, 100, 3000, heads, 0)
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
    size = env[1].kv8_attention_bytes(cache.arg, len(q), n, int(counts.max()), 9000, heads, 0)
    for workspace in (size, size // 2 & ~15):
        got = run_attention(env, dev, cache, q, starts, lengths, table, longest=9000, workspace=workspace)
        check_attention(cache, q, got, starts, lengths, table)


def test_attention_scales(env, dev):
    """A scale of 0, a negative one and a large one."""
    lengths, counts = [100, 64], [20, 1]
    cache, q, starts, table = make_attention(env, dev, lengths, counts, 4, 2, 64, 16, 8)
    for scale in (0.0, -0.125, 3.0):
        got = run_attention(env, dev, cache, q, starts, lengths, table, scale=scale)
        check_attention(cache, q, got, starts, lengths, table, scale=scale)


def test_attention_far_pages(env, dev):
    """Pages past 2^32 bytes into the code arrays."""
    rt, kern, stream = env
    pages, page_tokens, kv_heads, width = 70000, 128, 4, 128    # 4.6 GB each
    lengths, counts = [300], [3]
    small, q, starts, table = make_attention(env, dev, lengths, counts, 8, kv_heads, width, page_tokens, 9)
    codes, scales = kern.kv8_bytes(pages, page_tokens, kv_heads, width)
    at = [rt.malloc(n) for n in (codes, codes, scales, scales)]
    dev.ptrs += at
    far = np.array([[69999, 3, 65999]], np.int32)
    for (c, codes_at, scales_at) in ((small.k, at[0], at[2]), (small.v, at[1], at[3])):
        packed = c.packed().reshape(c.codes.shape[0], -1)
        for j in range(3):
            rt.upload(codes_at + int(far[0, j]) * packed.shape[1], packed[table[0, j]])
            rt.upload(scales_at + int(far[0, j]) * 4 * kv_heads, c.scales[table[0, j]])
    big = DeviceCache.__new__(DeviceCache)
    big.arg = Kv8(*at, pages, page_tokens, kv_heads, width)
    got = run_attention(env, dev, big, q, starts, lengths, far)
    check_attention(small, q, got, starts, lengths, table)
    # A store and a load there.
    x = np.random.default_rng(1).standard_normal((1, 2 * kv_heads * width)).astype(np.float32)
    slot, n = dev.put(np.array([69999 * page_tokens], np.int32)), kv_heads * width
    src, back = dev.put(x), dev.put(np.zeros_like(x))
    kern.kv8_store(big.arg, slot, 1, src, 2 * n, src + 4 * n, 2 * n, 0, 0, 0, 0, 0, 0, 0, 0, stream)
    kern.kv8_load(big.arg, slot, 1, back, 2 * n, back + 4 * n, 2 * n, stream)
    rt.sync(stream)
    got = dev.get(back, x).reshape(-1, width)
    step = np.abs(x.reshape(-1, width)).max(1, keepdims=True) / 127
    assert np.all(np.abs(got - x.reshape(-1, width)) <= step * (0.5 + 1e-5))


# ---- a step as it is used -------------------------------------------------

class Server:
    """One layer of a server: requests that come, decode, take drafts back and finish."""

    def __init__(self, env, dev, heads=8, kv_heads=2, width=64, page_tokens=16, requests=5, max_tokens=160, pages=60):
        self.env, self.dev = env, dev
        rt, kern, _ = env
        self.rng = np.random.default_rng(11)
        self.heads, self.kv_heads, self.width, self.max_tokens = heads, kv_heads, width, max_tokens
        self.cache = DeviceCache(env, dev, pages, page_tokens, kv_heads, width, self.rng)
        self.state = Pages(requests, 20, pages, page_tokens, self.rng.permutation(pages))
        self.pages = DevicePages(env, dev, self.state, max_tokens)
        self.rotated = 32
        self.frequencies, _ = kern.rope_frequencies(self.rotated, 10000.0, scaling="bands", factor=4.0, original=128,
                                                    low=1, high=4)
        self.f = dev.put(self.frequencies)
        n = (heads + 2 * kv_heads) * width
        self.x = np.zeros((max_tokens, n), np.float32)
        self.px = dev.put(self.x)
        self.pa = dev.put(np.zeros((max_tokens, self.rotated // 2, 2), np.float32))
        self.pq = dev.put(np.zeros((max_tokens, heads * width), np.float32))
        self.out = np.full((max_tokens, heads * width), 0.25, np.float32)
        self.po = dev.put(self.out)
        self.size = kern.kv8_attention_bytes(self.cache.arg, max_tokens, requests, max_tokens, 320, heads, 0)
        self.scratch = dev.put(np.full(max(self.size, 16), 0xFF, np.uint8))

    def launch(self, stream=None):
        rt, kern, default = self.env
        stream = default if stream is None else stream
        p, n, h, kvh, w = self.pages, self.x.shape[1], self.heads, self.kv_heads, self.width
        p.launch(stream)
        kern.rope_angles(p.positions, self.max_tokens, self.f, self.rotated, 1.0, self.pa, stream)
        kern.kv8_store(self.cache.arg, p.slots, self.max_tokens, self.px + 4 * h * w, n, self.px + 4 * (h + kvh) * w, n,
                       self.pa, self.rotated, 1, self.px, n, self.pq, h * w, h, stream)
        kern.kv8_attention(self.cache.arg, self.pq, h * w, self.po, h * w, self.max_tokens, p.starts, p.lengths,
                           p.table, p.stride, len(self.state.held), self.max_tokens, 320, h, 0, w ** -0.5, self.scratch,
                           self.size, stream)

    def inputs(self, lengths, counts):
        rt = self.env[0]
        self.x = self.rng.standard_normal(self.x.shape).astype(np.float32)
        rt.upload(self.px, self.x)
        rt.upload(self.po, self.out)
        rt.upload(self.pages.lengths, np.asarray(lengths, np.int32))
        rt.upload(self.pages.counts, np.asarray(counts, np.int32))

    def check(self, lengths, counts):
        h, kvh, w = self.heads, self.kv_heads, self.width
        starts, positions, slots = self.state.step(lengths, counts, self.max_tokens)
        self.pages.check(starts, positions, slots)
        x = self.x.reshape(self.max_tokens, -1, w)
        angles = angles_of(positions, self.frequencies, 1.0).astype(np.float32)
        q, k = (rotate(x[:, a:b], angles, True).astype(np.float32) for a, b in ((0, h), (h, h + kvh)))
        self.cache.k.store(slots, k)
        self.cache.v.store(slots, x[:, h + kvh:])
        self.cache.check()
        got = self.dev.get(self.po, self.out).reshape(q.shape)
        check_attention(self.cache, q, got, starts, lengths, self.state.table)


STEPS = [([40, 0, 0, 0, 0], [40, 0, 0, 0, 0]),                     # a prompt
         ([41, 100, 17, 0, 0], [1, 100, 17, 0, 0]),                # two more beside its first token
         ([42, 101, 18, 1, 0], [1, 1, 1, 1, 0]),
         ([47, 106, 23, 6, 5], [5, 5, 5, 5, 5]),                   # drafts
         ([44, 104, 20, 3, 5], [1, 2, 1, 1, 1]),                   # some taken back
         ([0, 105, 48, 4, 6], [0, 1, 28, 1, 1]),                   # one finishes, one gets a longer turn
         ([33, 106, 49, 0, 7], [33, 1, 1, 0, 1]),
         ([34, 320, 50, 300, 8], [1, 60, 1, 60, 1])]               # positions that were never stored read as they may


def test_serving_steps(env, dev):
    server = Server(env, dev)
    for lengths, counts in STEPS:
        server.inputs(lengths, counts)
        server.launch()
        env[0].sync(env[2])
        server.check(lengths, counts)


def test_serving_steps_captured(env, dev):
    """The whole step captured once and replayed for every step, with eager work between, on another stream."""
    rt, kern, stream = env
    server, other = Server(env, dev), rt.stream()
    graph = Graph(rt, other, [lambda: server.launch(other)])
    eager = Server(env, dev)
    for lengths, counts in STEPS:
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
    """Two attention calls on two streams with workspaces of their own."""
    rt, kern, stream = env
    other = rt.stream()
    calls = []
    for seed, s in ((21, stream), (22, other)):
        lengths = [4000]
        cache, q, starts, table = make_attention(env, dev, lengths, [1], 8, 2, 128, 64, seed)
        size = kern.kv8_attention_bytes(cache.arg, 1, 1, 1, 4000, 8, 0)
        out = dev.put(np.zeros(q.shape, np.float32))
        args = (cache.arg, dev.put(q), 1024, out, 1024, 1, dev.put(starts), dev.put(np.array(lengths, np.int32)),
                dev.put(table), table.shape[1], 1, 1, 4000, 8, 0, 128 ** -0.5, dev.put(np.zeros(max(size, 16), np.uint8)),
                size, s)
        calls.append((cache, q, starts, table, lengths, out, args))
    for _ in range(20):
        for c in calls:
            kern.kv8_attention(*c[-1])
    rt.sync(stream)
    rt.sync(other)
    for cache, q, starts, table, lengths, out, _ in calls:
        got = dev.get(out, q)
        check_attention(cache, q[:1], got[:1], starts, lengths, table)
