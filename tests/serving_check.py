"""The serving operators (include/fyodor_hip_serving.h) stated in numpy, in 64
bits and in plain loops, and device arrays for their tests."""
import math

import numpy as np

F32_HALF = 2.0 ** -24   # half a step of fp32, relative
SCALE_FLOOR = 2.0 ** -100


class Dev:
    """Device arrays, freed together."""

    def __init__(self, rt):
        self.rt, self.ptrs = rt, []

    def put(self, a, extra=0):
        a = np.ascontiguousarray(a)
        p = self.rt.malloc(a.nbytes + extra + 16)
        self.ptrs.append(p)
        if a.nbytes:
            self.rt.upload(p + extra, a)
        return p + extra

    def get(self, p, like):
        return self.rt.download(p, np.empty_like(like))

    def close(self):
        for p in self.ptrs:
            self.rt.free(p)


# ---- pages ----------------------------------------------------------------

class Pages:
    """The page bookkeeping of nya_hip_page_step."""

    def __init__(self, requests, stride, pages, page_tokens, order):
        self.page_tokens, self.pages = page_tokens, pages
        self.table = np.full((requests, stride), -1, np.int32)
        self.held = np.zeros(requests, np.int32)
        self.free_pages = np.asarray(order, np.int32).copy()
        self.free_count = np.array([pages, 0], np.int32)

    def step(self, lengths, counts, max_tokens):
        """starts, positions, slots of the step."""
        requests, stride = self.table.shape
        top, refused, asked = int(self.free_count[0]), 0, 0
        need = [-(-max(int(n), 0) // self.page_tokens) for n in lengths]
        for r in range(requests):
            if need[r] > stride:
                continue
            for j in range(need[r], int(self.held[r])):
                self.free_pages[top] = self.table[r, j]
                self.table[r, j] = -1
                top += 1
            self.held[r] = min(self.held[r], need[r])
        available = top
        for r in range(requests):
            if need[r] > stride:
                refused += 1
                continue
            asked += max(0, need[r] - int(self.held[r]))
            if need[r] > self.held[r] and asked > available:
                refused += 1
                continue
            while self.held[r] < need[r]:
                top -= 1
                self.table[r, self.held[r]] = self.free_pages[top]
                self.held[r] += 1
        self.free_count[:] = top, refused
        starts = np.zeros(requests + 1, np.int32)
        positions, slots = np.full(max_tokens, -1, np.int32), np.full(max_tokens, -1, np.int32)
        row = 0
        for r in range(requests):
            starts[r] = min(row, 2**31 - 1)
            count = max(int(counts[r]), 0)
            for j in range(min(count, max(max_tokens - row, 0))):
                p = max(int(lengths[r]), 0) - count + j
                positions[row + j] = p
                if p >= 0 and p // self.page_tokens < self.held[r]:
                    slots[row + j] = self.table[r, p // self.page_tokens] * self.page_tokens + p % self.page_tokens
            row += count
        starts[requests] = min(row, 2**31 - 1)
        return starts, positions, slots


# ---- rotary positions -----------------------------------------------------

def angles_of(positions, frequencies, magnitude):
    a = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)
    return np.stack([np.cos(a), np.sin(a)], -1) * float(magnitude)


def rotate(x, angles, halves):
    """x [rows][heads][width] by angles [rows][pairs][2], in 64 bits."""
    y, half = x.astype(np.float64), angles.shape[1]
    j = np.arange(half)
    first, second = (j, j + half) if halves else (2 * j, 2 * j + 1)
    a, b = y[..., first], y[..., second]
    c, s = (angles[:, None, :, i].astype(np.float64) for i in range(2))
    out = y.copy()
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out


# ---- the 8-bit cache ------------------------------------------------------

class Cache:
    """One of the two caches: codes [page][head][token][width] and scales."""

    def __init__(self, pages, page_tokens, kv_heads, width, rng, kind):
        self.kind, self.page_tokens = kind, page_tokens
        # Whatever the memory held before: codes of any kind, scales too.
        self.codes = rng.integers(-127, 128, (pages, kv_heads, page_tokens, width)).astype(np.int8)
        self.scales = rng.choice(np.array([np.nan, np.inf, -1, 0, 1e30, 1e-30], np.float32), (pages, kv_heads))
        # A page that reads as NaN holds no codes that mean anything.
        self.known = np.ones((pages, kv_heads), bool)

    def packed(self):
        p, h, t, w = self.codes.shape
        if self.kind == "k":
            return np.ascontiguousarray(self.codes.reshape(p, h, t, w // 16, 16).transpose(0, 1, 3, 2, 4))
        return np.ascontiguousarray(self.codes.reshape(p, h, t // 16, 16, w).transpose(0, 1, 2, 4, 3))

    def unpack(self, raw):
        p, h, t, w = self.codes.shape
        if self.kind == "k":
            return raw.reshape(p, h, w // 16, t, 16).transpose(0, 1, 3, 2, 4).reshape(p, h, t, w)
        return raw.reshape(p, h, t // 16, w, 16).transpose(0, 1, 2, 4, 3).reshape(p, h, t, w)

    def store(self, slots, rows):
        """fp32 rows [n][head][width] into their slots."""
        pages, _, size, _ = self.codes.shape
        i = 0
        while i < len(slots):
            s = int(slots[i])
            if s < 0 or s >= pages * size:
                i += 1
                continue
            j = i + 1
            while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % size:
                j += 1
            self._run(s // size, s % size, rows[i:j])
            i = j

    def _run(self, page, at, rows):
        for h in range(rows.shape[1]):
            x = rows[:, h]
            old = self.scales[page, h]
            with np.errstate(all="ignore"):
                wanted = np.float32(np.max(np.abs(x))) * (np.float32(1) / np.float32(127))
                if wanted < SCALE_FLOOR:
                    wanted = np.float32(SCALE_FLOOR)
                scale = wanted
                if at:
                    if wanted <= old or np.isnan(old):
                        scale = old
                    elif np.isfinite(wanted):
                        c = np.rint(self.codes[page, h].astype(np.float64) * float(old) / float(wanted))
                        self.codes[page, h] = np.clip(c, -127, 127).astype(np.int8)
                if np.isfinite(scale):
                    c = np.clip(np.rint(x.astype(np.float64) / float(scale)), -127, 127)
                    self.codes[page, h, at:at + len(x)] = c.astype(np.int8)
                self.known[page, h] = np.isfinite(scale) and (self.known[page, h] or len(x) == self.page_tokens)
                self.scales[page, h] = scale

    def values(self):
        with np.errstate(all="ignore"):
            return self.codes.astype(np.float64) * self.scales.astype(np.float64)[..., None, None]


# ---- attention ------------------------------------------------------------

def attention(q, out, keys, values, starts, lengths, table, pages, page_tokens, window, scale, count):
    """Rows of `out` [count][heads][width] that the batch covers; keys and values [page][head][token][width] in 64
    bits. Returns (out, the largest sum |q k| scale of each (row, head), the largest |v| it sees)."""
    out, group = out.astype(np.float64), q.shape[1] // keys.shape[1]
    weight, top = np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
    for r in range(len(lengths)):
        begin, end = max(int(starts[r]), 0), min(int(starts[r + 1]), count)
        for row in range(begin, end):
            p = int(lengths[r]) - (int(starts[r + 1]) - begin) + row - begin
            p = min(p, table.shape[1] * page_tokens - 1) if p >= 0 else -1
            first = max(0, int(lengths[r]) - (int(starts[r + 1]) - begin) + row - begin - window + 1) if window else 0
            t = np.arange(first, p + 1)
            page = table[r, t // page_tokens] if t.size else t
            t = t[(page >= 0) & (page < pages)]
            page = table[r, t // page_tokens] if t.size else t
            for h in range(q.shape[1]):
                if not t.size:
                    out[row, h] = 0
                    continue
                k, v = keys[page, h // group, t % page_tokens], values[page, h // group, t % page_tokens]
                with np.errstate(invalid="ignore"):
                    s = k @ q[row, h].astype(np.float64) * scale
                    e = np.exp(s - s.max())
                    out[row, h] = e @ v / e.sum()
                weight[row, h] = (np.abs(k) @ np.abs(q[row, h].astype(np.float64))).max() * abs(scale)
                top[row, h] = np.abs(v).max()
    return out, weight, top


def attention_bound(weight, top, width, longest):
    """How far fp32 may be off. A score is a sum of `width` products of q's two pieces (2^-22 of each) in MFMA steps
    of 16 or 32 (at most width / 16 + 8 roundings), scaled and shifted (4 more): `weight` bounds the sum of their
    magnitudes. A score off by d moves the softmax's weights by a factor e^d each and so the output by at most 2 d of
    the largest value. The weights enter in two pieces (2^-22), exp2 is off by two steps, and they are summed in
    chains of 16 and more positions, over and under the fraction line."""
    score = weight * (2.0 ** -22 + (width / 16 + 12) * F32_HALF)
    return top * (2 * score + 2.0 ** -22 + (2 * longest / 16 + 48) * F32_HALF)


def bands(rotated, base, factor, original, low, high):
    j = np.arange(rotated // 2)
    f = base ** (-2.0 * j / rotated)
    g = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
    return g * f + (1 - g) * f / factor
