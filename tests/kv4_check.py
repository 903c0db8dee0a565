"""The 4-bit paged cache (include/fyodor_hip_kv4.h) and log probabilities (include/fyodor_hip_logprobs.h) stated in
numpy, in 64 bits and in plain loops."""
import numpy as np

from serving_check import F32_HALF

BLOCK, MOST = 32, 8160.0


# ---- the 4-bit cache ------------------------------------------------------

def step_of(block):
    """A block's step, an fp16 number of 8 bits, from its 32 fp32 elements."""
    low, high = float(block.min()), float(block.max())
    m = low if -low >= high else high
    d = m / -8
    if d:
        # The nearest of 8 significant bits, ties to even (Python's round).
        unit = 2.0 ** (np.frexp(abs(d))[1] - 8)
        d = float(np.copysign(round(abs(d) / unit) * unit, d))
    return np.float16(np.clip(d, -MOST, MOST))


def quantised(rows):
    """(codes 0 .. 15, steps) of finite fp32 rows [..][width]."""
    blocks = rows.reshape(-1, BLOCK)
    codes, steps = np.empty(blocks.shape, np.uint8), np.empty(len(blocks), np.float16)
    for i, b in enumerate(blocks):
        steps[i] = step_of(b)
        d = float(steps[i])
        codes[i] = 8 if d == 0 else np.clip(np.rint(b.astype(np.float64) / d) + 8, 0, 15)
    return codes.reshape(rows.shape), steps.reshape(rows.shape[:-1] + (-1,))


class Cache4:
    """One of the two caches: codes [page][head][token][width] and steps [page][head][token][block]."""

    def __init__(self, pages, page_tokens, kv_heads, width, rng, kind):
        self.kind, self.page_tokens = kind, page_tokens
        # Whatever the memory held before: codes and steps of any bits, NaN and infinity among them.
        self.codes = rng.integers(0, 16, (pages, kv_heads, page_tokens, width)).astype(np.uint8)
        bits = rng.integers(0, 1 << 16, (pages, kv_heads, page_tokens, width // BLOCK)).astype(np.uint16)
        bits[rng.random(bits.shape) < 0.3] = 0x7E00
        self.steps = bits.view(np.float16)

    def packed(self):
        p, h, t, w = self.codes.shape
        out = np.zeros((p, h, t * w // 2), np.uint8)
        at, shift = self._places()
        np.bitwise_or.at(out, (np.arange(p)[:, None, None, None], np.arange(h)[None, :, None, None], at[None, None]),
                         self.codes << shift)
        return out

    def _places(self):
        """Byte and shift of element d of position t."""
        _, _, size, w = self.codes.shape
        t, d = np.arange(size)[:, None], np.arange(w)[None]
        if self.kind == "k":
            nibble = ((d // 32 * size + t) * 4 + d % 32 // 8) * 8 + d % 2 * 4 + d % 8 // 2
        else:
            nibble = ((t // 8 * (w // 4) + d // 4) * 8 + t % 8) * 4 + d % 4
        return nibble // 2, (nibble % 2 * 4).astype(np.uint8)

    def unpack(self, raw):
        p, h, t, w = self.codes.shape
        at, shift = self._places()
        return raw.reshape(p, h, -1)[:, :, at] >> shift & 15

    def _step_places(self):
        _, _, t, blocks = self.steps.shape
        i, b = np.arange(t)[:, None], np.arange(blocks)[None]
        return (i // 16 * blocks + b) * 16 + i % 4 * 4 + i % 16 // 4 if self.kind == "k" else b * t + i

    def packed_steps(self):
        p, h, t, blocks = self.steps.shape
        out = np.empty((p, h, t * blocks), np.float16)
        out[:, :, self._step_places()] = self.steps
        return out

    def unpack_steps(self, raw):
        p, h, t, blocks = self.steps.shape
        return raw.reshape(p, h, -1)[:, :, self._step_places()]

    def values(self):
        with np.errstate(all="ignore"):
            steps = np.repeat(self.steps.astype(np.float64), BLOCK, -1)
            return (self.codes.astype(np.float64) - 8) * steps


def store(keys, values, slots, k, v):
    """fp32 rows [n][head][width] into their slots of both caches."""
    pages, _, size, _ = keys.codes.shape
    for i, s in enumerate(int(s) for s in slots):
        if s < 0 or s >= pages * size:
            continue
        at = (s // size, slice(None), s % size)
        bad = ~(np.isfinite(k[i]).all(1) & np.isfinite(v[i]).all(1))
        for c, x in ((keys, k[i]), (values, v[i])):
            c.codes[at], c.steps[at] = quantised(np.where(bad[:, None], np.float32(0), x))
        keys.steps[at] = np.where(bad[:, None], np.float16(np.nan), keys.steps[at])


def held(keys, values):
    """What is held of each, in 64 bits: NaN in both where a position is marked."""
    k, v = keys.values(), values.values()
    return k, np.where(np.isnan(np.repeat(keys.steps, BLOCK, -1)), np.nan, v)


# ---- log probabilities ----------------------------------------------------

def masked(x, mask):
    """Rows in 64 bits with minus infinity where the mask's bits are set."""
    x = x.astype(np.float64)
    if mask is not None:
        off = (mask[np.arange(x.shape[1]) // 32] >> (np.arange(x.shape[1]) % 32).astype(np.uint32)) & 1
        x = np.where(off[None] == 1, -np.inf, x)
    return x


def logprobs(x, mask, scale, tokens, top):
    """(logprobs, ranks, entropies, top_ids, top_logprobs) and how far fp32 may be off in (logprobs, entropies)."""
    rows, n = x.shape
    x = masked(x, mask)
    lp, ranks = np.full(rows, np.nan), np.full(rows, -1, np.int32)
    entropy, ids, top_lp = np.full(rows, np.nan), np.full((rows, top), -1, np.int32), np.full((rows, top), np.nan)
    off = np.zeros((2, rows))
    for i, r in enumerate(x):
        t = int(tokens[i])
        if not 0 <= t < n:
            lp[i] = 0
        if np.isnan(r).any() or r.max() == np.inf or r.max() == -np.inf:
            continue
        z = (r - r.max()) * float(np.float32(scale))
        e = np.exp(z)
        total, some = e.sum(), e > 0
        lse, p, w = np.log(total), e[some] / total, -z[some]
        entropy[i] = lse + (p * w).sum()
        order = np.lexsort((np.arange(n), -r))
        if 0 <= t < n:
            lp[i] = z[t] - lse
        if 0 <= t < n and r[t] > -np.inf:
            ranks[i] = np.flatnonzero(order == t)[0]
        first = order[:top]
        first = first[r[first] > -np.inf]
        ids[i, :len(first)] = first
        top_lp[i] = -np.inf
        top_lp[i, :len(first)] = z[first] - lse
        # An exponential of z: its argument (a difference, a product) is off by 3 roundings of |z|, exp2 by two steps.
        # A thread adds up at most n / 256 + 64 of them one after another, 256 threads and 64 shares meet in 16 more
        # steps. Terms below 2^-126 may be missing: 2^-126 n at most.
        chain = n / 256 + 64 + 16
        each = (p * (3 * w + 4 + chain)).sum() * F32_HALF + n * 2.0 ** -126
        off[0, i] = each
        off[1, i] = each + (p * w * (3 * w + 8 + chain)).sum() * F32_HALF + (p * w).sum() * each
    return lp, ranks, entropy, ids, top_lp, off
