"""Calls of the serving operators (include/fyodor_hip_serving.h) at the ends of what they allow, on an MI355X against
the statements in serving_check.py."""
import numpy as np
import pytest

from serving_check import attention_bound
from test_gpu_serving import dev, env, make_attention, run_attention   # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


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
