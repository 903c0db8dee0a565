"""The operators of a serving step over a paged 4-bit cache, and of its answers, as measurable cases.

A case is one pass through

``store``      ``kv4_store`` (rotating q and k) and ``kv4_load`` of every row that it stored;
``load``       ``kv4_load`` alone: a prefix handed on;
``attention``  ``kv4_attention``: causal attention of the batch's rows over their requests' pages;
``logprobs``   ``logprobs``: of each row of logits the given token's log probability and rank, the entropy, and the
               most likely tokens with theirs;
``step``       store, attention and log probabilities in turn, as one layer and the end of a serving step run them.

Head shapes, page sizes and vocabularies are the ones this repository's decoders, benchmark and tests use, and their
neighbours. Requests' lengths and their new tokens come from the case alone (``_batch``); values from the seed. Keys
and values are normal with a per-channel spread, as a decoder's projections have; logits are normal with a few likely
tokens in each row, in the precision of fp32 or rounded to 8 bits, as a model that computes in bf16 gives them (then
tokens tie).
"""
import math
import random

import torch

own = False

INTERLEAVED, HALVES = 0, 1
SCRATCH = 64 << 20   # scratch a serving program keeps
BLOCK = 32           # elements that share a step
MOST = 8160.0        # the largest step


def _case(name, op, shape=(32, 8, 128), page=64, requests=1, shortest=1, longest=1, prompts=0, chunk=0, single=1,
          idle=0, window=0, rotated=0, layout=INTERLEAVED, mix=1, rows=0, vocabulary=0, top=0, scale=1.0, mask=False,
          rounded=False):
    heads, kv_heads, width = shape
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "width": width, "page": page, "requests": requests,
         "shortest": shortest, "longest": longest, "prompts": prompts, "chunk": chunk, "single": single, "idle": idle,
         "window": window, "rotated": rotated or width, "layout": layout, "mix": mix, "rows": rows,
         "vocabulary": vocabulary, "top": top, "scale": scale, "mask": mask, "rounded": rounded}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decode token for each of 61 requests into their last pages: bound by its launches.
        _case("store-decode", "store", (32, 8, 128), 64, 61, 100, 4096, mix=21),
        # Prompts of odd lengths, small heads and pages, the other rotary layout.
        _case("store-prompt", "store", (32, 4, 64), 32, 3, 900, 2333, prompts=3, chunk=1601, layout=HALVES, mix=22),
        # A prefix of 5 requests read back in fp32.
        _case("load-prefix", "load", (16, 8, 256), 16, 5, 200, 1111, prompts=5, chunk=1111, mix=23),
        # The smallest batch over the longest cache: one token.
        _case("attend-long", "attention", (32, 8, 128), 64, 1, 65536, 65536, mix=24),
        # Steady decoding of 64 requests of every length.
        _case("attend-decode", "attention", (32, 8, 128), 64, 64, 500, 8192, mix=25),
        # Draft tokens of eight requests checked at once, small heads and pages.
        _case("attend-verify", "attention", (32, 4, 64), 16, 8, 300, 2048, single=5, mix=26),
        # The largest call: a 1024-token prompt chunk at the end of 8192 positions.
        _case("attend-prompt", "attention", (32, 8, 128), 64, 1, 8192, 8192, prompts=1, chunk=1024, mix=27),
        # Prompts and single tokens in wide heads with a local window, one request of the batch idle.
        _case("attend-window", "attention", (16, 8, 256), 32, 6, 300, 3001, prompts=4, chunk=700, idle=1, window=1024,
              mix=28),
        # One sampled token's answer with five alternatives: where latency counts.
        _case("answer-one", "logprobs", rows=1, vocabulary=32000, top=5),
        # The answers of a batch of 64 with twenty alternatives, some tokens suppressed, at temperature 0.8.
        _case("answer-batch", "logprobs", rows=64, vocabulary=128256, top=20, scale=1.25, mask=True, rounded=True),
        # A long text scored: no alternatives, an odd vocabulary.
        _case("score-text", "logprobs", rows=2047, vocabulary=50257),
        # A layer's step and its answers: two prompts join 22 requests that decode.
        _case("serve-step", "step", (32, 8, 128), 64, 24, 64, 2048, prompts=2, chunk=256, mix=29, rows=24,
              vocabulary=32000, top=8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choices(["store", "load", "attention", "logprobs", "step"], [2, 1, 5, 4, 1])[0]
    shape = rng.choice([(32, 8, 128), (32, 4, 64), (16, 8, 256), (32, 32, 128), (8, 1, 512), (20, 4, 128), (6, 2, 64)])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice([INTERLEAVED, HALVES])
    rotated = rng.choice([shape[2], shape[2] // 2, shape[2] // 4])
    window, mix = rng.choice([0, 0, 0, 512, 1000]), rng.randrange(1 << 20)
    rows, vocabulary = _log(rng, 1, 4096), _log(rng, 500, 262144)
    top, scale = rng.choice([0, 1, 5, 8, 20, 33, 64]), rng.choice([1.0, 1.0, 1.25, 0.5])
    mask, rounded = rng.random() < 0.3, rng.random() < 0.5
    if op == "logprobs":
        rows = max(1, min(rows, 100_000_000 // vocabulary))
        return _case(None, op, rows=rows, vocabulary=vocabulary, top=top, scale=scale, mask=mask, rounded=rounded,
                     mix=mix)
    requests, longest = _log(rng, 1, 64), _log(rng, 64, 65536)
    prompts = rng.choice([0, 0, 1, min(requests, 4)])
    chunk = min(longest, _log(rng, 9, 700)) // max(1, prompts // 2) or 1
    single = rng.choice([1, 1, 1, rng.randint(2, 33)])
    if prompts or single > 1:
        longest, requests = min(longest, 4096), min(requests, 24)
    idle = rng.randint(0, 1) if requests > prompts + 1 else 0
    share = rng.randint(1, 30)
    while True:
        longest = max(longest, single, chunk if prompts else 1)
        case = _case(None, op, shape, page, requests, max(1, longest // share), longest, prompts, chunk, single, idle,
                     window if op in ("attention", "step") else 0, rotated, layout, mix,
                     rows=requests if op == "step" else 0, vocabulary=min(vocabulary, 32768) if op == "step" else 0,
                     top=top, scale=scale, mask=mask, rounded=rounded)
        # At most the largest listed calls' bytes and flops.
        cost = work(case)
        if cost["bytes"] <= 300e6 and cost["flops"] <= 125e9:
            return case
        longest, chunk, requests = longest // 2, (chunk + 1) // 2, max(requests // 2, prompts + idle, 1)


def _batch(case):
    """(positions each request holds after the step, how many of them are new), from the case alone."""
    rng, lengths, counts = random.Random(case["mix"]), [], []
    for r in range(case["requests"]):
        n = case["single"]
        if r < case["prompts"]:
            n = case["chunk"] if r == 0 else rng.randint((case["chunk"] + 1) // 2, case["chunk"])
        elif r >= case["requests"] - case["idle"]:
            n = 0
        total = case["longest"] if r == 0 else _log(rng, case["shortest"], case["longest"])
        lengths.append(max(total, n))
        counts.append(n)
    return lengths, counts


# ---- inputs ---------------------------------------------------------------

def _normal(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


class State:
    """What a serving program holds before the call: the cache, its page tables, the batch and its buffers."""


def _prepare_answers(s, seed):
    c, rows, n = s.case, s.case["rows"], s.case["vocabulary"]
    g = torch.Generator(device="cuda").manual_seed(7 * seed + 6)
    s.logits = _normal((rows, n), 7 * seed + 5) * 2.5
    likely = torch.randint(0, n, (rows, 12), generator=g, device="cuda")
    s.logits.scatter_add_(1, likely, 6 + 2 * torch.randn((rows, 12), generator=g, device="cuda"))
    if c["rounded"]:
        s.logits = s.logits.bfloat16().float()
    # Most of the given tokens are likely ones.
    any_token = torch.randint(0, n, (rows,), generator=g, device="cuda")
    s.tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, likely[:, 0], any_token).to(torch.int32)
    s.mask = None
    if c["mask"]:
        # A tenth of the vocabulary is suppressed, none of the given tokens.
        off = torch.rand(-(-n // 32) * 32, generator=g, device="cuda") < 0.1
        off[s.tokens.long()] = False
        s.mask = (off.view(-1, 32).long() << torch.arange(32, device="cuda")).sum(1).to(torch.int32)
    s.logprob, s.entropy = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    s.rank = torch.empty(rows, dtype=torch.int32, device="cuda")
    s.top_ids = torch.empty((rows, c["top"]), dtype=torch.int32, device="cuda")
    s.top_logprobs = torch.empty((rows, c["top"]), device="cuda")


def prepare(case, seed):
    s = State()
    s.case = case
    s.scratch = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    if case["rows"]:
        _prepare_answers(s, seed)
    if case["op"] == "logprobs":
        return s
    s.lengths, s.counts = _batch(case)
    page, heads, kv_heads, width = case["page"], case["heads"], case["kv_heads"], case["width"]
    need = _pages_of(s.lengths, page)
    s.rows = sum(s.counts)
    s.count = s.rows + 3   # a batch padded past its last row
    s.requests, s.stride = case["requests"], max(need) + 1
    s.page_count = sum(need) + 2
    s.most, s.longest = max(s.counts), max(s.lengths)
    g = torch.Generator(device="cuda").manual_seed(7 * seed + 4)
    order = torch.randperm(s.page_count, generator=g, device="cuda").to(torch.int32)
    s.table = torch.full((s.requests, s.stride), -1, dtype=torch.int32, device="cuda")
    taken = 0
    for r, n in enumerate(need):
        s.table[r, :n] = order[taken:taken + n]
        taken += n
    s.new_lengths = _ints(s.lengths)
    starts, at, request = [0], [], []
    for r, (n, c) in enumerate(zip(s.lengths, s.counts)):
        starts.append(starts[-1] + c)
        at += range(n - c, n)
        request += [r] * c
    s.starts = _ints(starts)
    at, request = torch.tensor(at, device="cuda"), torch.tensor(request, device="cuda")
    s.slots = torch.full((s.count,), -1, dtype=torch.int32, device="cuda")
    s.slots[:s.rows] = s.table[request, at // page] * page + (at % page).to(torch.int32)
    # The cache as rows of the same kind left it.
    s.spread = torch.exp(0.5 * _normal((2, kv_heads, 1, width), 7 * seed + 3))
    s.codes, s.steps = [], []
    for kind in range(2):
        x = _normal((s.page_count, kv_heads, page, width), 7 * seed + 1 + kind) * s.spread[kind]
        codes, steps = _quantise(x)
        s.codes.append(_pack(codes, kind))
        s.steps.append(_pack_steps(steps, kind))
    if case["op"] in ("store", "step"):
        j = torch.arange(case["rotated"] // 2, dtype=torch.float64, device="cuda")
        turn = torch.zeros(s.count, dtype=torch.float64, device="cuda")
        turn[:s.rows] = at.double()
        turn = turn[:, None] * 500000.0 ** (-2.0 * j / case["rotated"])
        s.angles = torch.stack([torch.cos(turn), torch.sin(turn)], -1).float()
        # One row of q | k | v products per token.
        qkv = _normal((s.count, heads + 2 * kv_heads, width), 7 * seed)
        qkv[:, heads:heads + kv_heads] *= s.spread[0, :, 0]
        qkv[:, heads + kv_heads:] *= s.spread[1, :, 0]
        s.qkv = qkv.reshape(s.count, -1)
        s.q, s.k, s.v = s.qkv.split([heads * width, kv_heads * width, kv_heads * width], 1)
        s.q_out = torch.zeros((s.count, heads * width), device="cuda")
    else:
        # Scores with a standard deviation of 2 under the 1 / sqrt(width) scale.
        s.q = _normal((s.count, heads * width), 7 * seed)
    if case["op"] in ("store", "load"):
        s.k_rows = torch.zeros((s.count, kv_heads * width), device="cuda")
        s.v_rows = torch.zeros_like(s.k_rows)
    s.out = torch.full((s.count, heads * width), 0.25, device="cuda")
    s.scale = 1.0 / math.sqrt(width)
    return s


# ---- the plain forms ------------------------------------------------------

def _quantise(x):
    """(codes 0 .. 15, fp16 steps) of blocks of 32 along the last axis of x: the element of the largest magnitude (of
    two the negative one) is -8 steps."""
    b = x.unflatten(-1, (-1, BLOCK))
    low, high = b.amin(-1), b.amax(-1)
    m = torch.where(-low >= high, low, high)
    step = (m * -0.125).bfloat16().float().clamp(-MOST, MOST).half()
    wide = step.double()[..., None]
    code = torch.where(wide == 0, 0.0, torch.round(b.double() / wide)).clamp(-8, 7) + 8
    return code.flatten(-2).to(torch.uint8), step


def _pack(codes, kind):
    """[pages][heads][tokens][width] codes as the cache lays them out."""
    p, h, t, w = codes.shape
    if kind == 0:
        # 8 elements in a word, the even ones in its low half.
        n = codes.view(p, h, t, w // BLOCK, 4, 4, 2).transpose(5, 6).reshape(p, h, t, w // BLOCK, 16, 2)
        return (n[..., 0] | n[..., 1] << 4).transpose(2, 3).contiguous()
    n = codes.view(p, h, t // 8, 8, w // 4, 2, 2)
    return (n[..., 0] | n[..., 1] << 4).transpose(3, 4).contiguous()


def _unpack(packed, kind):
    """The codes [pages][heads][tokens][width] again."""
    if kind == 0:
        p, h, blocks, t = packed.shape[:4]
        n = torch.stack([packed & 15, packed >> 4], -1).transpose(2, 3)
        return n.reshape(p, h, t, blocks, 4, 2, 4).transpose(5, 6).reshape(p, h, t, blocks * BLOCK)
    p, h, granules, quads = packed.shape[:4]
    n = torch.stack([packed & 15, packed >> 4], -1).transpose(3, 4)
    return n.reshape(p, h, granules * 8, quads * 4)


def _pack_steps(steps, kind):
    """[pages][heads][tokens][blocks] steps as the cache lays them out."""
    p, h, t, b = steps.shape
    if kind == 0:
        return steps.view(p, h, t // 16, 4, 4, b).permute(0, 1, 2, 5, 4, 3).contiguous()
    return steps.transpose(2, 3).contiguous()


def _unpack_steps(packed, kind):
    if kind == 0:
        p, h, granules, b = packed.shape[:4]
        return packed.permute(0, 1, 2, 5, 4, 3).reshape(p, h, granules * 16, b)
    return packed.transpose(2, 3)


def _values(s, pages, kind):
    """fp32 rows [..][heads][tokens][width] of the cache's pages."""
    shape = pages.shape
    codes = _unpack(s.codes[kind][pages.flatten()], kind)
    steps = _unpack_steps(s.steps[kind][pages.flatten()], kind)
    x = (codes.unflatten(-1, (-1, BLOCK)).float() - 8) * steps.float()[..., None]
    return x.flatten(-2).unflatten(0, shape)


def _plain_rotate(case, x, angles, double=False):
    """Rotated rows of heads; in 64 bits where the result is next to be rounded to a code."""
    n, width, rotated = x.shape[0], case["width"], case["rotated"]
    y = x.reshape(n, -1, width).to(torch.float64 if double else torch.float32).clone()
    c, d = (angles[:, None, :, i].to(y.dtype) for i in range(2))
    head = y[..., :rotated]
    a, b = (head[..., 0::2], head[..., 1::2]) if case["layout"] == INTERLEAVED else head.split(rotated // 2, -1)
    u, w = a * c - b * d, a * d + b * c
    y[..., :rotated] = torch.stack([u, w], -1).flatten(-2) if case["layout"] == INTERLEAVED else torch.cat([u, w], -1)
    return y.float().reshape(n, -1)


def _plain_store(s, kind, x):
    """Rows x of the live slots into one of the two caches, element by element."""
    case, page, width = s.case, s.case["page"], s.case["width"]
    slots = s.slots[:s.rows].long()
    codes, steps = _quantise(x[:s.rows].reshape(s.rows, case["kv_heads"], width))
    at, t = slots // page, slots % page
    if kind == 0:
        n = codes.view(s.rows, -1, width // BLOCK, 4, 4, 2).transpose(4, 5).reshape(s.rows, -1, width // BLOCK, 16, 2)
        s.codes[0][at, :, :, t] = n[..., 0] | n[..., 1] << 4
        s.steps[0][at, :, t // 16, :, t % 4, t % 16 // 4] = steps
    else:
        n = codes.view(s.rows, -1, width // 4, 2, 2)
        s.codes[1][at, :, t // 8, :, t % 8] = n[..., 0] | n[..., 1] << 4
        s.steps[1][at, :, :, t] = steps


def _plain_load(s, kind):
    case, page, slots = s.case, s.case["page"], s.slots[:s.rows].long()
    at, t = slots // page, slots % page
    if kind == 0:
        b = s.codes[0][at, :, :, t]
        n = torch.stack([b & 15, b >> 4], -1).unflatten(3, (4, 4)).flatten(4).unflatten(4, (2, 4)).transpose(4, 5)
        steps = s.steps[0][at, :, t // 16, :, t % 4, t % 16 // 4]
    else:
        b = s.codes[1][at, :, t // 8, :, t % 8]
        n = torch.stack([b & 15, b >> 4], -1)
        steps = s.steps[1][at, :, :, t]
    x = n.reshape(s.rows, case["kv_heads"], -1, BLOCK).float() - 8
    return (x * steps.float()[..., None]).reshape(s.rows, -1)


def _plain_attention(s, q):
    case, page = s.case, s.case["page"]
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    group, most, pages = heads // kv_heads, s.most, s.stride - 1
    lengths, starts = s.new_lengths.long(), s.starts.long()
    table = s.table[:, :pages].long()
    keys, values = (_values(s, table.clamp(min=0), kind).transpose(1, 2).reshape(s.requests, kv_heads, pages * page,
                                                                                 width) for kind in range(2))
    row = torch.arange(most, device=q.device)[None]
    counts = (starts[1:] - starts[:-1])[:, None]
    source = torch.where(row < counts, starts[:-1, None] + row, s.count - 1)
    position = lengths[:, None] - counts + row
    x = q[source].reshape(s.requests, most, kv_heads, group, width).transpose(1, 2).flatten(2, 3)
    scores = (x @ keys.transpose(2, 3).contiguous()) * s.scale
    t = torch.arange(pages * page, device=q.device)
    seen = (t <= position[..., None]) & (table.repeat_interleave(page, 1) >= 0)[:, None]
    if case["window"]:
        seen &= t > position[..., None] - case["window"]
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(3, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(3, keepdim=True)
    o = torch.where(total > 0, (p @ values) / total, 0.0)
    o = o.unflatten(2, (most, group)).transpose(1, 2).reshape(s.requests * most, heads * width)
    live = (row < counts).reshape(-1)
    s.out[source.reshape(-1)[live]] = o[live]
    return s.out


def _plain_answers(s):
    c, x, t = s.case, s.logits, s.tokens.long()[:, None]
    if s.mask is not None:
        off = (s.mask[:, None] >> torch.arange(32, dtype=torch.int32, device=x.device)) & 1
        x = x.masked_fill(off.reshape(-1)[None, :x.shape[1]].bool(), -math.inf)
    top = x.amax(1, keepdim=True)
    z = (x - top) * c["scale"]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    logprob = (z.gather(1, t) - lse)[:, 0]
    entropy = (lse - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total)[:, 0]
    given = x.gather(1, t)
    index = torch.arange(x.shape[1], device=x.device)
    rank = ((x > given) | ((x == given) & (index < t))).sum(1).to(torch.int32)
    order = s.top_ids.long()   # none asked for
    if c["top"]:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    return {"logprob": logprob, "rank": rank, "entropy": entropy, "ids": order.to(torch.int32),
            "logprobs": z.gather(1, order) - lse}


# ---- one pass -------------------------------------------------------------

_library = None


def _kernels():
    global _library
    if _library is None:
        from fyodor_amd.hip import Kernels
        _library = Kernels()
    return _library


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(s):
    return _kernels().kv4(s.codes[0].data_ptr(), s.codes[1].data_ptr(), s.steps[0].data_ptr(), s.steps[1].data_ptr(),
                          s.page_count, s.case["page"], s.case["kv_heads"], s.case["width"])


def _store(s):
    c = s.case
    if not own:
        _plain_store(s, 0, _plain_rotate(c, s.k, s.angles, double=True))
        _plain_store(s, 1, s.v)
        return _plain_rotate(c, s.q, s.angles)
    _kernels().kv4_store(_cache(s), s.slots.data_ptr(), s.count, s.k.data_ptr(), s.qkv.stride(0), s.v.data_ptr(),
                         s.qkv.stride(0), s.angles.data_ptr(), c["rotated"], c["layout"], s.q.data_ptr(),
                         s.qkv.stride(0), s.q_out.data_ptr(), s.q_out.stride(0), c["heads"], _stream())
    return s.q_out


def _load(s):
    if not own:
        return _plain_load(s, 0), _plain_load(s, 1)
    _kernels().kv4_load(_cache(s), s.slots.data_ptr(), s.count, s.k_rows.data_ptr(), s.k_rows.stride(0),
                        s.v_rows.data_ptr(), s.v_rows.stride(0), _stream())
    return s.k_rows[:s.rows], s.v_rows[:s.rows]


def _attention(s, q):
    if not own:
        return _plain_attention(s, q)
    _kernels().kv4_attention(_cache(s), q.data_ptr(), q.stride(0), s.out.data_ptr(), s.out.stride(0), s.count,
                             s.starts.data_ptr(), s.new_lengths.data_ptr(), s.table.data_ptr(), s.stride, s.requests,
                             s.most, s.longest, s.case["heads"], s.case["window"], s.scale, s.scratch.data_ptr(),
                             SCRATCH, _stream())
    return s.out


def _answers(s):
    if not own:
        return _plain_answers(s)
    c = s.case
    _kernels().logprobs(s.logits.data_ptr(), s.logits.stride(0), c["vocabulary"], c["rows"],
                        s.mask.data_ptr() if s.mask is not None else 0, c["scale"], s.tokens.data_ptr(),
                        s.logprob.data_ptr(), s.rank.data_ptr(), s.entropy.data_ptr(), c["top"],
                        s.top_ids.data_ptr() if c["top"] else 0, s.top_logprobs.data_ptr() if c["top"] else 0,
                        s.scratch.data_ptr(), SCRATCH, _stream())
    return {"logprob": s.logprob, "rank": s.rank, "entropy": s.entropy, "ids": s.top_ids, "logprobs": s.top_logprobs}


def run(s):
    op = s.case["op"]
    if op == "logprobs":
        return _answers(s)
    if op == "load":
        k, v = _load(s)
        return {"k": k, "v": v}
    if op == "attention":
        return _attention(s, s.q)
    q = _store(s)
    if op == "store":
        k, v = _load(s)
        return {"q": q[:s.rows], "k": k, "v": v}
    out = _attention(s, q)
    return {"out": out, "answers": _answers(s)}


# ---- what a pass cannot do without ----------------------------------------

def _spans(case, lengths, counts):
    """(positions read per request, (row, position) pairs) of its attention."""
    span = pairs = 0
    for n, c in zip(lengths, counts):
        first = n - c
        seen = [min(p + 1, case["window"] or p + 1) for p in range(first, n)]
        pairs += sum(seen)
        span += n - max(0, first + 1 - seen[0]) if c else 0
    return span, pairs


def work(case):
    # Codes of 4 bits and a step of 16 for 32 of them.
    held = 0.5 + 2 / BLOCK
    n, top = case["vocabulary"], case["top"]
    answers = {"bytes": case["rows"] * (4 * n + 16 + 8 * top) + (n / 8 if case["mask"] else 0),
               "flops": 5 * case["rows"] * n}
    if case["op"] == "logprobs":
        return answers
    lengths, counts = _batch(case)
    rows, rotated = sum(counts), case["rotated"]
    q, kv = case["heads"] * case["width"], case["kv_heads"] * case["width"]
    store = {"bytes": rows * (4 * (2 * q + 2 * kv + rotated + 1) + 2 * kv * held),
             "flops": rows * (6 * kv + 3 * rotated * case["heads"])}
    load = {"bytes": rows * (4 + kv * 2 * (held + 4)), "flops": rows * kv * 2}
    span, pairs = _spans(case, lengths, counts)
    attention = {"bytes": 8 * rows * q + 2 * span * kv * held, "flops": 4 * q * pairs}
    parts = {"store": [store, load], "load": [load], "attention": [attention],
             "step": [store, attention, answers]}[case["op"]]
    return {k: sum(p[k] for p in parts) for k in ("bytes", "flops")}


# ---- the same from the definitions, in 64 bits ----------------------------

def _exact_rotate(case, x, angles):
    """x [rows][heads][width] rotated by fp32 (cos, sin)."""
    x, half = x.double(), case["rotated"] // 2
    turn = torch.complex(angles[..., 0].double(), angles[..., 1].double())
    first = torch.arange(half, device=x.device) * (2 if case["layout"] == INTERLEAVED else 1)
    second = first + (1 if case["layout"] == INTERLEAVED else half)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_held(x):
    """What the cache holds of rows x [..][width] (fp32), in 64 bits."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    m = torch.where((b == -top).any(-1, keepdim=True), -top, top)
    # The step to 8 bits: a mantissa from 128 to 256, ties to even.
    fraction, exponent = torch.frexp(m / -8)
    step = torch.ldexp(torch.round(fraction * 256), exponent - 8).clamp(-MOST, MOST).half().double()
    n = torch.round(b / torch.where(step == 0, 1.0, step))
    return (n.clamp(-8, 7) * step).flatten(-2)


def _exact_cache(s, kind):
    """[page][head][token][width] of what the cache holds, each value from its own place."""
    case = s.case
    page, width, kv_heads = case["page"], case["width"], case["kv_heads"]
    t, d = torch.arange(page, device="cuda")[:, None], torch.arange(width, device="cuda")[None]
    if kind == 0:
        e = d % 8
        nibble = ((d // 32 * page + t) * 16 + d % 32 // 8 * 4) * 2 + e % 2 * 4 + e // 2
        step = (t // 16 * (width // 32) + d // 32) * 16 + t % 4 * 4 + t % 16 // 4
    else:
        nibble = ((t // 8 * (width // 4) + d // 4) * 8 + t % 8) * 4 + d % 4
        step = d // 32 * page + t
    flat = s.codes[kind].reshape(s.page_count, kv_heads, -1)
    code = (flat[:, :, nibble // 2] >> (4 * (nibble % 2)).to(torch.uint8)) & 15
    return (code.double() - 8) * s.steps[kind].reshape(s.page_count, kv_heads, -1)[:, :, step].double()


def _exact_attention(case, s, q, keys, values):
    out = torch.full((s.count, case["heads"], case["width"]), 0.25, dtype=torch.float64, device="cuda")
    group, at = case["heads"] // case["kv_heads"], 0
    for r, (n, c) in enumerate(zip(s.lengths, s.counts)):
        if not c:
            continue
        pages = s.table[r, :-(-n // case["page"])].long()
        position = torch.arange(n - c, n, device="cuda")[:, None]
        t = torch.arange(n, device="cuda")[None]
        hidden = (t > position) | ((t <= position - case["window"]) if case["window"] else (t < 0))
        for h in range(case["kv_heads"]):
            k, v = keys[pages, h].flatten(0, 1)[:n], values[pages, h].flatten(0, 1)[:n]
            for g in range(h * group, (h + 1) * group):
                scores = (q[at:at + c, g] @ k.T) * s.scale
                out[at:at + c, g] = torch.softmax(scores.masked_fill(hidden, -math.inf), 1) @ v
        at += c
    return out.flatten(1)


def _exact_answers(s):
    c, result = s.case, {"logprob": [], "entropy": [], "logprobs": []}
    for begin in range(0, c["rows"], 256):
        x = s.logits[begin:begin + 256].double()
        if s.mask is not None:
            i = torch.arange(x.shape[1], device="cuda")
            x[:, (s.mask[i // 32].long() >> (i % 32) & 1).bool()] = -math.inf
        p = torch.log_softmax(x * c["scale"], 1)
        result["logprob"].append(p.gather(1, s.tokens[begin:begin + 256].long()[:, None])[:, 0])
        result["entropy"].append(-(p.exp() * p.clamp(min=-1e300)).sum(1))
        result["logprobs"].append(p.topk(c["top"], 1).values)
    return dict({k: torch.cat(v) for k, v in result.items()}, rank=None, ids=None)


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "logprobs":
        return {k: _exact_answers(s)[k] for k in ("logprob", "rank", "entropy", "ids", "logprobs")}
    if op == "attention":
        keys, values = (_exact_cache(s, kind) for kind in range(2))
        return _exact_attention(case, s, s.q.reshape(s.count, -1, case["width"]).double(), keys, values)
    at, t = s.slots[:s.rows].long() // case["page"], s.slots[:s.rows].long() % case["page"]
    if op == "load":
        return {k: _exact_cache(s, kind)[at, :, t].flatten(1) for kind, k in enumerate("kv")}
    # What is held stands for values rotated by fp32 (cos, sin), rounded to fp32.
    rows = (s.rows, -1, case["width"])
    k = _exact_held(_exact_rotate(case, s.k[:s.rows].reshape(rows), s.angles[:s.rows]).float())
    v = _exact_held(s.v[:s.rows].reshape(rows))
    q = _exact_rotate(case, s.q[:s.rows].reshape(rows), s.angles[:s.rows])
    if op == "store":
        return {"q": q.flatten(1), "k": k.flatten(1), "v": v.flatten(1)}
    keys, values = (_exact_cache(s, kind) for kind in range(2))
    keys[at, :, t], values[at, :, t] = k, v
    answers = _exact_answers(s)
    return {"out": _exact_attention(case, s, q, keys, values),
            "answers": {k: answers[k] for k in ("logprob", "rank", "entropy", "ids", "logprobs")}}
