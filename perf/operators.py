"""The operators of a step that serves many requests over one paged 8-bit cache, as measurable cases.

A case is one pass through

``pages``      ``page_step``: block tables, rows, positions and slots of a batch from its request lengths;
``rope``       ``rope_angles`` and ``rope``: the rotary step of q and k rows;
``store``      ``kv8_store`` (rotating q and k) and ``kv8_load`` of every row held in the pages it touched;
``attention``  ``kv8_attention``: causal attention of the batch's rows over their requests' pages;
``step``       all of them in turn, as one layer of a serving step runs them.

Head shapes and page sizes are the ones this repository's decoders and tests use, and their neighbours. Requests'
lengths and their new tokens come from the case alone (``_batch``); values from the seed. Activations are normal with
a per-channel spread, as a decoder's normalized residual has.
"""
import math
import random

import torch

own = False

INTERLEAVED, HALVES = 0, 1
SCRATCH = 64 << 20   # attention scratch a serving program keeps
FLOOR = 2.0 ** -100  # the smallest scale of a page


def _case(name, op, shape, page, requests, shortest, longest, prompts=0, chunk=0, single=1, idle=0, window=0,
          rotated=0, layout=INTERLEAVED, scaled=1.0, mix=1, turnover=False):
    heads, kv_heads, width = shape
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "width": width, "page": page, "requests": requests,
         "shortest": shortest, "longest": longest, "prompts": prompts, "chunk": chunk, "single": single, "idle": idle,
         "window": window, "rotated": rotated or width, "layout": layout, "scaled": scaled, "mix": mix,
         "turnover": turnover}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decode token for each of 64 running requests: where it goes.
        _case("pages-decode", "pages", (32, 8, 128), 64, 64, 200, 4096, mix=1),
        # A finished batch's pages go back and 193 prompts take them: the
        # largest bookkeeping of a step.
        _case("pages-turnover", "pages", (32, 8, 128), 16, 193, 16, 512, prompts=193, chunk=512, mix=2, turnover=True),
        # The rotary step of 16 decode tokens: bound by its launches.
        _case("rope-decode", "rope", (32, 8, 128), 64, 16, 500, 4096, mix=3),
        # A prompt chunk far into a long context, a quarter of wide heads
        # rotated with stretched frequencies.
        _case("rope-long", "rope", (16, 8, 256), 64, 1, 120001, 120001, prompts=1, chunk=2049, rotated=64,
              layout=HALVES, scaled=8.0, mix=4),
        # One decode token for each of 61 requests into their last pages.
        _case("store-decode", "store", (32, 8, 128), 64, 61, 100, 4096, mix=5),
        # Three prompts of odd lengths, one of them going on inside a page.
        _case("store-prompt", "store", (32, 4, 64), 32, 3, 400, 1333, prompts=3, chunk=801, layout=HALVES, mix=6),
        # The smallest batch over the longest cache: one token.
        _case("attend-long", "attention", (32, 8, 128), 64, 1, 32768, 32768, mix=7),
        # Steady decoding of 64 requests of every length.
        _case("attend-decode", "attention", (32, 8, 128), 64, 64, 500, 8192, mix=8),
        # Draft tokens of eight requests checked at once, small heads and pages.
        _case("attend-verify", "attention", (32, 4, 64), 16, 8, 300, 2048, single=5, mix=9),
        # The largest call: a 1024-token prompt chunk at the end of 8192 positions.
        _case("attend-prompt", "attention", (32, 8, 128), 64, 1, 8192, 8192, prompts=1, chunk=1024, mix=10),
        # Prompts of mixed lengths in wide heads with a local window, one
        # request of the batch idle.
        _case("attend-window", "attention", (16, 8, 256), 32, 6, 300, 3001, prompts=4, chunk=700, idle=1, window=1024,
              mix=11),
        # A whole layer's step: two prompts join 22 requests that decode.
        _case("serve-step", "step", (32, 8, 128), 64, 24, 64, 2048, prompts=2, chunk=256, mix=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choices(["pages", "rope", "store", "attention", "step"], [1, 1, 2, 5, 1])[0]
    shape = rng.choice([(32, 8, 128), (32, 4, 64), (16, 8, 256), (32, 32, 128), (8, 1, 512), (20, 4, 128), (6, 2, 64)])
    page = rng.choice([16, 32, 64, 128])
    layout, scaled = rng.choice([INTERLEAVED, HALVES]), rng.choice([1.0, 1.0, 4.0, 8.0])
    rotated = rng.choice([shape[2], shape[2] // 2, shape[2] // 4])
    window, mix = rng.choice([0, 0, 0, 512, 1000]), rng.randrange(1 << 20)
    requests = _log(rng, 1, 64)
    longest = _log(rng, 64, 32768)
    if op == "pages":
        requests, longest = _log(rng, 1, 200), _log(rng, 16, 512)
        return _case(None, op, shape, page, requests, 1, longest, prompts=rng.choice([0, requests]), chunk=longest,
                     mix=mix, turnover=rng.random() < 0.5)
    prompts = rng.choice([0, 0, 1, min(requests, 4)])
    chunk = min(longest, _log(rng, 9, 700)) // max(1, prompts // 2) or 1
    single = rng.choice([1, 1, 1, rng.randint(2, 33)])
    if prompts or single > 1:
        longest = min(longest, 4096)
        requests = min(requests, 24)
    idle = rng.randint(0, 1) if requests > prompts + 1 else 0
    share = rng.randint(1, 30)
    while True:
        longest = max(longest, single, chunk if prompts else 1)
        case = _case(None, op, shape, page, requests, max(1, longest // share), longest, prompts, chunk, single, idle,
                     window if op == "attention" else 0, rotated, layout, scaled, mix)
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


def _frequencies(case):
    """fp32 frequencies; stretched ones keep the pairs that turn often within 8192 positions."""
    j = torch.arange(case["rotated"] // 2, dtype=torch.float64)
    f = 500000.0 ** (-2.0 * j / case["rotated"])
    if case["scaled"] > 1:
        keep = ((8192 * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        f = (1 - keep) * f / case["scaled"] + keep * f
    return f.float().cuda()


def _pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


class State:
    """What a serving program holds before the call: the cache, its page tables, the batch and its buffers."""


def prepare(case, seed):
    s = State()
    s.case, s.lengths, s.counts = case, *_batch(case)
    page, heads, kv_heads, width = case["page"], case["heads"], case["kv_heads"], case["width"]
    s.need = _pages_of(s.lengths, page)
    s.rows = sum(s.counts)
    s.count = s.rows + 3 if case["op"] != "rope" else s.rows   # a batch padded past its last row
    s.requests, s.stride = case["requests"], max(s.need) + 1
    s.page_count = sum(s.need) + 2
    s.most, s.longest = max(s.counts), max(s.lengths)
    g = torch.Generator(device="cuda").manual_seed(5 * seed + 4)
    order = torch.randperm(s.page_count, generator=g, device="cuda").to(torch.int32)
    # What the requests held before their new tokens (all of it where the
    # case does not run the page step itself).
    own_pages = case["op"] in ("pages", "step")
    before = _pages_of([n - c for n, c in zip(s.lengths, s.counts)], page) if own_pages else s.need
    if case["turnover"]:
        before = s.need
    s.table = torch.full((s.requests, s.stride), -1, dtype=torch.int32, device="cuda")
    taken = 0
    for r, n in enumerate(before):
        s.table[r, :n] = order[taken:taken + n]
        taken += n
    s.held = _ints(before)
    s.free_pages = torch.cat([order[taken:], torch.full((taken,), -1, dtype=torch.int32, device="cuda")])
    s.free_count = _ints([s.page_count - taken, 0])
    s.new_lengths, s.new_counts = _ints(s.lengths), _ints(s.counts)
    s.none = torch.zeros_like(s.new_lengths)
    s.starts = torch.zeros(s.requests + 1, dtype=torch.int32, device="cuda")
    s.positions = torch.full((s.count,), -1, dtype=torch.int32, device="cuda")
    s.slots = torch.full((s.count,), -1, dtype=torch.int32, device="cuda")
    if not own_pages:
        starts, at = [0], []
        for n, c in zip(s.lengths, s.counts):
            starts.append(starts[-1] + c)
            at += range(n - c, n)
        s.starts.copy_(_ints(starts))
        s.positions[:s.rows] = _ints(at)
        request = torch.repeat_interleave(torch.arange(s.requests, device="cuda"), s.new_counts.long())
        p = s.positions[:s.rows].long()
        s.slots[:s.rows] = s.table[request, p // page] * page + p % page
    if case["op"] == "pages":
        return s
    spread = torch.exp(0.5 * _normal((2, kv_heads, 1, width), 5 * seed + 3))
    if case["op"] != "attention":
        s.frequencies = _frequencies(case)
        s.magnitude = 1.0 if case["scaled"] == 1 else 0.1 * math.log(case["scaled"]) + 1.0
        s.angles = torch.empty((s.count, case["rotated"] // 2, 2), device="cuda")
        if case["op"] == "store":
            s.angles.copy_(_plain_angles(s))
        # One row of q | k | v products per token.
        qkv = _normal((s.count, heads + 2 * kv_heads, width), 5 * seed)
        qkv[:, heads:heads + kv_heads] *= spread[0, :, 0]
        qkv[:, heads + kv_heads:] *= spread[1, :, 0]
        s.qkv = qkv.reshape(s.count, -1)
        s.q, s.k, s.v = s.qkv.split([heads * width, kv_heads * width, kv_heads * width], 1)
        s.q_out, s.k_out = torch.zeros((s.count, heads * width), device="cuda"), torch.zeros_like(s.k)
    else:
        # Scores with a standard deviation of 2 under the 1 / sqrt(width) scale.
        s.q = _normal((s.count, heads * width), 5 * seed)
    if case["op"] == "rope":
        return s
    s.codes, s.scales = [], []
    for kind in range(2):
        x = _normal((s.page_count, kv_heads, page, width), 5 * seed + 1 + kind) * spread[kind]
        scale = (x.abs().amax((2, 3)) / 127).clamp(min=FLOOR)
        c = torch.round(x / scale[:, :, None, None]).to(torch.int8)
        c = c.view(s.page_count, kv_heads, page, width // 16, 16).transpose(2, 3) if kind == 0 else \
            c.view(s.page_count, kv_heads, page // 16, 16, width).transpose(3, 4)
        s.codes.append(c.contiguous())
        s.scales.append(scale.contiguous())
    if case["op"] == "store":
        # Every row held in the pages that the call touches.
        s.read = torch.cat([s.table[r, torch.arange((n - c) // page * page, n, device="cuda") // page] * page +
                            torch.arange(n - (n - c) // page * page, device="cuda") % page
                            for r, (n, c) in enumerate(zip(s.lengths, s.counts))]).to(torch.int32)
        s.k_rows = torch.empty((s.read.numel(), kv_heads * width), device="cuda")
        s.v_rows = torch.empty_like(s.k_rows)
    s.out = torch.full((s.count, heads * width), 0.25, device="cuda")
    s.scratch = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    s.scale = 1.0 / math.sqrt(width)
    return s


# ---- the plain forms ------------------------------------------------------

def _plain_pages(s, lengths, counts):
    page, stride, dev = s.case["page"], s.stride, s.table.device
    lengths, counts = lengths.long(), counts.long()
    need, held = (lengths + page - 1) // page, s.held.long()
    index = torch.arange(stride, device=dev)[None]
    # Pages past the need go back on the stack, in request order.
    back = (index >= need[:, None]) & (index < held[:, None])
    place = s.free_count[0] + torch.cumsum(back.reshape(-1).long(), 0) - 1
    stack = torch.cat([s.free_pages, s.free_pages.new_zeros(1)])
    stack[torch.where(back.reshape(-1), place, stack.numel() - 1)] = s.table.reshape(-1)
    free = s.free_count[0] + back.sum()
    s.table.masked_fill_(back, -1)
    held = torch.minimum(held, need)
    # Requests that grow take pages from its top, in request order.
    grow = need - held
    grow = torch.where((torch.cumsum(grow, 0) <= free), grow, 0)
    taken = torch.cumsum(grow, 0) - grow
    fresh = (index >= held[:, None]) & (index < (held + grow)[:, None])
    source = (free - 1 - taken[:, None] - (index - held[:, None])).clamp(0, stack.numel() - 1)
    s.table.copy_(torch.where(fresh, stack[source], s.table))
    s.free_pages.copy_(stack[:-1])
    s.free_count.copy_(torch.stack([free - grow.sum(), (need > held + grow).sum()]))
    s.held.copy_(held + grow)
    # Rows.
    s.starts[1:] = torch.cumsum(counts, 0)
    row = torch.arange(s.count, device=dev)
    request = torch.searchsorted(s.starts[1:].long(), row, right=True).clamp(max=s.requests - 1)
    position = lengths[request] - counts[request] + row - s.starts[request]
    live = row < s.starts[-1]
    known = live & (position < s.held[request] * page) & (position >= 0)
    at = s.table[request, (position // page).clamp(0, stride - 1)]
    s.positions.copy_(torch.where(live, position, -1))
    s.slots.copy_(torch.where(known, at * page + position % page, -1))
    return {"table": s.table, "held": s.held, "free_pages": s.free_pages, "free_count": s.free_count,
            "starts": s.starts, "positions": s.positions, "slots": s.slots}


def _plain_angles(s):
    a = s.positions.double()[:, None] * s.frequencies.double()
    return (torch.stack([torch.cos(a), torch.sin(a)], -1) * s.magnitude).float()


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


def _token_order(codes, kind):
    """[pages][heads][tokens][width] of codes as the cache lays them out."""
    p, h = codes.shape[:2]
    return codes.transpose(2, 3).flatten(3) if kind == 0 else codes.transpose(3, 4).flatten(2, 3)


def _plain_store(s, kind, x):
    """Rows x of the live slots into the pages of one of the two caches."""
    case, page, codes, scales = s.case, s.case["page"], s.codes[kind], s.scales[kind]
    kv_heads, width = case["kv_heads"], case["width"]
    slots = s.slots[:s.rows].long()
    x = x[:s.rows].reshape(-1, kv_heads, width)
    touched, which = torch.unique(slots // page, return_inverse=True)
    top = x.abs().amax(2)
    amax = torch.zeros((touched.numel(), kv_heads), device=x.device)
    amax.scatter_reduce_(0, which[:, None].expand(-1, kv_heads), top, "amax")
    wanted = (amax / 127).clamp(min=FLOOR)
    first = torch.zeros(touched.numel(), device=x.device)
    first.scatter_reduce_(0, which, (slots % page == 0).float(), "amax")
    old = scales[touched]
    grew = (first[:, None] == 0) & (wanted > old)
    scale = torch.where(first[:, None] > 0, wanted, torch.maximum(old, wanted))
    ratio = old.double() / scale.double()
    held = codes[touched]
    held = torch.where(grew[..., None, None, None],
                       torch.round(held.double() * old.double()[..., None, None, None] /
                                   scale.double()[..., None, None, None]).clamp(-127, 127).to(torch.int8), held)
    c = torch.round(x.double() / scale[which].double()[..., None]).clamp(-127, 127).to(torch.int8)
    at = slots % page
    if kind == 0:
        held[which, :, :, at] = c.reshape(-1, kv_heads, width // 16, 16)
    else:
        held[which, :, at // 16, :, at % 16] = c
    codes[touched] = held
    scales[touched] = scale


def _plain_load(s, kind):
    page = s.case["page"]
    slots = s.read.long()
    rows = _token_order(s.codes[kind], kind)[slots // page, :, slots % page]
    return (rows.float() * s.scales[kind][slots // page][..., None]).flatten(1)


def _plain_attention(s, q):
    case, page = s.case, s.case["page"]
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    group, most, pages = heads // kv_heads, s.most, s.stride - 1
    lengths, starts = s.new_lengths.long(), s.starts.long()
    table = s.table[:, :pages].long()
    cache = []
    for kind in range(2):
        at = table.clamp(min=0)
        x = _token_order(s.codes[kind][at].flatten(0, 1), kind).unflatten(0, at.shape).float()
        x = x * s.scales[kind][at][..., None, None]
        cache.append(x.transpose(1, 2).reshape(s.requests, kv_heads, pages * page, width))
    row = torch.arange(most, device=q.device)[None]
    counts = (starts[1:] - starts[:-1])[:, None]
    source = torch.where(row < counts, starts[:-1, None] + row, s.count - 1)
    position = lengths[:, None] - counts + row
    x = q[source].reshape(s.requests, most, kv_heads, group, width).transpose(1, 2).flatten(2, 3)
    scores = (x @ cache[0].transpose(2, 3).contiguous()) * s.scale
    t = torch.arange(pages * page, device=q.device)
    seen = (t <= position[..., None]) & (table.repeat_interleave(page, 1) >= 0)[:, None]
    if case["window"]:
        seen &= t > position[..., None] - case["window"]
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(3, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(3, keepdim=True)
    o = torch.where(total > 0, (p @ cache[1]) / total, 0.0)
    o = o.unflatten(2, (most, group)).transpose(1, 2).reshape(s.requests * most, heads * width)
    live = (row < counts).reshape(-1)
    s.out[source.reshape(-1)[live]] = o[live]
    return s.out


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


def _page_step(s, lengths, counts):
    if not own:
        return _plain_pages(s, lengths, counts)
    _kernels().page_step(lengths.data_ptr(), counts.data_ptr(), s.requests, s.case["page"], s.table.data_ptr(),
                         s.stride, s.held.data_ptr(), s.free_pages.data_ptr(), s.page_count, s.free_count.data_ptr(),
                         s.starts.data_ptr(), s.positions.data_ptr(), s.slots.data_ptr(), s.count, _stream())
    return {"table": s.table, "held": s.held, "free_pages": s.free_pages, "free_count": s.free_count,
            "starts": s.starts, "positions": s.positions, "slots": s.slots}


def _angles(s):
    if not own:
        s.angles.copy_(_plain_angles(s))
    else:
        _kernels().rope_angles(s.positions.data_ptr(), s.count, s.frequencies.data_ptr(), s.case["rotated"],
                               s.magnitude, s.angles.data_ptr(), _stream())
    return s.angles


def _rope(s):
    c = s.case
    if not own:
        return _plain_rotate(c, s.q, s.angles), _plain_rotate(c, s.k, s.angles)
    _kernels().rope(s.q.data_ptr(), s.qkv.stride(0), s.q_out.data_ptr(), s.q_out.stride(0), c["heads"],
                    s.k.data_ptr(), s.qkv.stride(0), s.k_out.data_ptr(), s.k_out.stride(0), c["kv_heads"], c["width"],
                    s.count, s.angles.data_ptr(), c["rotated"], c["layout"], _stream())
    return s.q_out, s.k_out


def _cache(s):
    return _kernels().kv8(s.codes[0].data_ptr(), s.codes[1].data_ptr(), s.scales[0].data_ptr(),
                          s.scales[1].data_ptr(), s.page_count, s.case["page"], s.case["kv_heads"], s.case["width"])


def _store(s):
    c = s.case
    if not own:
        _plain_store(s, 0, _plain_rotate(c, s.k, s.angles, double=True))
        _plain_store(s, 1, s.v)
        return _plain_rotate(c, s.q, s.angles)
    _kernels().kv8_store(_cache(s), s.slots.data_ptr(), s.count, s.k.data_ptr(), s.qkv.stride(0), s.v.data_ptr(),
                         s.qkv.stride(0), s.angles.data_ptr(), c["rotated"], c["layout"], s.q.data_ptr(),
                         s.qkv.stride(0), s.q_out.data_ptr(), s.q_out.stride(0), c["heads"], _stream())
    return s.q_out


def _load(s):
    if not own:
        return _plain_load(s, 0), _plain_load(s, 1)
    _kernels().kv8_load(_cache(s), s.read.data_ptr(), s.read.numel(), s.k_rows.data_ptr(), s.k_rows.stride(0),
                        s.v_rows.data_ptr(), s.v_rows.stride(0), _stream())
    return s.k_rows, s.v_rows


def _attention(s, q):
    if not own:
        return _plain_attention(s, q)
    _kernels().kv8_attention(_cache(s), q.data_ptr(), q.stride(0), s.out.data_ptr(), s.out.stride(0), s.count,
                             s.starts.data_ptr(), s.new_lengths.data_ptr(), s.table.data_ptr(), s.stride, s.requests,
                             s.most, s.longest, s.case["heads"], s.case["window"], s.scale, s.scratch.data_ptr(),
                             SCRATCH, _stream())
    return s.out


def run(s):
    op = s.case["op"]
    if op == "pages":
        if s.case["turnover"]:
            _page_step(s, s.none, s.none)
        return _page_step(s, s.new_lengths, s.new_counts)
    if op == "rope":
        angles = _angles(s)
        q, k = _rope(s)
        return {"angles": angles, "q": q, "k": k}
    if op == "store":
        q = _store(s)
        k, v = _load(s)
        return {"q": q[:s.rows], "k": k, "v": v, "key_scales": s.scales[0], "value_scales": s.scales[1]}
    if op == "attention":
        return _attention(s, s.q)
    pages = _page_step(s, s.new_lengths, s.new_counts)
    angles = _angles(s)
    q = _store(s)
    out = _attention(s, q)
    return {"pages": pages, "angles": angles[:s.rows], "out": out, "key_scales": s.scales[0],
            "value_scales": s.scales[1]}


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
    lengths, counts = _batch(case)
    rows, requests = sum(counts), case["requests"]
    q, kv, rotated = case["heads"] * case["width"], case["kv_heads"] * case["width"], case["rotated"]
    need = _pages_of(lengths, case["page"])
    new = sum(need) - sum(_pages_of([n - c for n, c in zip(lengths, counts)], case["page"]))
    moved = 2 * sum(need) if case["turnover"] else new
    pages = {"bytes": 4 * (5 * requests + 2 * moved + 2 * rows), "flops": requests + rows}
    rope = {"bytes": 4 * rows * (2 * (q + kv) + 1 + rotated), "flops": 3 * rows * rotated * (case["heads"] +
                                                                                              case["kv_heads"])}
    read = sum(n - (n - c) // case["page"] * case["page"] for n, c in zip(lengths, counts))
    store = {"bytes": rows * (4 * (2 * q + 2 * kv + rotated) + 2 * kv),
             "flops": rows * (6 * kv + 3 * rotated * case["heads"])}
    load = {"bytes": read * kv * 2 * (1 + 4), "flops": read * kv * 2}
    span, pairs = _spans(case, lengths, counts)
    attention = {"bytes": 8 * rows * q + 2 * span * kv, "flops": 4 * q * pairs}
    angles = {"bytes": 4 * rows * (1 + rotated), "flops": 4 * rows * rotated}
    parts = {"pages": [pages], "rope": [rope], "store": [store, load], "attention": [attention],
             "step": [pages, angles, store, attention]}[case["op"]]
    return {k: sum(p[k] for p in parts) for k in ("bytes", "flops")}


# ---- the same from the definitions, in 64 bits ----------------------------

def _exact_rotate(case, x, positions, frequencies, magnitude, angles=None):
    """x [rows][heads][width] rotated; by fp32 (cos, sin) where they are given."""
    x, half = x.double(), case["rotated"] // 2
    if angles is None:
        phase = positions.double()[:, None] * frequencies.double()
        turn = torch.complex(torch.cos(phase), torch.sin(phase)) * magnitude
    else:
        turn = torch.complex(angles[..., 0].double(), angles[..., 1].double())
    first = torch.arange(half, device=x.device) * (2 if case["layout"] == INTERLEAVED else 1)
    second = first + (1 if case["layout"] == INTERLEAVED else half)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_cache(case, codes, scales, kind):
    """[page, head] -> the values of its rows [tokens][width] in 64 bits, as a tensor."""
    p, h, width, page = codes.shape[0], case["kv_heads"], case["width"], case["page"]
    t, d = torch.arange(page, device="cuda")[:, None], torch.arange(width, device="cuda")[None]
    place = (d // 16 * page + t) * 16 + d % 16 if kind == 0 else (t // 16 * width + d) * 16 + t % 16
    return codes.reshape(p, h, -1)[:, :, place].double() * scales.double()[..., None, None]


def _exact_put(case, values, scales, slots, x):
    """Rows x [rows][head][width] (fp32) into the pages' values; scales change with them."""
    page = case["page"]
    i = 0
    slots = slots.tolist()
    while i < len(slots):
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % page:
            j += 1
        p, at, new = slots[i] // page, slots[i] % page, x[i:j].double().transpose(0, 1)
        wanted = (new.abs().amax((1, 2)) / 127).float().clamp(min=FLOOR)
        scale = wanted if at == 0 else torch.maximum(scales[p], wanted)
        kept = torch.round(values[p] / scale.double()[:, None, None])
        values[p] = torch.where((scale == scales[p])[:, None, None], values[p], kept * scale.double()[:, None, None])
        values[p][:, at:at + j - i] = torch.round(new / scale.double()[:, None, None]) * scale.double()[:, None, None]
        scales[p] = scale
        i = j


def _exact_attention(case, s, q, keys, values, table):
    out = torch.full((s.count, case["heads"], case["width"]), 0.25, dtype=torch.float64, device="cuda")
    group, at = case["heads"] // case["kv_heads"], 0
    for r, (n, c) in enumerate(zip(s.lengths, s.counts)):
        if not c:
            continue
        pages = table[r, :s.need[r]].long()
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


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None
    s = prepare(case, seed)
    shape = (s.count, -1, case["width"])
    if op == "rope":
        phase = s.positions.double()[:, None] * s.frequencies.double()
        angles = torch.stack([torch.cos(phase), torch.sin(phase)], -1) * s.magnitude
        q, k = (_exact_rotate(case, x.reshape(shape), s.positions, s.frequencies, s.magnitude).flatten(1)
                for x in (s.q, s.k))
        return {"angles": angles, "q": q, "k": k}
    keys, values = (_exact_cache(case, s.codes[i], s.scales[i], i) for i in range(2))
    if op == "attention":
        return _exact_attention(case, s, s.q.reshape(shape).double(), keys, values, s.table)
    scales = [x.clone() for x in s.scales]
    if op == "step":
        # The tables, held pages and rows as their definition gives them.
        table, stack = s.table.tolist(), s.free_pages.tolist()[:int(s.free_count[0])]
        before, slots, at = s.held.tolist(), [], []
        for r, (n, c) in enumerate(zip(s.lengths, s.counts)):
            for j in range(before[r], s.need[r]):
                table[r][j] = stack.pop()
            at += range(n - c, n)
            slots += [table[r][p // case["page"]] * case["page"] + p % case["page"] for p in range(n - c, n)]
        table, s.slots[:s.rows], s.positions[:s.rows] = _ints(table), _ints(slots), _ints(at)
        phase = s.positions[:s.rows].double()[:, None] * s.frequencies.double()
        angles = torch.stack([torch.cos(phase), torch.sin(phase)], -1) * s.magnitude
    else:
        angles = s.angles[:s.rows]
    # Codes stand for values rotated by fp32 (cos, sin), rounded to fp32.
    live = s.slots[:s.rows]
    rows = (s.rows, -1, case["width"])
    k = _exact_rotate(case, s.k[:s.rows].reshape(rows), None, None, None, angles.float()).float()
    _exact_put(case, keys, scales[0], live, k)
    _exact_put(case, values, scales[1], live, s.v[:s.rows].reshape(rows))
    q = _exact_rotate(case, s.q[:s.rows].reshape(rows), None, None, None, angles.float())
    if op == "store":
        page = case["page"]
        read = s.read.long()
        k_rows, v_rows = (x[read // page, :, read % page].flatten(1) for x in (keys, values))
        return {"q": q.flatten(1), "k": k_rows, "v": v_rows, "key_scales": scales[0].double(),
                "value_scales": scales[1].double()}
    out = _exact_attention(case, s, q, keys, values, table)
    return {"pages": None, "angles": angles, "out": out, "key_scales": scales[0].double(),
            "value_scales": scales[1].double()}
