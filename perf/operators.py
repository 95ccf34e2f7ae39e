"""The paged 4-bit KV cache's operators, as cases that can be timed and compared.

A request's keys and values are held in pages of P tokens, in 4 bits: blocks of 32 features, each feature one of
+-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times the block's power of two.  A block whose largest magnitude is a has the exponent
e = floor(log2 a) - 2, one more where a > 7 * 2^e (half way between the grid's 6 and the next power's 8), kept within
[-125, 125]; a feature takes the nearest value, ties to the even code (codes count the magnitudes from 0).  Codes are
packed two to a byte, the even feature in the low four bits, sign in the highest of the four; a block's scale byte is
e + 127.  For each page and KV head the codes are [P, D/2] bytes and the scales [D/32, P].

The operators: pages, slots and positions of a step from the rows' lengths (`reserve`); quantising new keys and values
into the cache, and reading them back (`append`); the norm and rotation of queries and keys in front of that (`norm`);
attention over the cache (`attention`).  The shapes are those of perf/cases.py: 16 query / 8 KV heads of 128 features,
16 / 4 of 256, 8 / 8 of 64, 32 / 8 of 128.

`counts` and `lengths` are comma-separated texts, one number a row: the new tokens, and the keys after the append.
"""

import math

import torch

own = False

SHAPES = {  # (query heads, KV heads, features, rotated features, what is added to a norm weight)
    "16x8x128": (16, 8, 128, 128, 0.0),
    "16x4x256": (16, 4, 256, 64, 1.0),
    "8x8x64": (8, 8, 64, 64, 0.0),
    "32x8x128": (32, 8, 128, 128, 0.0),
}
EPS = 1e-6
BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _numbers(text):
    return [int(x) for x in str(text).split(",")]


def _text(numbers):
    return ",".join(str(int(n)) for n in numbers)


def _attention(name, shape, page, counts, lengths):
    return {"name": name, "kind": "attention", "shape": shape, "page": page, "counts": _text(counts),
            "lengths": _text(lengths)}


def listed():
    return [
        # The page tables of a decode step of 64 requests: a few rows cross into a new page.
        {"name": "reserve_decode_b64", "kind": "reserve", "rows": 64, "tokens": 1, "page": 64, "pages_per_row": 256},
        # Prompt chunks enter while other requests decode or end: many pages and slots at once.
        {"name": "reserve_prompts_b256", "kind": "reserve", "rows": 256, "tokens": 512, "page": 64,
         "pages_per_row": 512},
        # One new token in each of eight rows.
        {"name": "append_b8_t1", "kind": "append", "shape": "16x8x128", "page": 64, "tokens": 1, "counts": _text([1] * 8)},
        # Prompt chunks of eight rows, 256 features.
        {"name": "append_b8_t512_d256", "kind": "append", "shape": "16x4x256", "page": 128, "tokens": 512,
         "counts": "512,138,422,459,512,298,113,509"},
        # The step in front of the attention for one new token in each of eight rows.
        {"name": "norm_b8_t1", "kind": "norm", "shape": "16x8x128", "page": 64, "tokens": 1, "counts": _text([1] * 8)},
        # The same for prompt chunks, rotating 64 of 256 features.
        {"name": "norm_b8_t512_d256", "kind": "norm", "shape": "16x4x256", "page": 128, "tokens": 512,
         "counts": "512,138,422,459,512,298,113,509"},
        # One request, one new token, a short context: the smallest attention call (latency).
        _attention("decode_b1_l1024", "16x8x128", 64, [1], [1024]),
        # A ragged decode batch of eight requests, log-uniform contexts up to 16384 keys.
        _attention("decode_b8_ragged", "16x8x128", 64, [1] * 8, [13312, 2162, 386, 9459, 1399, 3852, 55, 182]),
        # A full server: 64 requests with long contexts.
        _attention("decode_b64_long", "16x8x128", 128, [1] * 64, [16384 - (r * 5081) % 15000 for r in range(64)]),
        # Six new tokens a row over long contexts: checking drafted tokens; 24 query vectors a KV head.
        _attention("chunk_b8_t6", "32x8x128", 64, [6, 6, 5, 6, 2, 6, 6, 4],
                   [9010, 1203, 4777, 305, 15021, 2650, 640, 6111]),
        # One 512-token chunk of a prompt at offset 1536.
        _attention("prefill_b1_n512", "16x8x128", 64, [512], [2048]),
        # Prompt chunks at long offsets beside requests that decode, 256 features: the largest call.
        _attention("mixed_b8_d256", "16x4x256", 256, [356, 1, 422, 459, 1, 298, 512, 1],
                   [14244, 13896, 2059, 4214, 12262, 14086, 12837, 9315]),
    ]


def _log_uniform(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    most = [max(work(case)[k] for case in listed()) for k in ("bytes", "flops")]
    while True:
        case = _draw_once(rng)
        if all(work(case)[k] <= m for k, m in zip(("bytes", "flops"), most)):
            return case


def _draw_once(rng):
    kind = rng.choice(("reserve", "append", "norm", "attention", "attention", "attention"))
    page = rng.choice((64, 128, 256))
    if kind == "reserve":
        tokens = _log_uniform(rng, 1, 512)
        return {"kind": kind, "rows": _log_uniform(rng, 1, 256), "tokens": tokens, "page": page,
                "pages_per_row": _log_uniform(rng, 1 + -(-tokens // page), 512)}
    shape = rng.choice(tuple(SHAPES))
    if kind in ("append", "norm"):
        rows, tokens = _log_uniform(rng, 1, 8), _log_uniform(rng, 1, 512)
        counts = [rng.randint(0, tokens) if rng.random() < 0.5 else tokens for _ in range(rows)]
        return {"kind": kind, "shape": shape, "page": page, "tokens": tokens, "counts": _text(counts)}
    heads, kv_heads, dim = SHAPES[shape][:3]
    form = rng.choice(("decode", "decode", "chunk", "prefill", "mixed"))
    if form == "decode":
        counts = [1] * _log_uniform(rng, 1, 64)
    elif form == "chunk":
        counts = [rng.randint(1, 8) for _ in range(_log_uniform(rng, 1, 8))]
    elif form == "prefill":
        counts = [_log_uniform(rng, 9, 512) for _ in range(_log_uniform(rng, 1, 4))]
    else:
        counts = [rng.choice((1, _log_uniform(rng, 9, 512))) for _ in range(_log_uniform(rng, 2, 8))]
    lengths = [n + _log_uniform(rng, 1, 16384 - n) - 1 for n in counts]
    return {"kind": kind, "shape": shape, "page": page, "counts": _text(counts), "lengths": _text(lengths)}


# ---- the inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _cache(pages, kv_heads, page, dim):
    codes, scales = (pages, kv_heads, page, dim // 2), (pages, kv_heads, dim // BLOCK, page)
    return [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in (codes, scales, codes, scales)]


def _slots(g, counts, tokens, page):
    """[B, T] slots of each row's new tokens, at the end of a page or across two, -1 for the others; and the pages."""
    need = [-(-(n + page) // page) + 1 for n in counts]
    order = torch.randperm(sum(need), generator=g, device="cuda")
    slots = torch.full((len(counts), tokens), -1, dtype=torch.int64, device="cuda")
    first = 0
    for r, n in enumerate(counts):
        at = torch.arange(n, device="cuda") + (page - 7 if n > 1 else 37 + r)
        slots[r, :n] = order[first + at // page] * page + at % page
        first += need[r]
    return slots, sum(need)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "reserve":
        return _prepare_reserve(case, g)
    heads, kv_heads, dim, rotary, offset = SHAPES[case["shape"]]
    counts, page = _numbers(case["counts"]), case["page"]
    rows = len(counts)
    state = dict(case, dim=dim)
    if case["kind"] == "attention":
        lengths, tokens = _numbers(case["lengths"]), max(counts)
        need = [-(-n // page) for n in lengths]
        total = sum(need)
        table = torch.zeros(rows, max(need), dtype=torch.int32)
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        first = 0
        for r, n in enumerate(need):
            table[r, :n] = order[first: first + n]
            first += n
        cache = _cache(total, kv_heads, page, dim)
        some = max(1, (64 << 20) // (kv_heads * page * dim))
        for first in range(0, total, some):
            for tensor in (0, 2):
                x = _randn(g, min(some, total - first), kv_heads, page, dim)
                codes, exponent = quantise(x.float())
                cache[tensor][first: first + some] = pack(codes)
                cache[tensor + 1][first: first + some] = (exponent + 127).to(torch.uint8).transpose(-1, -2)
        state.update(q=_randn(g, rows, heads, tokens, dim), cache=cache, table=table.cuda(),
                     lengths=torch.tensor([counts, lengths], dtype=torch.int32, device="cuda"),
                     longest=max(lengths), scale=dim ** -0.5)
        return state
    tokens = case["tokens"]
    slots, pages = _slots(g, counts, tokens, page)
    state.update(slots=slots, cache=_cache(pages, kv_heads, page, dim))
    if case["kind"] == "append":
        # The adapters' projections viewed per head: [B, T, H, D] seen as [B, H, T, D].
        state.update(key=_randn(g, rows, tokens, kv_heads, dim).transpose(1, 2),
                     value=_randn(g, rows, tokens, kv_heads, dim).transpose(1, 2))
    else:
        angles = torch.rand(rows, tokens, rotary // 2, generator=g, device="cuda", dtype=torch.float64) * 2 * math.pi
        angles = torch.cat((angles, angles), dim=-1)
        state.update(q=_randn(g, rows, tokens, heads, dim), key=_randn(g, rows, tokens, kv_heads, dim),
                     value=_randn(g, rows, tokens, kv_heads, dim),
                     q_weight=(1 - offset + 0.1 * _randn(g, dim).float()).to(torch.bfloat16),
                     k_weight=(1 - offset + 0.1 * _randn(g, dim).float()).to(torch.bfloat16),
                     cos=angles.cos().to(torch.bfloat16), sin=angles.sin().to(torch.bfloat16), offset=offset)
    return state


def _prepare_reserve(case, g):
    rows, tokens, page, width = case["rows"], case["tokens"], case["page"], case["pages_per_row"]
    integers = lambda high: torch.randint(0, high, (rows,), generator=g, device="cuda")  # noqa: E731
    capacity = width * page
    before = integers(capacity - tokens + 1)
    counts = 1 + integers(tokens)
    fate = integers(16)
    # Most rows go on; one in 16 takes back drafted tokens, one in 16 ends, one in 16 starts, one in 16 waits.
    keep = torch.where(fate == 0, (before - integers(64)).clamp_min(0), before)
    before = torch.where(fate == 2, 0, before)
    keep = torch.where((fate == 1) | (fate == 2), 0, keep)
    counts = torch.where((fate == 1) | (fate == 3), 0, counts)
    after = keep + counts
    held = (before + page - 1) // page
    total = rows * width
    order = torch.randperm(total, generator=g, device="cuda")
    column = torch.arange(width, device="cuda")
    index = (held.cumsum(0) - held)[:, None] + column
    table = torch.where(column < held[:, None], order[index.clamp_max(total - 1)], -1)
    taken = int(held.sum())
    head = int(torch.randint(0, 1 << 40, (1,), generator=g, device="cuda")) * total + taken
    return dict(case, before=before.int(), after=after.int(), counts=counts.int(), table=table.int().contiguous(),
                ring=order.int(), counters=torch.tensor([head, head + total - taken], device="cuda"))


# ---- one pass


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "reserve":
        return reserve_plain(s)
    if s["kind"] == "append":
        written = s["slots"] >= 0
        return [round_trip(x.float(), written).to(torch.bfloat16) for x in (s["key"], s["value"])]
    if s["kind"] == "norm":
        written = s["slots"] >= 0
        q = norm_rope(s["q"], s["q_weight"], s).transpose(1, 2)
        k = norm_rope(s["key"], s["k_weight"], s).transpose(1, 2)
        v = s["value"].float().transpose(1, 2)
        return [q.to(torch.bfloat16), round_trip(k, written).to(torch.bfloat16),
                round_trip(v, written).to(torch.bfloat16)]
    return attention_plain(s)


def _run_own(s):
    from xinfer_amd import paged_kv4 as ops

    if s["kind"] == "reserve":
        lengths, positions, slots, counters = ops.paged_kv_reserve(
            s["before"], s["after"], s["counts"], s["tokens"], s["page"], s["counters"], s["table"], s["ring"])
        return [lengths, positions, slots, counters, s["table"], s["ring"]]
    if s["kind"] == "append":
        ops.append_kv4(s["key"], s["value"], s["slots"], s["cache"])
        return list(ops.read_kv4(s["cache"], s["slots"]))
    if s["kind"] == "norm":
        q = ops.qk_norm_rope_append_kv4(s["q"], s["key"], s["value"], s["q_weight"], s["k_weight"], EPS, s["offset"],
                                        s["cos"], s["sin"], s["slots"], s["cache"])
        return [q, *ops.read_kv4(s["cache"], s["slots"])]
    return ops.paged_attention_kv4(s["q"], s["cache"], s["table"], s["lengths"], s["longest"], s["scale"])


def reserve_plain(s):
    """New pages from the ring's head, in row order; pages given back at its tail; slots of the new tokens."""
    page, tokens, table, ring = s["page"], s["tokens"], s["table"], s["ring"]
    size, width = ring.shape[0], table.shape[1]
    before, after, counts = (s[k].long() for k in ("before", "after", "counts"))
    held, need = (before + page - 1) // page, (after + page - 1) // page
    fits = after <= width * page
    demand = torch.where(fits, (need - held).clamp_min(0), 0)
    running = demand.cumsum(0)
    head, tail = s["counters"][0], s["counters"][1]
    granted = fits & ((demand == 0) | (running <= tail - head))
    column = torch.arange(width, device=table.device)
    fresh = granted[:, None] & (column >= held[:, None]) & (column < need[:, None])
    at = (head + (running - demand)[:, None] + column - held[:, None]).remainder(size)
    new_table = torch.where(fresh, ring[at], table)
    back = torch.where(granted, (held - need).clamp_min(0), 0)
    given = back.cumsum(0)
    gone = granted[:, None] & (column >= need[:, None]) & (column < held[:, None])
    to = (tail + (given - back)[:, None] + column - need[:, None]).remainder(size)
    longer = torch.cat((ring, ring[:1]))
    new_ring = longer.scatter(0, torch.where(gone, to, size).flatten(), table.flatten())[:size]
    counts, length = torch.where(granted, counts, 0), torch.where(granted, after, before)
    step = torch.arange(tokens, device=table.device)
    real = step < counts[:, None]
    position = torch.where(real, (after - counts)[:, None] + step, 0)
    slots = torch.gather(new_table, 1, position // page).long() * page + position % page
    taken = torch.where(granted, demand, 0).sum()
    return [torch.stack((counts, length)).int(), position, torch.where(real, slots, -1),
            torch.stack((head + taken, tail + given[-1])), new_table, new_ring]


def quantise(x):
    """Codes 0..7 (a negative feature's plus 8) of each feature and exponents of each block, x fp32 [..., D]."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    fraction, exponent = torch.frexp(blocks.abs().amax(-1))
    exponent = torch.where(fraction > 0, exponent - 3 + (fraction > 0.875).int(), -125).clamp(-125, 125)
    y = torch.ldexp(blocks, -exponent[..., None])
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    return (code + 8 * (y < 0).int()).flatten(-2), exponent


def pack(codes):
    pairs = codes.unflatten(-1, (-1, 2))
    return (pairs[..., 0] + 16 * pairs[..., 1]).to(torch.uint8)


def values(codes, exponent):
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    return torch.ldexp(grid[codes.long()].unflatten(-1, (-1, BLOCK)), exponent[..., None]).flatten(-2)


def round_trip(x, written):
    """What the cache holds of x [B, H, T, D], zero where nothing is written."""
    return values(*quantise(x)).masked_fill(~written[:, None, :, None], 0)


def norm_rope(x, weight, s):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (weight.float() + s["offset"])
    cos, sin = s["cos"].float()[:, :, None], s["sin"].float()[:, :, None]
    turn, rest = y.split((cos.shape[-1], y.shape[-1] - cos.shape[-1]), dim=-1)
    low, high = turn.chunk(2, dim=-1)
    return torch.cat((turn * cos + torch.cat((-high, low), dim=-1) * sin, rest), dim=-1)


def attention_plain(s):
    """softmax(scale q k^T) v over each row's pages, query i of n seeing the keys up to L - n + i."""
    q, table, page = s["q"].float(), s["table"].long(), s["page"]
    rows, heads, tokens, dim = q.shape

    def gathered(codes, scales):
        codes, exponent = codes[table], scales[table].transpose(-1, -2).int() - 127  # [B, M, H, P, ...]
        codes = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
        x = values(codes, exponent).transpose(1, 2)
        return x.reshape(rows, x.shape[1], -1, dim)

    keys, vals = gathered(*s["cache"][:2]), gathered(*s["cache"][2:])
    counts, lengths = s["lengths"].long()
    step, at = torch.arange(tokens, device=q.device), torch.arange(keys.shape[2], device=q.device)
    real = step < counts[:, None]
    seen = real[..., None] & (at <= (lengths - counts)[:, None, None] + step[:, None])  # [B, T, L]
    group = heads // keys.shape[1]
    q = q.unflatten(1, (-1, group)).flatten(2, 3)  # [B, Hkv, G * T, D]
    scores = torch.matmul(q, keys.transpose(-1, -2).contiguous()) * s["scale"]
    scores = scores.unflatten(2, (group, tokens)).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    weights = torch.exp(scores - top)
    weights = weights / weights.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(weights.flatten(2, 3), vals).unflatten(2, (group, tokens))
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)


# ---- the definition in 64 bits


def _stored(x):
    """The nearest values that the format holds, x fp64 [..., D]."""
    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = blocks.abs().max(dim=-1, keepdim=True).values
    power = torch.frexp(top)[1].double() - 1  # 2^power <= top < 2^(power + 1)
    unit = torch.exp2(power - 2)
    unit = torch.where(top > 7 * unit, 2 * unit, unit)
    unit = torch.where(top > 0, unit, 1.0).clamp(2.0 ** -125, 2.0 ** 125)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    above = torch.searchsorted(grid, (blocks.abs() / unit).clamp_max(6.0).contiguous())
    below = (above - 1).clamp_min(0)
    up, down = grid[above] - (blocks.abs() / unit).clamp_max(6.0), (blocks.abs() / unit).clamp_max(6.0) - grid[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (grid[pick] * unit * torch.sign(blocks)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "reserve":
        return None  # whole numbers
    counts = _numbers(case["counts"])
    if case["kind"] == "attention":
        return _exact_attention(s, counts, _numbers(case["lengths"]))
    hidden = (s["slots"] < 0)[:, None, :, None]
    stored = lambda x: _stored(x).masked_fill(hidden, 0.0)  # noqa: E731
    if case["kind"] == "append":
        return [stored(s["key"].double()), stored(s["value"].double())]

    def turned(x, weight):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (weight.double() + s["offset"])
        half = s["cos"].shape[-1] // 2
        c, d = s["cos"].double()[..., None, :], s["sin"].double()[..., None, :]
        y = x.clone()
        y[..., :half] = x[..., :half] * c[..., :half] - x[..., half: 2 * half] * d[..., :half]
        y[..., half: 2 * half] = x[..., half: 2 * half] * c[..., half:] + x[..., :half] * d[..., half:]
        return y.permute(0, 2, 1, 3)

    return [turned(s["q"], s["q_weight"]), stored(turned(s["key"], s["k_weight"])),
            stored(s["value"].double().permute(0, 2, 1, 3))]


def _exact_attention(s, counts, lengths):
    q, page = s["q"].double(), s["page"]
    rows, heads, tokens, dim = q.shape
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=q.device)
    out = torch.zeros(rows, tokens, heads, dim, dtype=torch.float64, device=q.device)
    kv_heads = s["cache"][0].shape[1]
    group = heads // kv_heads
    for r, (n, length) in enumerate(zip(counts, lengths)):
        pages = s["table"][r, : -(-length // page)].long()
        for h in range(kv_heads if n else 0):
            sides = []
            for codes, scales in (s["cache"][:2], s["cache"][2:]):
                byte = codes[pages, h].reshape(-1, dim // 2)[:length].int()
                x = torch.empty(length, dim, dtype=torch.float64, device=q.device)
                x[:, 0::2], x[:, 1::2] = grid[byte % 16], grid[byte // 16]
                unit = torch.exp2(scales[pages, h].permute(0, 2, 1).reshape(-1, dim // BLOCK)[:length].double() - 127)
                sides.append(x * unit.repeat_interleave(BLOCK, dim=1))
            keys, vals = sides
            hidden = torch.arange(length, device=q.device) > length - n + torch.arange(n, device=q.device)[:, None]
            for j in range(h * group, (h + 1) * group):
                weights = (torch.mm(q[r, j, :n], keys.t().contiguous()) * s["scale"]).masked_fill(hidden, -math.inf)
                out[r, :n, j] = torch.mm(torch.softmax(weights, dim=-1), vals)
    return out


def work(case):
    if case["kind"] == "reserve":
        rows, tokens = case["rows"], case["tokens"]
        # Three numbers a row in, two out; a position and a slot a token; about a page read and written a page of tokens.
        return {"bytes": 20 * rows + 16 * rows * tokens + 8 * rows * (tokens // (2 * case["page"]) + 1) + 32, "flops": 0}
    heads, kv_heads, dim, rotary, _ = SHAPES[case["shape"]]
    counts = _numbers(case["counts"])
    held = dim // 2 + dim // BLOCK  # bytes of one vector in the cache
    if case["kind"] == "attention":
        lengths = _numbers(case["lengths"])
        pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
        keys = sum(length for n, length in zip(counts, lengths) if n)
        slots = sum(-(-length // case["page"]) for length in lengths)
        return {"bytes": 2 * kv_heads * held * keys + 2 * heads * dim * (sum(counts) + len(counts) * max(counts)) + 4 * slots,
                "flops": 4 * heads * dim * pairs}
    tokens, every = sum(counts), len(counts) * case["tokens"]
    # The new tokens in, their cache entries out, and those read back for comparison.
    moved = 2 * kv_heads * (2 * dim * tokens + 2 * held * tokens + 2 * dim * every) + 16 * every
    if case["kind"] == "append":
        return {"bytes": moved, "flops": 6 * kv_heads * dim * tokens}
    return {"bytes": moved + 4 * heads * dim * every + 4 * rotary * every + 4 * dim,
            "flops": 10 * (heads + 2 * kv_heads) * dim * every}
