"""The paged 4-bit KV cache's operators against a float64 oracle (oracle/kv4.py).

Sizes go where the kernels can go wrong: one token and one key, counts and lengths around the 64-key steps and the
page sizes, rows without queries or without keys, missing pages, odd strides, non-finite tokens, values around the
format's borders.

Tolerances.  Codes, scales, slots and positions are compared whole.  A normalised query is rounded to bf16 once: half
a step, 2^-8 of its value at most, plus the fp32 arithmetic in front of it (some 10 roundings and one rsqrt of 1 ulp,
under 2^-19 of the row's largest value).  An attention output is a weighted mean of values whose weights sum to one: the
output's rounding is at most 2^-8 |out|; weights rounded to bf16 are off by at most 2^-8 of themselves and move the
mean by at most 2^-8 sum(w |v|), and by as much again where the sum of the weights is taken after their rounding; the
scores' arithmetic (sums of up to 256 products that keep 2^-17 of their largest term, below 8 here, then one
exponential) adds a relative 2^-12 of the weights.  So |error| <= 2^-8 |out| + (2^-7 + 2^-11) sum(w |v|).
"""

import numpy as np
import pytest
import torch

from attn_helpers import log
from oracle import kv4 as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_ops):
    from xinfer_amd import paged_kv4

    return paged_kv4


def randn(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16)


def f64(t):
    return t.detach().cpu().double().numpy()


def host(cache):
    return [t.cpu().numpy().copy() for t in cache]


def new_cache(ops, pages, kv_heads, size, dim, seed=0):
    """A cache full of bytes a fresh allocation may hold, so that writing too far shows."""
    g = torch.Generator().manual_seed(seed)
    cache = ops.paged_kv4_cache(pages, kv_heads, size, dim, "cuda")
    for t in cache:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    return cache


# ---- append and read-back


def border_values(g, *shape):
    """Values around the format's decisions: halves between grid values, powers of two, zeros, tiny and huge ones."""
    x = torch.randn(*shape, generator=g)
    kind = torch.randint(0, 8, shape, generator=g)
    grid = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    halves = grid[torch.randint(0, 10, shape, generator=g)]
    power = torch.randint(-3, 4, (*shape[:-1], 1), generator=g)
    x = torch.where(kind < 4, torch.ldexp(halves, power), torch.ldexp(x, power))
    x = torch.where(kind == 7, -x, x)
    row = torch.randint(0, 12, (*shape[:-1], 1), generator=g)
    x = torch.where(row == 0, torch.zeros(()), x)
    x = torch.where(row == 1, x * 2.0**-120 * 2.0**-10, x)
    x = torch.where(row == 2, x * 2.0**120, x)
    return x.clamp(-3.38e38, 3.38e38).to(torch.bfloat16)


@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("dim,kv_heads,batch,tokens", [(64, 8, 3, 1), (64, 1, 1, 67), (128, 8, 1, 1), (128, 5, 2, 130),
                                                       (256, 4, 3, 33), (256, 1, 1, 1)])
def test_append_and_read(ops, dim, kv_heads, batch, tokens, size):
    log(f"append_kv4 D={dim} Hkv={kv_heads} B={batch} T={tokens} P={size}")
    g = torch.Generator().manual_seed(dim + tokens)
    pages = -(-batch * tokens // size) + 2
    cache = new_cache(ops, pages, kv_heads, size, dim)
    expected = host(cache)
    key, value = border_values(g, batch, kv_heads, tokens, dim), border_values(g, batch, kv_heads, tokens, dim)
    slots = torch.randperm(pages * size, generator=g)[: batch * tokens].reshape(batch, tokens)
    if tokens > 2:  # padded tokens, slots past the cache, tokens that are not finite
        slots[-1, -1], slots[0, 1] = -1, pages * size
        key[0, 0, 0, 3], value[-1, -1, tokens // 2, 5] = float("inf"), float("nan")
    # [B, T, H, D] storage seen as [B, H, T, D], as the adapters' projections are.
    strided = key.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    ops.append_kv4(strided, value.cuda(), slots.cuda(), cache)
    torch.cuda.synchronize()
    oracle.append(expected, f64(key), f64(value), slots.numpy())
    got = host(cache)
    for name, a, b in zip(("key scales", "value scales"), got[1::2], expected[1::2]):
        assert np.array_equal(a, b), name
    positive = lambda c: np.where(c & 7, c, 0)  # noqa: E731  (a zero may carry either sign)
    for name, a, b in zip(("key codes", "value codes"), got[0::2], expected[0::2]):
        assert np.array_equal(positive(a & 15), positive(b & 15)), name
        assert np.array_equal(positive(a >> 4), positive(b >> 4)), name
    k, v = ops.read_kv4(cache, slots.cuda())
    keys, vals = oracle.unpack(expected)
    for b, t in np.ndindex(batch, tokens):
        slot = slots[b, t].item()
        there = 0 <= slot < pages * size
        for out, ref in ((k, keys), (v, vals)):
            want = ref[slot // size, :, slot % size] if there else np.zeros((kv_heads, dim))
            np.testing.assert_array_equal(f64(out[b, :, t]), want)


def test_append_copies_odd_strides(ops):
    log("append_kv4 odd strides")
    g = torch.Generator().manual_seed(5)
    key = randn(g, 2, 3, 5, 128).cuda()
    wide = torch.zeros(2, 3, 5, 131, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:129] = key
    slots = torch.arange(10, device="cuda").flip(0).reshape(5, 2).t()  # strided too
    caches = [ops.paged_kv4_cache(1, 3, 64, 128, "cuda") for _ in range(2)]
    ops.append_kv4(key, key, slots, caches[0])
    ops.append_kv4(wide[..., 1:129], key.transpose(2, 3).contiguous().transpose(2, 3), slots, caches[1])
    for a, b in zip(*caches):
        assert torch.equal(a, b) and a.any()


# ---- norm, rotation and append


@pytest.mark.parametrize("heads,kv_heads,dim,rotary,offset,batch,tokens", [
    (16, 8, 128, 128, 0.0, 3, 1), (16, 8, 128, 128, 0.0, 2, 37), (16, 4, 256, 64, 1.0, 2, 5), (8, 2, 256, 256, 1.0, 1, 1),
    (5, 5, 64, 64, 0.0, 1, 9), (6, 2, 64, 16, 1.0, 4, 3), (3, 1, 128, 96, 0.0, 1, 65), (7, 1, 256, 48, 0.0, 1, 2)])
def test_norm_rope_append(ops, heads, kv_heads, dim, rotary, offset, batch, tokens):
    log(f"qk_norm_rope_append_kv4 {heads}/{kv_heads} D={dim} R={rotary} B={batch} T={tokens}")
    g = torch.Generator().manual_seed(heads + dim)
    size = 64
    pages = -(-batch * tokens // size) + 1
    cache = new_cache(ops, pages, kv_heads, size, dim)
    start = host(cache)
    q, key, value = (randn(g, batch, tokens, h, dim) for h in (heads, kv_heads, kv_heads))
    qw, kw = ((1 - offset + 0.1 * torch.randn(dim, generator=g)).to(torch.bfloat16) for _ in range(2))
    angle = 6.28 * torch.rand(batch, tokens, rotary // 2, generator=g)
    cos, sin = (torch.cat((f(angle), f(angle)), -1).to(torch.bfloat16) for f in (torch.cos, torch.sin))
    slots = torch.randperm(pages * size, generator=g)[: batch * tokens].reshape(batch, tokens)
    if tokens > 2:
        q[0, 0, 0] = 0  # only eps under the root
        slots[-1, -1] = -1
        value[0, 1, 0, 0] = float("-inf")
    # q is half of a [.., 2D] projection, as beside an output gate.
    wide = torch.cat((q, torch.full_like(q, float("nan"))), dim=-1).cuda()
    out = ops.qk_norm_rope_append_kv4(wide[..., :dim], key.cuda(), value.cuda(), qw.cuda(), kw.cuda(), 1e-6, offset,
                                      cos.cuda(), sin.cuda(), slots.cuda(), cache)
    want = oracle.norm_rope(f64(q), f64(qw), offset, 1e-6, f64(cos), f64(sin)).transpose(0, 2, 1, 3)
    error = np.abs(f64(out) - want)
    assert (error <= 2.0**-8 * np.abs(want) + 2.0**-19 * np.abs(want).max(-1, keepdims=True)).all()
    k = oracle.norm_rope(f64(key), f64(kw), offset, 1e-6, f64(cos), f64(sin)).transpose(0, 2, 1, 3)
    expected = [t.copy() for t in start]
    oracle.append(expected, k, f64(value).transpose(0, 2, 1, 3), slots.numpy())
    got = host(cache)
    used = np.zeros((pages, size), bool)
    for s in slots.flatten().tolist():
        if s >= 0:
            used[s // size, s % size] = True
    keys, vals = oracle.unpack(got)
    ref_keys, ref_vals = oracle.unpack(expected)
    np.testing.assert_array_equal(vals, ref_vals)
    for b, t in np.ndindex(batch, tokens):
        s = slots[b, t].item()
        if s < 0:
            continue
        a, ref, x = keys[s // size, :, s % size], ref_keys[s // size, :, s % size], k[b, :, t]
        assert np.array_equal(np.isnan(a), np.isnan(ref))
        # A key within the fp32 arithmetic (2^-19 of its row's largest) of a border may take either side of it, and a
        # block whose largest is that near a border of the scale may take the other scale.
        near = np.abs(x).max(-1, keepdims=True) * 2.0**-19
        fine = np.isnan(ref) | (a == ref) | (np.abs(a - x) <= np.abs(ref - x) + 2 * near)
        e = oracle.block_exponents(x)
        top = np.abs(x).reshape(kv_heads, -1, 32).max(-1)
        border = np.minimum(np.abs(top - 7 * np.exp2(e * 1.0)), np.abs(top - 3.5 * np.exp2(e * 1.0))) <= 2 * near
        assert (fine | np.repeat(border, 32, axis=-1)).all()
    for a, b, axis in zip(got, start, (2, 3, 2, 3)):  # nothing but the slots is written
        np.testing.assert_array_equal(np.moveaxis(a, axis, 1)[~used], np.moveaxis(b, axis, 1)[~used])


# ---- page tables


def reserve_both(ops, before, after, counts, tokens, size, counters, table, ring):
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    t, f = as_int(table.tolist()).reshape(table.shape), as_int(ring.tolist())
    want = oracle.reserve(before, after, counts, tokens, size, counters, table, ring)
    for _ in range(2):  # the same again
        got = ops.paged_kv_reserve(as_int(before), as_int(after), as_int(counts), tokens, size,
                                   torch.tensor(counters, device="cuda"), t, f)
        for a, b in zip([*got, t, f], want):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
    return want


@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("rows,tokens,width,spare", [(1, 1, 1, 1), (8, 1, 40, 1000), (64, 7, 9, 12), (3, 513, 20, 7),
                                                     (300, 3, 5, 40), (700, 2, 3, 0), (257, 1, 2, 5000)])
def test_reserve(ops, rows, tokens, width, spare, size):
    rng = np.random.default_rng(rows + size)
    capacity = width * size
    for seed in range(3):
        log(f"paged_kv_reserve rows={rows} tokens={tokens} width={width} spare={spare} P={size} seed={seed}")
        before = rng.integers(0, capacity + 1, rows)
        before[rng.random(rows) < 0.2] = 0
        counts = rng.integers(0, tokens + 1, rows)
        keep = np.where(rng.random(rows) < 0.3, np.maximum(before - rng.integers(0, 2 * size, rows), 0), before)
        keep[rng.random(rows) < 0.1] = 0
        after = keep + counts  # may be more than the table's row holds
        held = -(-before // size)
        pages = rng.permutation(int(held.sum()) + spare + 1)
        table = np.full((rows, width), -1)
        at = 0
        for r, n in enumerate(held):
            table[r, :n] = pages[at: at + n]
            at += n
        free = pages[at:]
        ring = rng.permutation(len(pages) + 3)
        head = int(rng.integers(0, 1 << 40))
        ring[(head + np.arange(len(free))) % len(ring)] = free
        reserve_both(ops, before.tolist(), after.tolist(), counts.tolist(), tokens, size, [head, head + len(free)], table,
                     ring)


def test_reserve_refuses_rows_in_order(ops):
    """Five free pages, demands 3, 0, 4, 1, 0: the third row and the later one that needs a page wait."""
    log("paged_kv_reserve refusals")
    table = np.arange(100, 110).reshape(5, 2)
    table = np.concatenate((table, np.full((5, 4), -1)), axis=1)
    want = reserve_both(ops, [64, 10, 64, 64, 128], [256, 11, 320, 65, 63], [192, 1, 256, 1, 0], 256, 64, [7, 12], table,
                        np.arange(9))
    assert want[0].tolist() == [[192, 1, 0, 0, 0], [256, 11, 64, 64, 63]]
    assert want[3].tolist() == [10, 13]


def test_reserve_without_rows(ops):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    ring, counters = ops.free_page_ring(4, "cuda")
    lengths, positions, slots, after = ops.paged_kv_reserve(e, e, e, 3, 64, counters, e.reshape(0, 5), ring)
    assert lengths.shape == (2, 0) and positions.shape == slots.shape == (0, 3) and after.tolist() == [0, 4]


# ---- attention


def filled_cache(ops, g, pages, kv_heads, size, dim):
    cache = ops.paged_kv4_cache(pages, kv_heads, size, dim, "cuda")
    key, value = randn(g, 1, kv_heads, pages * size, dim), randn(g, 1, kv_heads, pages * size, dim)
    ops.append_kv4(key.cuda(), value.cuda(), torch.arange(pages * size, device="cuda")[None], cache)
    return cache


def make_table(g, lengths, size, extra=0):
    need = [-(-n // size) for n in lengths]
    order = torch.randperm(sum(need) + extra, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at: at + n]
        at += n
    return table, sum(need) + extra


def check_attention(out, q, cache, table, lengths, scale, max_length=None):
    args = (f64(q), host(cache), table.cpu().numpy(), lengths.cpu().numpy(), scale, max_length)
    want, spread = oracle.attention(*args), oracle.attention(*args, magnitudes=True)
    got = f64(out)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    error = np.abs(np.nan_to_num(got - want))
    allowed = 2.0**-8 * np.abs(np.nan_to_num(want)) + (2.0**-7 + 2.0**-11) * np.nan_to_num(spread)
    assert (error <= allowed).all(), (error - allowed).max()


SHAPES = [(16, 8, 128), (16, 4, 256), (8, 8, 64), (32, 8, 128), (8, 1, 128), (3, 3, 256), (12, 4, 64)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("counts,lengths,size", [
    ([1], [1], 64), ([1, 1, 1, 1], [1, 64, 65, 700], 64), ([1, 0, 1], [300, 40, 257], 128), ([2, 1], [2, 130], 256),
    ([5, 3, 0, 1], [260, 3, 0, 64], 64), ([17], [1100], 128), ([40, 1, 33], [40, 513, 400], 64), ([130], [131], 256)])
def test_attention(ops, heads, kv_heads, dim, counts, lengths, size):
    log(f"paged_attention_kv4 {heads}/{kv_heads}/{dim} counts={counts} lengths={lengths} P={size}")
    g = torch.Generator().manual_seed(dim + len(counts))
    table, pages = make_table(g, lengths, size, extra=1)
    cache = filled_cache(ops, g, pages, kv_heads, size, dim)
    q = randn(g, len(counts), heads, max(counts), dim)
    rows = torch.tensor([counts, lengths], dtype=torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), rows.cuda(), max(lengths), dim**-0.5)
    check_attention(out, q, cache, table, rows, dim**-0.5)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES[:4])
@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_attention_over_long_rows(ops, heads, kv_heads, dim, tokens):
    """Rows long enough to be split, short and empty ones beside them; every bound on the length gives the same."""
    lengths, counts = [4100, 1, 2047, 70, 0, 6001], [tokens, 1, tokens, tokens, 0, 1]
    log(f"paged_attention_kv4 long {heads}/{kv_heads}/{dim} T={tokens}")
    g = torch.Generator().manual_seed(tokens)
    table, pages = make_table(g, lengths, 64)
    cache = filled_cache(ops, g, pages, kv_heads, 64, dim)
    q = randn(g, len(counts), heads, tokens, dim)
    rows = torch.tensor([counts, lengths], dtype=torch.int32)
    rows[0].clamp_(max=rows[1])
    outs = [ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), rows.cuda(), bound, dim**-0.5) for bound in (6001, 0, 0)]
    assert torch.equal(outs[1], outs[2])
    for out in outs[:2]:
        check_attention(out, q, cache, table, rows, dim**-0.5)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES[:3])
@pytest.mark.parametrize("tokens", [1, 4, 50])
def test_attention_absent_pages_and_foreign_bytes(ops, heads, kv_heads, dim, tokens):
    """Entries outside the cache count as absent, a row may have none left; bytes past a row's length, 255 among them,
    and lengths past the bounds change nothing."""
    log(f"paged_attention_kv4 absent pages {heads}/{kv_heads}/{dim} T={tokens}")
    g = torch.Generator().manual_seed(3)
    lengths, size = [200, 300, 130, 65], 64
    table, pages = make_table(g, lengths, size, extra=2)
    cache = filled_cache(ops, g, pages, kv_heads, size, dim)
    for r, length in enumerate(lengths):  # the places behind a row's last token
        page = table[r, (length - 1) // size].item()
        for t, tail in zip(cache, (2, 3, 2, 3)):
            t[page].narrow(tail - 1, length % size, size - length % size).fill_(255)
    table[0, 1], table[1, 4], table[2, :] = -1, pages, -5
    q = randn(g, 4, heads, tokens, dim)
    rows = torch.tensor([[tokens] * 4, lengths], dtype=torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), rows.cuda(), 0, dim**-0.5)
    check_attention(out, q, cache, table, rows, dim**-0.5)
    assert not out[2].any()
    wild = torch.tensor([[tokens + 9, -3, tokens, tokens], [200, 300, 130, 1 << 30]], dtype=torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), wild.cuda(), 100, dim**-0.5)
    check_attention(out, q, cache, table, wild, dim**-0.5, max_length=100)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES[:3])
@pytest.mark.parametrize("tokens", [2, 6, 70])
def test_attention_of_tokens_that_are_not_finite(ops, heads, kv_heads, dim, tokens):
    """A NaN or an infinity reaches the queries that see its token and no others."""
    log(f"paged_attention_kv4 not finite {heads}/{kv_heads}/{dim} T={tokens}")
    g = torch.Generator().manual_seed(4)
    size, length = 128, 200
    table, pages = make_table(g, [length, length], size)
    cache = filled_cache(ops, g, pages, kv_heads, size, dim)
    key, value = randn(g, 1, kv_heads, 1, dim), randn(g, 1, kv_heads, 1, dim)
    value[0, 0, 0, 7] = float("nan")
    at = length - tokens // 2  # seen by the later half of row 0's queries
    slot = table[0, at // size].item() * size + at % size
    ops.append_kv4(key.cuda(), value.cuda(), torch.tensor([[slot]], device="cuda"), cache)
    q = randn(g, 2, heads, tokens, dim)
    rows = torch.tensor([[tokens, tokens], [length, length]], dtype=torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), rows.cuda(), 0, dim**-0.5)
    check_attention(out, q, cache, table, rows, dim**-0.5)
    poisoned = torch.isnan(out[0, :, 0, 0])
    assert poisoned.any() and not poisoned.all() and not torch.isnan(out[1]).any()


def test_attention_of_large_and_small_queries(ops):
    """Queries of very different sizes within a block of features, a half and a whole query of zeros."""
    log("paged_attention_kv4 query sizes")
    g = torch.Generator().manual_seed(6)
    table, pages = make_table(g, [333], 64)
    cache = filled_cache(ops, g, pages, 2, 64, 128)
    q = randn(g, 1, 4, 3, 128) * torch.exp2(torch.randint(-20, 2, (1, 4, 3, 128), generator=g).float()).to(torch.bfloat16)
    q[0, 1, 1], q[0, 0, 0, 64:] = 0, 0
    rows = torch.tensor([[3], [333]], dtype=torch.int32)
    for scale in (128**-0.5, 1e-3):
        out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), rows.cuda(), 333, scale)
        check_attention(out, q, cache, table, rows, scale)


@pytest.mark.parametrize("tokens", [1, 20])
def test_attention_strides_streams_and_graphs(ops, tokens):
    """A strided query, another stream than the default, and a captured call replayed with other lengths."""
    log(f"paged_attention_kv4 graph T={tokens}")
    g = torch.Generator().manual_seed(9)
    lengths = [900, 64, 3000]
    table, pages = make_table(g, [3200, 3200, 3200], 64)
    cache = filled_cache(ops, g, pages, 8, 64, 128)
    q = randn(g, 3, tokens, 16, 128).cuda().transpose(1, 2)
    t = table.cuda()
    rows = torch.tensor([[tokens] * 3, lengths], dtype=torch.int32, device="cuda")
    plain = ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1)
    assert torch.equal(plain, ops.paged_attention_kv4(q.contiguous(), cache, t, rows, 0, 0.1))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(plain, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1)
    for step in ([900, 64, 3000], [tokens, 3200, 1700], [3199, 130, tokens + 1]):
        rows[1] = torch.tensor(step, dtype=torch.int32, device="cuda")
        graph.replay()
        eager = ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES[:2])
@pytest.mark.parametrize("rows,tokens", [(65, 1), (130, 1), (70, 3), (67, 40), (64, 40)])
def test_attention_of_many_rows(ops, heads, kv_heads, dim, rows, tokens):
    """Batches past a wave's 64 lanes, which the plan takes 64 rows at a time; a few of the last rows are long."""
    log(f"paged_attention_kv4 rows={rows} {heads}/{kv_heads}/{dim} T={tokens}")
    g = torch.Generator().manual_seed(rows + tokens)
    counts = torch.randint(0, tokens + 1, (rows,), generator=g)
    lengths = counts + torch.randint(0, 100, (rows,), generator=g)
    lengths[-3:] = torch.tensor([1500, 70, 2500])
    counts[-3:] = torch.tensor([tokens, 0, tokens])
    table, pages = make_table(g, lengths.tolist(), 64)
    cache = filled_cache(ops, g, pages, kv_heads, 64, dim)
    q = randn(g, rows, heads, tokens, dim)
    state = torch.stack((counts, lengths)).to(torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), state.cuda(), 2500, dim**-0.5)
    check_attention(out, q, cache, table, state, dim**-0.5)


@pytest.mark.parametrize("heads,kv_heads,dim,longest", [(16, 8, 128, 600), (16, 8, 128, 768), (16, 8, 64, 1024), (8, 8, 64, 1300),
                                                        (16, 8, 128, 1025)])
@pytest.mark.parametrize("rows", [1, 20])
def test_attention_of_short_rows(ops, heads, kv_heads, dim, longest, rows):
    """Single tokens over rows that a block takes whole, with its waves' shares from none to two groups."""
    log(f"paged_attention_kv4 short rows={rows} {heads}/{kv_heads}/{dim} L={longest}")
    g = torch.Generator().manual_seed(longest)
    lengths = torch.randint(0, longest + 1, (rows,), generator=g)
    lengths[-1] = longest
    table, pages = make_table(g, lengths.tolist(), 64)
    cache = filled_cache(ops, g, pages, kv_heads, 64, dim)
    q = randn(g, rows, heads, 1, dim)
    state = torch.stack((lengths.clamp(max=1), lengths)).to(torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), state.cuda(), longest, dim**-0.5)
    check_attention(out, q, cache, table, state, dim**-0.5)


@pytest.mark.parametrize("tokens", [4, 30])
def test_a_bound_below_the_new_tokens(ops, tokens):
    """``max_length`` below a row's count: only that many queries are answered, the others are zeros."""
    log(f"paged_attention_kv4 bound below T={tokens}")
    g = torch.Generator().manual_seed(8)
    table, pages = make_table(g, [100, 100], 64)
    cache = filled_cache(ops, g, pages, 2, 64, 128)
    q = randn(g, 2, 4, tokens, 128)
    state = torch.tensor([[tokens, 1], [100, 100]], dtype=torch.int32)
    out = ops.paged_attention_kv4(q.cuda(), cache, table.cuda(), state.cuda(), 3, 0.1)
    check_attention(out, q, cache, table, state, 0.1, max_length=3)
    assert not out[0, 3:].any()


@pytest.mark.parametrize("tokens", [1, 24])
def test_attention_copies_odd_strides(ops, tokens):
    log(f"paged_attention_kv4 odd strides T={tokens}")
    g = torch.Generator().manual_seed(11)
    table, pages = make_table(g, [90, 40], 64)
    cache = filled_cache(ops, g, pages, 8, 64, 128)
    q = randn(g, 2, 16, tokens, 128).cuda()
    wide = torch.full((2, 16, tokens, 131), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[..., 1:129] = q
    state = torch.tensor([[tokens, tokens], [90, 40]], dtype=torch.int32, device="cuda")
    want = ops.paged_attention_kv4(q, cache, table.cuda(), state, 0, 0.1)
    assert torch.equal(ops.paged_attention_kv4(wide[..., 1:129], cache, table.cuda(), state, 0, 0.1), want)


def test_a_cache_past_32_bits(ops):
    """Pages behind the first 4 GiB of codes: what is written, read and attended is what a small cache gives."""
    log("paged kv4 cache past 32 bits")
    g = torch.Generator().manual_seed(12)
    heads, size, dim, pages = 8, 256, 256, (1 << 14) + 300  # 256 KiB of codes a page
    places = [pages - 1, 5, (1 << 14) + 1]
    big, small = ops.paged_kv4_cache(pages, heads, size, dim, "cuda"), ops.paged_kv4_cache(3, heads, size, dim, "cuda")
    at = torch.arange(3 * size).reshape(3, size)
    far = torch.tensor(places)[:, None] * size + at % size
    x = [randn(g, 3, size, heads, dim).cuda() for _ in range(3)]
    weight, turn = torch.ones(dim, dtype=torch.bfloat16, device="cuda"), torch.ones(3, size, 64, dtype=torch.bfloat16, device="cuda")
    queries = [ops.qk_norm_rope_append_kv4(x[0], x[1], x[2], weight, weight, 1e-6, 0.0, turn, turn, s.cuda(), c)
               for s, c in ((far, big), (at, small))]
    assert torch.equal(*queries)
    for a, b in zip(ops.read_kv4(big, far.cuda()), ops.read_kv4(small, at.cuda())):
        assert torch.equal(a, b) and a.any()
    for b, s in zip(big, small):
        assert torch.equal(b[places], s)
    for tokens in (1, 100):
        q = queries[0][:1, :, :tokens]
        state = torch.tensor([[tokens], [3 * size]], dtype=torch.int32, device="cuda")
        outs = [ops.paged_attention_kv4(q, c, torch.tensor([t], dtype=torch.int32, device="cuda"), state, 0, 0.1)
                for c, t in ((big, places), (small, [0, 1, 2]))]
        assert torch.equal(*outs) and outs[0].any()


def test_operators_refuse(ops):
    """What the kernels do not serve is refused before a launch."""
    log("paged kv4 refusals")
    half = dict(dtype=torch.bfloat16, device="cuda")
    cache = ops.paged_kv4_cache(4, 8, 64, 128, "cuda")
    key, slots = torch.zeros(2, 8, 3, 128, **half), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    q, table = torch.zeros(2, 16, 3, 128, **half), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    rows = torch.tensor([[3, 3], [3, 3]], dtype=torch.int32, device="cuda")

    def refused(message, call, *args):
        with pytest.raises(RuntimeError, match=message):
            call(*args)

    refused("BF16", ops.append_kv4, key.half(), key.half(), slots, cache)
    refused("inference only", ops.append_kv4, key.clone().requires_grad_(), key, slots, cache)
    refused("int64 slots", ops.append_kv4, key, key, slots.int(), cache)
    refused("int64 slots", ops.append_kv4, key, key, slots[:, :2], cache)
    refused("colocated", ops.append_kv4, key, key, slots.cpu(), cache)
    refused("uint8 cache", ops.append_kv4, key, key, slots, [t.int() for t in cache])
    refused("uint8 cache", ops.read_kv4, [t[:, ::2] for t in cache], slots)
    refused("cache codes", ops.append_kv4, key, key, slots, (cache[0], cache[1][..., :32].contiguous(), *cache[2:]))
    refused("Tensors do not match", ops.append_kv4, key[..., :64], key[..., :64], slots, cache)
    by_token, weight = key.transpose(1, 2), torch.ones(128, **half)
    for width, message in ((24, "Tensors do not match"), (144, "Tensors do not match")):
        turn = torch.ones(2, 3, width, **half)
        refused(message, ops.qk_norm_rope_append_kv4, q.transpose(1, 2), by_token, by_token, weight, weight, 1e-6, 0.0, turn,
                turn, slots, cache)
    turn = torch.ones(2, 3, 64, **half)
    refused("inference only", ops.qk_norm_rope_append_kv4, q.transpose(1, 2).requires_grad_(), by_token, by_token, weight,
            weight, 1e-6, 0.0, turn, turn, slots, cache)
    refused("inference only", ops.paged_attention_kv4, q.clone().requires_grad_(), cache, table, rows, 0, 0.1)
    refused("block table", ops.paged_attention_kv4, q, cache, table.t(), rows, 0, 0.1)
    refused("int32 lengths", ops.paged_attention_kv4, q, cache, table, rows.long(), 0, 0.1)
    refused("scale", ops.paged_attention_kv4, q, cache, table, rows, 0, float("nan"))
    refused("pages", ops.paged_attention_kv4, q, cache, table, rows, -1, 0.1)
    refused("heads", ops.paged_attention_kv4, q[:, :12], cache, table, rows, 0, 0.1)
    ring, counters = ops.free_page_ring(4, "cuda")
    one = torch.zeros(2, dtype=torch.int32, device="cuda")
    refused("pages", ops.paged_kv_reserve, one, one, one, 1, 96, counters, table, ring)
    refused("row lengths", ops.paged_kv_reserve, one, one[:1], one, 1, 64, counters, table, ring)
    refused("counters", ops.paged_kv_reserve, one, one, one, 1, 64, counters.int(), table, ring)
    assert not any(t.any() for t in cache)


def test_tensors_on_two_streams(ops):
    """Calls of two streams at once, each with a workspace of its own, give what they give alone."""
    log("paged_attention_kv4 two streams")
    g = torch.Generator().manual_seed(14)
    lengths = [3000, 2500]
    table, pages = make_table(g, lengths, 64)
    cache, t = filled_cache(ops, g, pages, 8, 64, 128), table.cuda()
    work = []
    for tokens in (1, 60):
        q = randn(g, 2, 16, tokens, 128).cuda()
        rows = torch.tensor([[tokens] * 2, lengths], dtype=torch.int32, device="cuda")
        work.append((q, rows, ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        outs = []
        for q, rows, _, stream in work:
            with torch.cuda.stream(stream):
                outs.append(ops.paged_attention_kv4(q, cache, t, rows, 0, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out, (_, _, want, _) in zip(outs, work))
