"""A paged KV cache held in 4 bits, and the operators that fill and read it.

Python entries of the native operators ``xinfer::paged_kv_reserve``, ``append_kv4``, ``read_kv4``,
``qk_norm_rope_append_kv4`` and ``paged_attention_kv4`` (libxinfer_attention_ops.so).  A step of a serving loop is

    lengths, positions, slots, counters = paged_kv_reserve(before, after, new, T, P, counters, table, ring)
    for each layer:
        q = qk_norm_rope_append_kv4(q, key, value, ..., slots, cache)     # or append_kv4(key, value, slots, cache)
        out = paged_attention_kv4(q, cache, table, lengths, max_length, scale)

without reading a length on the host, so it can be captured in a HIP graph and replayed (``max_length`` is then the
most the graph serves).

A cache is four uint8 tensors for a layer: key codes [N, Hkv, P, D/2], key scales [N, Hkv, D/32, P], and the same for
values; N pages of P tokens (64, 128 or 256), D in {64, 128, 256}.  Blocks of 32 features share a power of two, each
feature takes one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it: 4.25 bits a feature where the bf16 cache takes 16.  A
block's largest feature is at most 7 times its power of two, and every feature takes the nearest value, ties to the
even code.  A token whose key or value is not finite is held as zeros and gives NaN to the queries that see it.
"""

from xinfer_amd.attention import load_attention_ops, require

PAGE_SIZES = (64, 128, 256)
HEAD_DIMS = (64, 128, 256)


# AOTInductor C-shim declarations (include/xinfer_attention_aoti.h).
_CACHE_SHIM = """AtenTensorHandle key_codes, AtenTensorHandle key_scales,
    AtenTensorHandle value_codes, AtenTensorHandle value_scales"""
PAGED_C_SHIMS = {
    "paged_kv_reserve": """AOTITorchError aoti_torch_cuda_paged_kv_reserve(
    AtenTensorHandle kv_before, AtenTensorHandle kv_lengths, AtenTensorHandle query_lengths, int64_t tokens,
    int64_t page_size, AtenTensorHandle counters, AtenTensorHandle block_table, AtenTensorHandle free_pages,
    AtenTensorHandle* lengths, AtenTensorHandle* positions, AtenTensorHandle* slots,
    AtenTensorHandle* new_counters)""",
    "append_kv4": f"""AOTITorchError aoti_torch_cuda_append_kv4(
    AtenTensorHandle key, AtenTensorHandle value, AtenTensorHandle slots, {_CACHE_SHIM},
    AtenTensorHandle* unused_output)""",
    "read_kv4": f"""AOTITorchError aoti_torch_cuda_read_kv4(
    {_CACHE_SHIM}, AtenTensorHandle slots, AtenTensorHandle* key, AtenTensorHandle* value)""",
    "qk_norm_rope_append_kv4": f"""AOTITorchError aoti_torch_cuda_qk_norm_rope_append_kv4(
    AtenTensorHandle q, AtenTensorHandle key, AtenTensorHandle value, AtenTensorHandle q_weight,
    AtenTensorHandle k_weight, double eps, double weight_offset, AtenTensorHandle cos, AtenTensorHandle sin,
    AtenTensorHandle slots, {_CACHE_SHIM}, AtenTensorHandle* output)""",
    "paged_attention_kv4": f"""AOTITorchError aoti_torch_cuda_paged_attention_kv4(
    AtenTensorHandle q, {_CACHE_SHIM}, AtenTensorHandle block_table, AtenTensorHandle lengths, int64_t max_length,
    double scale, AtenTensorHandle* output)""",
}
_calls = {}


def paged_c_shims():
    """Inductor's call declarations for the paged operators, to go with ``attention_c_shims()``."""
    return {_call(name): [text] for name, text in PAGED_C_SHIMS.items()}


def _call(name):
    """The operator ``name``, loading the library on first use."""
    found = _calls.get(name)
    if found is None:
        import torch

        if not hasattr(torch.ops.xinfer, name):
            load_attention_ops(model="qwen3")
        found = _calls[name] = getattr(torch.ops.xinfer, name).default
    return found


def paged_kv4_cache(pages, kv_heads, page_size, dim, device):
    """An empty cache of one layer: (key codes, key scales, value codes, value scales)."""
    import torch

    require(page_size in PAGE_SIZES, f"Expected a page size in {PAGE_SIZES}")
    require(dim in HEAD_DIMS, f"Expected a head dimension in {HEAD_DIMS}")
    shapes = ((pages, kv_heads, page_size, dim // 2), (pages, kv_heads, dim // 32, page_size)) * 2
    return tuple(torch.zeros(shape, dtype=torch.uint8, device=device) for shape in shapes)


def free_page_ring(pages, device):
    """The ring of free pages with all of them in it, and its counters (head, tail)."""
    import torch

    return (torch.arange(pages, dtype=torch.int32, device=device),
            torch.tensor([0, pages], dtype=torch.int64, device=device))


def paged_kv_reserve(kv_before, kv_lengths, query_lengths, tokens, page_size, counters, block_table, free_pages):
    """Pages, slots and positions of a step: (lengths [2,B], positions [B,T], slots [B,T], new counters).

    ``kv_before``, ``kv_lengths``, ``query_lengths``: int32 [B] on the device: each row's length before the step (what
    its pages were reserved for), after it, and how many of those are new (the last ones); ``tokens``: T, the padded
    number of new tokens.  A row may shrink (an ended request goes to 0, drafted tokens are taken back) and then gives
    pages back, which serve from the next call on.  ``block_table`` int32 [B,M] and the ring ``free_pages`` (a place for
    every page) are updated in place; ``counters`` int64 [2], the ring's head and tail, is returned updated as a new
    tensor.

    ``lengths`` holds each row's real new tokens and its length: those asked for, or 0 and the length before for a row
    whose pages were not to be had.  Slots of padded tokens are -1, their positions 0.  The call gives the same again
    for the same inputs.
    """
    return _call("paged_kv_reserve")(kv_before, kv_lengths, query_lengths, tokens, page_size, counters, block_table,
                                   free_pages)


def append_kv4(key, value, slots, cache):
    """Quantise key/value (bf16 [B,Hkv,T,D], any strides) into the cache's slots (int64 [B,T], distinct).

    Slots outside the cache (-1 for padded tokens) are skipped.
    """
    _call("append_kv4")(key, value, slots, *cache)


def read_kv4(cache, slots):
    """What the cache holds at ``slots`` int64 [B,T]: (key, value) bf16 [B,Hkv,T,D], zero for slots outside it."""
    return _call("read_kv4")(*cache, slots)


def qk_norm_rope_append_kv4(q, key, value, q_weight, k_weight, eps, weight_offset, cos, sin, slots, cache):
    """Normalise and rotate queries and keys, append keys and values; returns the query [B,Hq,T,D].

    ``q`` bf16 [B,T,Hq,D], ``key``/``value`` bf16 [B,T,Hkv,D]: the projections viewed per head; per row
    x * rsqrt(mean(x^2) + eps) * (weight + weight_offset) (0 for plain RMSNorm weights, 1 for weights stored minus
    one), then the rotation of the first R features by ``cos``/``sin`` bf16 [B,T,R].  The query is computed in
    fp32 and rounded to bf16 once; the key goes to its 4 bits directly, in 64 bits where fp32 could decide a code.
    """
    return _call("qk_norm_rope_append_kv4")(q, key, value, q_weight, k_weight, eps, weight_offset, cos, sin,
                                          slots, *cache)


def paged_attention_kv4(q, cache, block_table, lengths, max_length, scale):
    """Attention of q [B,Hq,T,D] over the cache, lower-right causal: bf16 [B,T,Hq,D], zero for padded queries.

    ``lengths`` int32 [2,B] on the device, as ``paged_kv_reserve`` returns it.  ``max_length``: the host's bound on the
    rows' lengths (0: what the table can hold); it sizes the launch, and longer rows are read up to it.
    """
    return _call("paged_attention_kv4")(q, *cache, block_table, lengths, max_length, scale)


def register_fakes():
    """Shape contracts of the operators (called by ``load_attention_ops`` once the library is loaded)."""
    import torch

    def check_cache(codes, scales, other_codes, other_scales):
        torch._check(codes.dim() == 4 and scales.dim() == 4)
        torch._check(other_codes.shape == codes.shape and other_scales.shape == scales.shape)
        torch._check(scales.shape == (codes.shape[0], codes.shape[1], codes.shape[3] // 16, codes.shape[2]))

    @torch.library.register_fake("xinfer::paged_kv_reserve")
    def fake_reserve(kv_before, kv_lengths, query_lengths, tokens, page_size, counters, block_table, free_pages):
        rows = kv_before.shape[0]
        torch._check(kv_lengths.shape == (rows,) and query_lengths.shape == (rows,))
        torch._check(counters.shape == (2,) and block_table.dim() == 2 and block_table.shape[0] == rows)
        return (kv_before.new_empty((2, rows)), counters.new_empty((rows, tokens)), counters.new_empty((rows, tokens)),
                counters.new_empty((2,)))

    @torch.library.register_fake("xinfer::append_kv4")
    def fake_append(key, value, slots, key_codes, key_scales, value_codes, value_scales):
        check_cache(key_codes, key_scales, value_codes, value_scales)
        torch._check(key.dim() == 4 and value.shape == key.shape and slots.shape == (key.shape[0], key.shape[2]))
        return None

    @torch.library.register_fake("xinfer::read_kv4")
    def fake_read(key_codes, key_scales, value_codes, value_scales, slots):
        check_cache(key_codes, key_scales, value_codes, value_scales)
        torch._check(slots.dim() == 2)
        shape = (slots.shape[0], key_codes.shape[1], slots.shape[1], 2 * key_codes.shape[3])
        return slots.new_empty(shape, dtype=torch.bfloat16), slots.new_empty(shape, dtype=torch.bfloat16)

    @torch.library.register_fake("xinfer::qk_norm_rope_append_kv4")
    def fake_norm_rope(q, key, value, q_weight, k_weight, eps, weight_offset, cos, sin, slots, key_codes, key_scales,
                       value_codes, value_scales):
        check_cache(key_codes, key_scales, value_codes, value_scales)
        torch._check(q.dim() == 4 and key.dim() == 4 and value.shape == key.shape and key.shape[:2] == q.shape[:2])
        torch._check(cos.dim() == 3 and sin.shape == cos.shape and slots.shape == q.shape[:2])
        return q.new_empty((q.shape[0], q.shape[2], q.shape[1], q.shape[3]))

    @torch.library.register_fake("xinfer::paged_attention_kv4")
    def fake_attention(q, key_codes, key_scales, value_codes, value_scales, block_table, lengths, max_length, scale):
        check_cache(key_codes, key_scales, value_codes, value_scales)
        torch._check(q.dim() == 4 and q.shape[1] % key_codes.shape[1] == 0 and q.shape[3] == 2 * key_codes.shape[3])
        torch._check(block_table.dim() == 2 and block_table.shape[0] == q.shape[0])
        torch._check(lengths.shape == (2, q.shape[0]))
        return q.new_empty((q.shape[0], q.shape[2], q.shape[1], q.shape[3]))
