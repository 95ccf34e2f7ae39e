"""Model steps over the paged 4-bit cache, as a serving loop runs them.

Two-layer Qwen3 and Qwen3.5 models (model_steps) through ``PagedModelStep``: prompts in chunks and in one piece,
decode steps captured in a HIP graph, requests that end and give their pages to others, a full pool, and a package.

Bounds.  The same tokens in other chunks pass the same weights; keys, values and weights of the softmax are
rounded alike, but sums run in another order and the projections have other shapes, so hidden states differ by bf16
roundings (about 2^-9 of a value in the mean, some tens of them a layer) and a key that such a difference moves over a border of the
4-bit grid by a whole step (up to a third of it; about one key in 50, each 2^-9 / 2^-3 of the way).  That is
sqrt(1 / 50) / 6, 2.4 % of a row's keys in norm, and less in a mean over keys: logits within a relative L2 of 5e-2.
Against the unmodified model with keys and values put through the same format the keys are rounded to bf16 before it
besides: 1e-1.
"""

from pathlib import Path

import numpy as np
import pytest
import torch

from attn_helpers import log
from model_steps import CAPACITY, LAYERS, VOCAB, build_model, transformers_row_logits
from oracle import kv4 as oracle

pytestmark = pytest.mark.gpu
SIZE = 64


@pytest.fixture(scope="module", params=["qwen3", "qwen35"])
def family(request, gpu_ops):
    return request.param


@pytest.fixture(scope="module")
def step(family):
    from xinfer_amd.adapters import PagedModelStep

    return PagedModelStep(build_model(family))


class Loop:
    """The serving loop's state: caches, page table, ring of free pages, lengths."""

    def __init__(self, step, rows, pages):
        from xinfer_amd.paged_kv4 import free_page_ring

        self.step, self.kv = step, step.cache(pages, SIZE)
        self.ring, self.counters = free_page_ring(pages, "cuda")
        self.table = torch.full((rows, CAPACITY // SIZE), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def run(self, ids, counts, after=None):
        counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
        after = self.lengths + counts if after is None else torch.tensor(after, dtype=torch.int32, device="cuda")
        with torch.inference_mode():
            logits, lengths, self.counters = self.step(ids, self.lengths, after, counts, self.kv, self.counters, self.table,
                                                       self.ring)
        self.lengths = lengths[1].clone()
        return logits, lengths


def tokens(rows, width, seed):
    return torch.randint(0, VOCAB, (rows, width), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def close(actual, expected, bound):
    actual, expected = actual.float(), expected.float()
    error = ((actual - expected).norm(dim=-1) / expected.norm(dim=-1)).max().item()
    assert torch.isfinite(actual).all() and error < bound, error


def test_chunks_and_single_tokens_agree_with_one_prompt(step, family):
    log(f"paged {family}: chunks")
    ids = tokens(3, 150, 1)
    whole = Loop(step, 3, 12)
    expected, _ = whole.run(ids, [150, 150, 150])
    parts = Loop(step, 3, 12)
    at = 0
    for width in (70, 1, 40, 6, 33):  # 150 together
        logits, lengths = parts.run(ids[:, at: at + width].contiguous(), [width] * 3)
        at += width
        assert lengths.tolist() == [[width] * 3, [at] * 3]
    close(logits, expected, 5e-2)
    assert parts.counters.tolist() == whole.counters.tolist() == [9, 12]
    # Ragged rows of one call are the rows of calls of their own.
    ragged = Loop(step, 3, 12)
    logits, _ = ragged.run(ids, [150, 0, 9])
    close(logits[0], expected[0], 5e-2)
    assert not logits[1].any()
    single = Loop(step, 1, 3)
    close(logits[2:], single.run(ids[2:, :9].contiguous(), [9])[0], 5e-2)


def test_against_the_unmodified_model_over_the_same_format(step, family):
    """transformers' own attention, its cache holding what the format keeps of its keys and values."""
    log(f"paged {family}: unmodified model")
    model = build_model(family)
    ids = tokens(1, 90, 2)
    loop = Loop(step, 1, 3)
    logits, _ = loop.run(ids, [90])

    import model_steps

    class FormatCache(model_steps.ReferenceCache):
        def update(self, key, value, layer_idx, cache_kwargs=None):
            held = oracle.store(key.double().cpu().numpy(), value.double().cpu().numpy())
            key, value = (torch.from_numpy(oracle.values(*x)).to(key) for x in held)
            return super().update(key, value, layer_idx, cache_kwargs)

    plain, model_steps.ReferenceCache = model_steps.ReferenceCache, FormatCache
    try:
        kv_heads, dim = model.config.num_key_value_heads, model.config.head_dim
        caches = tuple(torch.zeros(1, kv_heads, 128, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2 * LAYERS))
        with torch.inference_mode():
            expected = transformers_row_logits(model, ids, torch.arange(90, device="cuda")[None], caches)
    finally:
        model_steps.ReferenceCache = plain
    close(logits, expected, 1e-1)


def test_requests_end_and_a_full_pool_refuses(step, family):
    """Five pages: rows 0 and 1 take four, row 2 waits until row 0 has ended, whose pages it then holds."""
    log(f"paged {family}: full pool")
    loop = Loop(step, 3, 5)
    ids = tokens(3, 100, 3)
    logits, lengths = loop.run(ids, [100, 100, 100])
    assert lengths.tolist() == [[100, 100, 0], [100, 100, 0]] and not logits[2].any() and logits[:2].any()
    before = [t.clone() for t in loop.kv]
    logits, lengths = loop.run(ids[:, :1].contiguous(), [0, 1, 0], after=[0, 101, 0])
    assert lengths.tolist() == [[0, 1, 0], [0, 101, 0]]
    changed = [(a != b).any(dim=tuple(range(1, a.dim()))).nonzero().flatten().tolist() for a, b in zip(before, loop.kv)]
    held = loop.table[1, :2].tolist()
    assert all(set(pages) <= {held[1]} for pages in changed), (changed, held)
    logits, lengths = loop.run(ids, [0, 0, 100])
    assert lengths.tolist() == [[0, 0, 100], [0, 101, 100]]
    assert not set(loop.table[2, :2].tolist()) & set(held)
    fresh = Loop(step, 1, 2)
    close(logits[2:], fresh.run(ids[2:].contiguous(), [100])[0], 5e-2)
    # Drafted tokens taken back: the same row again from token 60.
    again, lengths = loop.run(ids[:, 60:].contiguous(), [0, 0, 40], after=[0, 101, 100])
    assert lengths.tolist() == [[0, 0, 40], [0, 101, 100]]
    close(again[2], logits[2], 5e-2)


def test_captured_decode_generates_the_eager_tokens(step, family):
    """A decode step captured once; its lengths, pages and tokens advance on the device from replay to replay."""
    log(f"paged {family}: captured decode")
    prompts, counts = tokens(2, 80, 4), [80, 61]

    def start():
        loop = Loop(step, 2, 8)
        logits, _ = loop.run(prompts, counts)
        return loop, logits.argmax(-1, keepdim=True)

    eager, ids = start()
    expected = [ids]
    for _ in range(12):
        logits, _ = eager.run(expected[-1], [1, 1])
        expected.append(logits.argmax(-1, keepdim=True))

    loop, ids = start()
    ids, ones = ids.clone(), torch.ones(2, dtype=torch.int32, device="cuda")
    state = (loop.lengths.clone(), loop.counters.clone())

    def one_step():
        logits, lengths, counters = step(ids, state[0], state[0] + ones, ones, loop.kv, state[1], loop.table, loop.ring)
        ids.copy_(logits.argmax(-1, keepdim=True))
        state[0].copy_(lengths[1])
        state[1].copy_(counters)

    with torch.inference_mode():
        saved = [t.clone() for t in (ids, *state, *loop.kv, loop.table, loop.ring)]
        one_step()  # warm
        for t, s in zip((ids, *state, *loop.kv, loop.table, loop.ring), saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_step()
        for t, s in zip((ids, *state, *loop.kv, loop.table, loop.ring), saved):
            t.copy_(s)
        got = [ids.clone()]
        for _ in range(12):
            graph.replay()
            got.append(ids.clone())
            torch.cuda.synchronize()
    assert torch.equal(torch.cat(got, 1), torch.cat(expected, 1))
    assert state[0].tolist() == eager.lengths.tolist() and torch.equal(loop.table, eager.table)


def test_adapters_refuse(step, family):
    from xinfer_amd.adapters import PagedStep

    adapter = step.model.model.layers[0].self_attn
    hidden = torch.zeros(1, 1, 1024, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="PagedStep"):
        adapter(hidden, (hidden, hidden), past_key_values=None)
    state = PagedStep((), torch.zeros(1, 1, dtype=torch.int64), None, None, None)
    with pytest.raises(ValueError, match="attention masks"):
        adapter(hidden, (hidden, hidden), attention_mask=hidden, past_key_values=state)
    with pytest.raises(ValueError, match="same position"):
        adapter(hidden, (hidden, hidden), past_key_values=state, cache_position=torch.zeros(1, 1, dtype=torch.int64))


def test_package_of_a_paged_step(step, family, tmp_path):
    """Exported, compiled with the C shims and loaded again: the eager step's lengths, pages and counters, its logits
    within the bound for other kernels around the native ones."""
    from xinfer_amd.attention import attention_c_shims, attention_library
    from xinfer_amd.package import compile_package, load_package
    from xinfer_amd.paged_kv4 import paged_c_shims

    log(f"paged {family}: package")
    loops = [Loop(step, 2, 6) for _ in range(2)]
    ids, counts = tokens(2, 20, 5), torch.tensor([20, 13], dtype=torch.int32, device="cuda")

    def inputs(loop):
        return (ids, loop.lengths, loop.lengths + counts, counts, loop.kv, loop.counters, loop.table, loop.ring)

    scratch = Loop(step, 2, 6)
    with torch.inference_mode():
        exported = torch.export.export(step, inputs(scratch), strict=False)
        targets = [node.target for node in exported.graph.nodes if node.op == "call_function"]
        ops = torch.ops.xinfer
        assert targets.count(ops.paged_kv_reserve.default) == 1
        assert targets.count(ops.qk_norm_rope_append_kv4.default) == targets.count(ops.paged_attention_kv4.default) == LAYERS
        compile_package(exported, tmp_path / "step.pt2", inductor_configs={"emulate_precision_casts": True},
                        native_libraries=[Path(attention_library())],
                        custom_op_shims={**attention_c_shims(), **paged_c_shims()})
        package = load_package(tmp_path / "step.pt2")
        expected = step(*inputs(loops[0]))
        got = package(*inputs(loops[1]))
    close(got[0], expected[0], 5e-2)
    for a, b in zip((*got[1:], loops[1].table, loops[1].ring), (*expected[1:], loops[0].table, loops[0].ring)):
        assert torch.equal(a, b)
    assert any(t.any() for t in loops[1].kv)
    same = np.mean([torch.equal(a, b) for a, b in zip(loops[1].kv[:4], loops[0].kv[:4])])
    log(f"layer 0 cache tensors equal to eager's: {same:.2f}")
