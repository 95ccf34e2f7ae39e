"""The paged 4-bit KV cache without a GPU: refusals, workspace sizes, fakes, and the oracle's own known answers.

Every C-ABI call below fails validation or only asks a size, so no HIP call is made.
"""

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import kv4 as oracle

ARGUMENT, LAYOUT, EPS, SCALE, HEADS, WORKSPACE, CACHE, SHAPE, PAGES = 14, 11, 16, 7, 4, 10, 19, 20, 21
BASE = 1 << 20


class View4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("size", ctypes.c_int64 * 4), ("stride", ctypes.c_int64 * 4)]


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("key", "key_scale", "value", "value_scale")] + [
        (n, ctypes.c_int64) for n in ("pages", "kv_heads", "page_size", "dim")]


def view(*sizes, strides=None, data=BASE):
    strides = strides or [sizes[1] * sizes[2] * sizes[3], sizes[2] * sizes[3], sizes[3], 1]
    return ctypes.byref(View4(data, (ctypes.c_int64 * 4)(*sizes), (ctypes.c_int64 * 4)(*strides)))


def cache(pages=10, kv_heads=8, page_size=64, dim=128, data=BASE):
    return ctypes.byref(Cache(data, BASE, BASE, BASE, pages, kv_heads, page_size, dim))


@pytest.fixture(scope="module")
def lib(library_path):
    torch.ops.load_library(str(library_path))
    handle = ctypes.CDLL(str(library_path))
    handle.xinfer_status_string.restype = ctypes.c_char_p
    handle.xinfer_paged_attention_kv4_workspace_size.restype = ctypes.c_size_t
    return handle


I64, F64, PTR = ctypes.c_int64, ctypes.c_double, ctypes.c_void_p


def test_messages(lib):
    for code, start in ((CACHE, "Expected a 4-bit KV cache"), (SHAPE, "Tensors do not match"), (PAGES, "Expected pages of 64")):
        assert lib.xinfer_status_string(code).decode().startswith(start)


def test_reserve_refusals(lib):
    def call(rows=4, tokens=2, size=64, width=8, ring=100, pointer=BASE, counters=BASE, after=2 * BASE):
        return lib.xinfer_paged_kv_reserve(PTR(pointer), PTR(BASE), PTR(BASE), I64(rows), I64(tokens), I64(size),
                                           PTR(counters), PTR(BASE), I64(width), PTR(BASE), I64(ring), PTR(BASE), PTR(BASE),
                                           PTR(BASE), PTR(after), None)

    assert call(size=32) == call(size=96) == call(size=512) == call(size=0) == PAGES
    assert call(width=0) == call(width=(1 << 24) + 1) == call(ring=0) == call(ring=1 << 31) == PAGES
    assert call(rows=1 << 29) == PAGES
    assert call(rows=65536, width=1) == ARGUMENT
    assert call(rows=-1) == call(tokens=-1) == call(pointer=0) == call(counters=0) == call(after=BASE) == ARGUMENT


def test_append_and_read_refusals(lib):
    def append(key=view(2, 8, 3, 128), value=view(2, 8, 3, 128), slots=BASE, held=cache()):
        return lib.xinfer_append_kv4(key, value, PTR(slots), I64(3), I64(1), held, None)

    for held in (cache(dim=96), cache(page_size=32), cache(pages=0), cache(kv_heads=0), cache(data=BASE + 8), cache(data=0)):
        assert append(held=held) == CACHE
        assert lib.xinfer_read_kv4(held, PTR(BASE), I64(3), I64(1), I64(2), I64(3), PTR(BASE), PTR(BASE), None) == CACHE
    assert append(key=view(2, 4, 3, 128)) == append(value=view(2, 8, 4, 128)) == append(key=view(2, 8, 3, 64)) == SHAPE
    assert append(view(1 << 20, 8, 1 << 20, 128), view(1 << 20, 8, 1 << 20, 128)) == SHAPE
    # A launch's threads are counted in 32 bits: 16 for each of 2^28 rows.
    assert append(view(1 << 12, 8, 1 << 13, 128), view(1 << 12, 8, 1 << 13, 128)) == SHAPE
    assert append(slots=0) == append(key=None) == append(held=None) == ARGUMENT
    odd = view(2, 8, 3, 128, strides=[8 * 3 * 132, 3 * 132, 132, 1])
    assert append(odd) == append(view(2, 8, 3, 128, data=BASE + 2)) == append(view(2, 8, 3, 128, strides=[9, 9, 9, 2])) == LAYOUT
    assert append(view(0, 8, 3, 128), view(0, 8, 3, 128), slots=0) == 0  # nothing to do
    read = lambda *a: lib.xinfer_read_kv4(cache(), *a, None)  # noqa: E731
    assert read(PTR(BASE), I64(3), I64(1), I64(-2), I64(3), PTR(BASE), PTR(BASE)) == SHAPE
    assert read(None, I64(3), I64(1), I64(2), I64(3), PTR(BASE), PTR(BASE)) == ARGUMENT
    assert read(PTR(BASE), I64(3), I64(1), I64(2), I64(3), PTR(BASE + 8), PTR(BASE)) == LAYOUT


def test_norm_rope_refusals(lib):
    def call(q=view(2, 16, 3, 128), key=view(2, 8, 3, 128), rope=view(2, 1, 3, 128), eps=1e-6, offset=0.0, slots=BASE,
             weight=BASE, held=cache()):
        return lib.xinfer_qk_norm_rope_append_kv4(q, key, key, PTR(weight), PTR(BASE), F64(eps), F64(offset), rope, rope,
                                                  PTR(slots), I64(3), I64(1), PTR(BASE), held, None)

    assert call(held=cache(dim=80)) == CACHE
    assert call(q=view(2, 16, 4, 128)) == call(q=view(2, 16, 3, 64)) == call(key=view(2, 4, 3, 128)) == SHAPE
    for width in (0, 8, 24, 144):
        assert call(rope=view(2, 1, 3, width)) == SHAPE
    assert call(rope=view(2, 2, 3, 128)) == call(rope=view(2, 1, 4, 128)) == SHAPE
    assert call(eps=-1.0) == call(eps=float("nan")) == EPS
    wide = [view(1 << 12, heads, 1 << 13, 128) for heads in (1, 8)]
    assert call(q=wide[0], key=wide[1], rope=view(1 << 12, 1, 1 << 13, 128)) == SHAPE
    assert call(offset=float("inf")) == call(slots=0) == call(weight=0) == ARGUMENT
    assert call(weight=BASE + 2) == call(q=view(2, 16, 3, 128, data=BASE + 4)) == LAYOUT


def test_attention_refusals_and_workspace(lib):
    def call(q=view(2, 16, 1, 128), held=cache(), width=8, longest=0, scale=0.1, workspace=BASE, size=1 << 40, table=BASE):
        return lib.xinfer_paged_attention_kv4(q, held, PTR(table), I64(width), PTR(BASE), I64(longest), F64(scale), PTR(BASE),
                                              PTR(workspace), ctypes.c_size_t(size), None)

    assert call(held=cache(page_size=16)) == CACHE
    assert call(view(2, 16, 1, 64)) == call(view(65536, 16, 1, 128)) == call(view(2, 16, 1 << 30, 128)) == SHAPE
    assert call(view(65535, 1024, 1, 128), cache(kv_heads=64), width=256) == SHAPE  # the merge's threads
    assert call(view(2, 12, 1, 128)) == call(view(2, 0, 1, 128)) == HEADS
    assert call(width=0) == call(width=(1 << 24) + 1) == call(longest=-1) == PAGES
    assert call(scale=0.0) == call(scale=float("inf")) == call(scale=float("nan")) == SCALE
    assert call(table=0) == call(q=None) == ARGUMENT
    assert call(view(2, 16, 1, 128, strides=[2052, 132, 128, 1])) == LAYOUT

    size = lambda q, held, width, longest: lib.xinfer_paged_attention_kv4_workspace_size(  # noqa: E731
        q, held, I64(width), I64(longest))
    # Rows of up to 512 keys are never cut; longer ones need records, however short the lengths turn out.
    assert size(view(8, 16, 1, 128), cache(), 8, 0) == size(view(8, 16, 1, 128), cache(), 100, 512) == 0
    decode = size(view(8, 16, 1, 128), cache(), 256, 0)
    assert decode == (64 + 1024) * 16 * 130 * 4
    assert call(view(8, 16, 1, 128), width=256, size=decode - 1) == call(view(8, 16, 1, 128), width=256, workspace=BASE + 8) == WORKSPACE
    assert size(view(8, 16, 512, 128), cache(), 256, 0) > decode
    # Records are those of cut rows, which are fewer than twice the items aimed at, whatever the batch.
    assert size(view(64, 16, 8192, 128), cache(), 1024, 0) <= 2 * (768 * 128 + 256 * 32) * 130 * 4
    assert size(view(4096, 16, 1, 128), cache(), 1024, 0) <= 2 * 1024 * 16 * 130 * 4


def test_operators_check_their_tensors(library_path):
    from xinfer_amd.attention import load_attention_ops
    from xinfer_amd import paged_kv4 as ops

    load_attention_ops(library_path)
    with pytest.raises(ValueError, match="page size"):
        ops.paged_kv4_cache(4, 8, 48, 128, "cpu")
    with pytest.raises(ValueError, match="head dimension"):
        ops.paged_kv4_cache(4, 8, 64, 96, "cpu")
    shapes = [tuple(t.shape) for t in ops.paged_kv4_cache(3, 8, 128, 256, "cpu")]
    assert shapes == [(3, 8, 128, 128), (3, 8, 8, 128)] * 2
    assert len(ops.paged_c_shims()) == 5
    assert all(f"aoti_torch_cuda_{name}" in text for name, text in ops.PAGED_C_SHIMS.items())
    with FakeTensorMode(allow_non_fake_inputs=True):
        options = dict(device="cuda")
        rows = torch.empty(3, dtype=torch.int32, **options)
        held = [torch.empty(s, dtype=torch.uint8, **options) for s in ((5, 8, 64, 64), (5, 8, 4, 64)) * 2]
        table = torch.empty(3, 7, dtype=torch.int32, **options)
        lengths, positions, slots, counters = ops.paged_kv_reserve(
            rows, rows, rows, 2, 64, torch.empty(2, dtype=torch.int64, **options), table,
            torch.empty(9, dtype=torch.int32, **options))
        assert lengths.shape == (2, 3) and positions.shape == slots.shape == (3, 2) and counters.shape == (2,)
        key = torch.empty(3, 8, 2, 128, dtype=torch.bfloat16, **options)
        assert ops.append_kv4(key, key, slots, held) is None
        assert [t.shape for t in ops.read_kv4(held, slots)] == [(3, 8, 2, 128)] * 2
        q = torch.empty(3, 2, 16, 128, dtype=torch.bfloat16, **options)
        weight, rope = torch.empty(128, dtype=torch.bfloat16, **options), torch.empty(3, 2, 64, dtype=torch.bfloat16, **options)
        kv = key.transpose(1, 2)
        q = ops.qk_norm_rope_append_kv4(q, kv, kv, weight, weight, 1e-6, 1.0, rope, rope, slots, held)
        assert q.shape == (3, 16, 2, 128)
        assert ops.paged_attention_kv4(q, held, table, lengths, 0, 0.1).shape == (3, 2, 16, 128)
        with pytest.raises(Exception):
            ops.paged_attention_kv4(q, held, table[:2], lengths, 0, 0.1)
        with pytest.raises(Exception):
            ops.append_kv4(key, key, slots[:, :1], held)


# ---- the oracle's known answers


def test_format_known_answers():
    x = np.zeros(32)
    x[:10] = [6.0, 5.0, 2.5, 0.25, 0.75, 1.25, -1.75, 3.5, 5.000001, 0.2]
    (codes, scale), _ = oracle.store(x, x)
    assert scale.tolist() == [127] and codes[:10].tolist() == [7, 6, 4, 0, 2, 2, 12, 6, 7, 0]
    # 7 is half way between this power's 6 and the next one's 8: it stays, anything above moves up.
    for top, exponent, held in ((7.0, 0, 6.0), (7.0000001, 1, 8.0), (7.99, 1, 8.0), (8.0, 1, 8.0), (2.0**-140, -125, 0.0)):
        y = np.zeros(32)
        y[3] = top
        (codes, scale), _ = oracle.store(y, y)
        assert scale.tolist() == [exponent + 127] and oracle.values(codes, scale)[3] == held
    bad = x.copy()
    bad[0] = np.inf
    (codes, scale), (value_codes, value_scale) = oracle.store(bad, x)
    assert scale.tolist() == [255] and value_scale.tolist() == [2] and not codes.any() and not value_codes.any()
    assert np.isnan(oracle.values(codes, scale)).all()


def test_attention_of_one_key_and_of_none():
    caches = [np.full(s, b, np.uint8) for s, b in (((2, 1, 64, 32), 0x22), ((2, 1, 2, 64), 127), ((2, 1, 64, 32), 0x75), ((2, 1, 2, 64), 128))]
    q = np.ones((2, 2, 1, 64))
    out = oracle.attention(q, caches, np.array([[1], [-1]]), np.array([[1, 1], [1, 5]]), 0.3)
    assert (out[0, 0, :, 0::2] == 6.0).all() and (out[0, 0, :, 1::2] == 12.0).all() and not out[1].any()
