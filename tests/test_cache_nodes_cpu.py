"""The operators of a paged 8-bit cache on the host: attributes, refusals with their reasons, scratch, and what supports_op says. The GPU's functions are stood for."""
import ctypes as C

import numpy as np
import pytest

from onnx_genai_amd import build
from onnx_genai_amd import ep as E

from .test_allocation_failure_cpu import host_only  # noqa: F401  (the fixture: the library's host sources without a GPU)

HOLD = np.zeros(1 << 22, np.uint8)
NONE = E.TensorView.absent()


@pytest.fixture
def provider(host_only):  # noqa: F811
    p = E.RocmExecutionProvider(0)
    yield p
    p.shutdown()


class Places:
    """Views at places of their own."""

    def __init__(self):
        self.at = (HOLD.ctypes.data + 255) // 256 * 256

    def __call__(self, dtype, shape, shift=0, **kw):
        here = self.at + shift
        self.at += (int(np.prod(shape)) * E._ITEM[dtype] + shift + 511) // 256 * 256
        return E.TensorView(here, dtype, shape, **kw)


def refused(kernel, inputs, outputs, message, **kw):
    with pytest.raises(E.EpError) as e:
        kernel.execute(inputs, outputs, **kw)
    assert e.value.code == 3 and message in e.value.message, e.value.message
    assert e.value.message.startswith(kernel.op_type + ": ")


def swapped(items, i, other):
    items = list(items)
    items[i] = other
    return items


@pytest.mark.parametrize("op_type,attrs,message", [
    ("RotaryEmbedding", dict(), "missing required integer attribute 'head_size'"),
    ("RotaryEmbedding", dict(head_size=1), "head_size must be 2..=65536"),
    ("RotaryEmbedding", dict(head_size=64, num_heads=-1), "num_heads must be"),
    ("RotaryEmbedding", dict(head_size=64, rotary_embedding_dim=33), "rotary_embedding_dim must be even"),
    ("RotaryEmbedding", dict(head_size=64, rotary_embedding_dim=66), "rotary_embedding_dim must be even"),
    ("RotaryEmbedding", dict(head_size=514), "rotary_embedding_dim must be even, 2..=512"),
    ("RotaryEmbedding", dict(head_size=63), "rotary_embedding_dim must be even"),
    ("RotaryEmbedding", dict(head_size=64, interleaved=2), "interleaved must be 0 or 1"),
    ("RotaryEmbedding", dict(head_size=64, scaling=4), "scaling must be 0 (none)"),
    ("RotaryEmbedding", dict(head_size=64, rope_theta=1.0), "rope_theta must be finite and above 1"),
    ("RotaryEmbedding", dict(head_size=64, rope_theta=float("inf")), "rope_theta must be finite and above 1"),
    ("RotaryEmbedding", dict(head_size=64, factor=0.0), "factor must be finite and positive"),
    ("RotaryEmbedding", dict(head_size=64, original_max_position=0), "original_max_position must be positive"),
    ("RotaryEmbedding", dict(head_size=64, scaling=2, low_freq_factor=4.0), "low_freq_factor must be below"),
    ("RotaryEmbedding", dict(head_size=64, scaling=3, beta_slow=32.0), "beta_slow must be positive"),
    ("RotaryEmbedding", dict(head_size=64, attention_factor=float("nan")), "attention_factor must be finite"),
    ("CacheAppend", dict(head_size=64), "missing required integer attribute 'kv_num_heads'"),
    ("CacheAppend", dict(kv_num_heads=2), "missing required integer attribute 'head_size'"),
    ("CacheAppend", dict(kv_num_heads=0, head_size=64), "kv_num_heads must be"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=24), "head_size must be a multiple of 16"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=272), "head_size must be a multiple of 16"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=64, num_heads=-2), "num_heads must be"),
    ("CacheAttention", dict(kv_num_heads=2, head_size=64), "missing required integer attribute 'num_heads'"),
    ("CacheAttention", dict(num_heads=2, head_size=64), "missing required integer attribute 'kv_num_heads'"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2), "missing required integer attribute 'head_size'"),
    ("CacheAttention", dict(num_heads=3, kv_num_heads=2, head_size=64), "num_heads must be a multiple of kv_num_heads"),
    ("CacheAttention", dict(num_heads=0, kv_num_heads=2, head_size=64), "num_heads must be a multiple of kv_num_heads"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=0, head_size=64), "kv_num_heads must be"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=72), "head_size must be 64, 80, 96, 128 or 256"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=64, local_window_size=0), "local_window_size must be -1"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=64, local_window_size=2 ** 31), "local_window_size must be -1"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=64, scale=-1.0), "scale must be finite and not negative"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=64, scale=1e39), "scale must be finite and not negative"),
    ("CacheAttention", dict(num_heads=2, kv_num_heads=2, head_size=64, softcap=float("nan")), "softcap must be finite and not negative"),
    ("CachePages", dict(compact=1), "missing required integer attribute 'page_size'"),
    ("CachePages", dict(page_size=0), "page_size must be 1..=2^20"),
    ("CachePages", dict(page_size=16, compact=2), "compact must be 0 or 1"),
])
def test_attributes(provider, op_type, attrs, message):
    with pytest.raises(E.EpError) as e:
        provider.get_kernel(attrs, op_type=op_type)
    assert message in e.value.message and e.value.message.startswith(op_type + ": ")
    ok, reason = provider.supports_op(attrs, op_type=op_type)
    assert not ok and message in reason


def test_a_shorter_struct_reads_as_absent(provider):
    a = E.make_node_attrs("CacheAttention", {"num_heads": 4, "kv_num_heads": 2, "head_size": 64, "softcap": -1.0})
    h = C.c_void_p()
    assert provider.lib.nxrt_rocm_cache_attention_create(provider.handle, C.byref(a), C.byref(h)).code == 3
    a.struct_size = E.CacheAttentionAttrs.softcap.offset
    assert provider.lib.nxrt_rocm_cache_attention_create(provider.handle, C.byref(a), C.byref(h)).code == 0
    provider.lib.nxrt_rocm_node_release(h)
    for name in ("rotary_embedding", "cache_append", "cache_attention", "cache_pages"):
        assert getattr(provider.lib, f"nxrt_rocm_{name}_create")(provider.handle, None, C.byref(h)).code == 3 and not h.value


CACHE = [((9, 2, 16, 64), E.I8), ((9, 2, 64, 16), E.I8), ((9, 2), E.F32), ((9, 2), E.F32), ((4,), E.I32), ((3,), E.I32), ((3, 5), E.I32)]


@pytest.mark.parametrize("op_type,attrs,inputs,message", [
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.F16), ((5,), E.I64)], ""),
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.F16), ((5,), E.I64), ((9, 32), E.F32), ((9, 32), E.F32)], ""),
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.F16), ((5,), E.I64), ((9, 32), E.F32)], "cos_cache and sin_cache go together"),
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.I8), ((5,), E.I64)], "input must have a float dtype"),
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.F16), ((5,), E.F32)], "position_ids must have dtype Int64 or Int32"),
    ("RotaryEmbedding", dict(head_size=64), [((5, 128), E.F16)], "expected 2..=4 inputs"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=64), [((5, 128), E.F16), ((5, 128), E.F16)] + CACHE, ""),
    ("CacheAppend", dict(kv_num_heads=2, head_size=64), [((5, 128), E.F16), ((5, 128), E.F16)] + swapped(CACHE, 0, ((9, 2, 16, 64), E.U8)), "k_cache must have dtype Int8 or Float8E4M3FN"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=64), [((5, 128), E.I32), ((5, 128), E.F16)] + CACHE, "key must have a float dtype"),
    ("CacheAppend", dict(kv_num_heads=2, head_size=64), CACHE, "expected 9..=9 inputs"),
    ("CacheAttention", dict(num_heads=4, kv_num_heads=2, head_size=64), [((5, 256), E.BF16)] + CACHE, ""),
    ("CacheAttention", dict(num_heads=4, kv_num_heads=2, head_size=64), [((5, 256), E.F32)] + CACHE, "query must have dtype Float16 or BFloat16"),
    ("CacheAttention", dict(num_heads=4, kv_num_heads=2, head_size=64), [((5, 256), E.F16)] + swapped(CACHE, 0, ((9, 2, 16, 64), E.F16)), "k_cache must have dtype Int8 or Float8E4M3FN"),
    ("CachePages", dict(page_size=16), [((3, 5), E.I32), ((3,), E.I32), (None, 0), (None, 0), ((1, 9, 7), E.I8)], ""),
    ("CachePages", dict(page_size=16), [((3, 5), E.I32), ((3,), E.I32)], "expected 5..=14 inputs"),
    ("CachePages", dict(page_size=16), [((3, 5), E.I64), ((3,), E.I32), (None, 0), (None, 0), ((1, 9, 7), E.I8)], "block_table must have dtype Int32"),
])
def test_supports(provider, op_type, attrs, inputs, message):
    ok, reason = provider.supports_op(attrs, inputs, op_type=op_type)
    assert ok == (not message) and message in reason


def test_rotary_refusals(provider):
    k = provider.get_kernel({"head_size": 8, "num_heads": 3, "rotary_embedding_dim": 4}, op_type="RotaryEmbedding")
    at = Places()
    x, p, c, s, y = at(E.F16, (4, 32)), at(E.I64, (4,)), at(E.F32, (10, 2)), at(E.F32, (10, 2)), at(E.F16, (4, 32))
    k.execute([x, p], [y])
    k.execute([x, p, c, s], [y])
    k.execute([x, p], [x])                                    # in place
    k.execute([x, at(E.I32, (1,))], [y])
    refused(k, [x], [y], "expected 2..=4 inputs")
    refused(k, [NONE, p], [y], "input is required")
    refused(k, [x, NONE], [y], "position_ids is required")
    refused(k, [x, p], [NONE], "output is required")
    refused(k, [at(E.I8, (4, 32)), p], [y], "input must have dtype")
    refused(k, [at(E.F16, (4, 23)), p], [y], "must hold num_heads=3 heads of 8")
    refused(k, [x, at(E.I64, (3,))], [y], "position_ids must have one element, or one for each of the 4 rows")
    refused(k, [x, at(E.F32, (4,))], [y], "position_ids must have dtype Int64 or Int32")
    refused(k, [x, p, c], [y], "cos_cache and sin_cache go together")
    refused(k, [x, p, NONE, s], [y], "cos_cache and sin_cache go together")
    refused(k, [x, p, at(E.F32, (10, 4)), s], [y], "cos_cache must have shape [M, 2]")
    refused(k, [x, p, c, at(E.F16, (10, 2))], [y], "sin_cache must have dtype Float32")
    refused(k, [x, p, c, at(E.F32, (9, 2))], [y], "sin_cache must have shape [10, 2]")
    refused(k, [x, p], [at(E.F32, (4, 32))], "output must have dtype")
    refused(k, [x, p], [at(E.F16, (4, 24))], "output must have shape")
    refused(k, [x, p], [E.TensorView(x.data + 64, E.F16, (4, 32))], "output overlaps input")
    refused(k, [x, E.TensorView(y.data, E.I64, (4,))], [y], "output overlaps position_ids")
    refused(k, [at(E.F16, (4, 32), strides=(64, 1)), p], [y], "input must be contiguous")
    refused(k, [at(E.F16, (4, 32), shift=1), p], [y], "input is not aligned to its elements")
    refused(k, [at(E.F16, (2, 4, 3, 8)), at(E.I64, (6,))], [at(E.F16, (2, 4, 3, 8))], "input must have num_heads=3 heads")
    refused(k, [at(E.F16, (2, 3, 3, 9)), at(E.I64, (6,))], [at(E.F16, (2, 3, 3, 9))], "last dimension head_size=8")
    k.execute([at(E.F16, (2, 3, 3, 8)), at(E.I64, (2, 3))], [at(E.F16, (2, 3, 3, 8))])
    k.execute([E.TensorView(None, E.F16, (0, 32)), NONE], [NONE])
    k.release()
    k = provider.get_kernel({"head_size": 8}, op_type="RotaryEmbedding")
    refused(k, [at(E.F16, (4, 20)), p], [y], "must be a multiple of head_size=8")
    refused(k, [E.TensorView(x.data, E.F16, (1, (1 << 20) + 1, 4, 8)), p], [y], "up to 2^20 heads")
    k.release()


def cache_views(at, pages=9, kv=2, page=16, d=64, n=3, width=5, code=E.I8):
    return [at(code, (pages, kv, page, d)), at(code, (pages, kv, d, page)), at(E.F32, (pages, kv)), at(E.F32, (pages, kv)), at(E.I32, (n + 1,)), at(E.I32, (n,)), at(E.I32, (n, width))]


CACHE_REFUSALS = [
    (0, lambda at: NONE, "k_cache is required"),
    (1, lambda at: NONE, "v_cache is required"),
    (2, lambda at: NONE, "k_scale is required"),
    (3, lambda at: NONE, "v_scale is required"),
    (4, lambda at: NONE, "cumulative_lengths is required"),
    (5, lambda at: NONE, "past_lengths is required"),
    (6, lambda at: NONE, "block_table is required"),
    (0, lambda at: at(E.U8, (9, 2, 16, 64)), "k_cache must have dtype Int8 or Float8E4M3FN"),
    (0, lambda at: at(E.I8, (9, 3, 16, 64)), "k_cache must have shape [P, 2, B, 64]"),
    (0, lambda at: at(E.I8, (9, 2, 16, 80)), "k_cache must have shape [P, 2, B, 64]"),
    (0, lambda at: at(E.I8, (9, 2, 24, 64)), "a page must have 16, 32, 64 or 128 tokens"),
    (0, lambda at: at(E.I8, (9, 2, 16, 64), shift=8), "must start at multiples of 16 bytes"),
    (1, lambda at: at(E.F8E4M3, (9, 2, 64, 16)), "v_cache must have dtype Int8"),
    (1, lambda at: at(E.I8, (9, 2, 16, 64)), "v_cache must have shape [9, 2, 64, 16]"),
    (1, lambda at: at(E.I8, (9, 2, 64, 16), shift=4), "must start at multiples of 16 bytes"),
    (2, lambda at: at(E.F16, (9, 2)), "k_scale must have dtype Float32"),
    (2, lambda at: at(E.F32, (9, 1)), "k_scale must have shape [9, 2]"),
    (3, lambda at: at(E.F32, (18,)), "v_scale must have shape [9, 2]"),
    (4, lambda at: at(E.I64, (4,)), "cumulative_lengths must have dtype Int32"),
    (4, lambda at: at(E.I32, (3,)), "cumulative_lengths must have shape [4]"),
    (5, lambda at: at(E.I32, (4,)), "past_lengths must have shape [3]"),
    (6, lambda at: at(E.I32, (15,)), "block_table must have shape [N, W]"),
    (6, lambda at: at(E.I32, (3, 0)), "block_table must have shape [N, W]"),
    (6, lambda at: E.TensorView(HOLD.ctypes.data // 16 * 16 + 16, E.I32, (3, 1 << 26)), "fewer than 2^30 slots"),
    (6, lambda at: E.TensorView(HOLD.ctypes.data // 16 * 16 + 16, E.I32, (1 << 19, 1)), "fewer than 2^20 sequences times key heads"),
    (6, lambda at: at(E.I32, (3, 5), strides=(8, 1)), "block_table must be contiguous"),
    (6, lambda at: at(E.I32, (3, 5), device_index=1), "block_table must live on ROCm device 0"),
]


@pytest.mark.parametrize("i,other,message", CACHE_REFUSALS)
def test_cache_refusals(provider, i, other, message):
    """The same for the node that writes a cache and the one that reads it."""
    at = Places()
    views = cache_views(at)
    bad = swapped(views, i, other(at))
    key, value, y = at(E.F16, (6, 128)), at(E.F16, (6, 128)), at(E.F16, (6, 256))
    append = provider.get_kernel({"kv_num_heads": 2, "head_size": 64}, op_type="CacheAppend")
    append.execute([key, value] + views, views[:4])
    refused(append, [key, value] + bad, bad[:4], message)
    append.release()
    attend = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAttention")
    q = at(E.F16, (6, 256))
    attend.execute([q] + views, [y])
    refused(attend, [q] + bad, [y], message)
    attend.release()


def test_append_refusals(provider):
    at = Places()
    views, key, value = cache_views(at), at(E.F16, (6, 128)), at(E.F16, (6, 128))
    k = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAppend")
    k.execute([at(E.F16, (6, 512)), NONE] + views, views[:4])                    # packed rows
    refused(k, [key, NONE] + views, views[:4], "packed rows (no value) must have shape [T, 512]")
    refused(k, [at(E.F16, (6, 512)), value] + views, views[:4], "key must have shape [T, 128]")
    refused(k, [key, at(E.F16, (5, 128))] + views, views[:4], "value must have shape [6, 128]")
    refused(k, [key, at(E.F32, (6, 128))] + views, views[:4], "value must have dtype Float16")
    refused(k, [at(E.F16, (6, 2, 64)), value] + views, views[:4], "key must have shape [T, 128]")
    refused(k, [key, value] + views, views[:3], "v_scale is required")
    refused(k, [key, value] + views, swapped(views[:4], 0, at(E.I8, (9, 2, 16, 64))), "k_cache is changed where it is")
    refused(k, [key, value] + views, swapped(views[:4], 3, at(E.F32, (9, 2))), "v_scale is changed where it is")
    refused(k, [key, value] + views, [views[1], views[0], *views[2:4]], "is changed where it is")
    same = swapped(views, 3, views[2])                                          # one tensor for both scales
    refused(k, [key, value] + same, same[:4], "overlaps")
    inside = E.TensorView(views[0].data, E.F16, (6, 128))
    refused(k, [inside, value] + views, views[:4], "k_cache overlaps key")
    refused(k, [E.TensorView(key.data, E.F16, (1 << 26, 128)), E.TensorView(value.data, E.F16, (1 << 26, 128))] + views, views[:4], "too many rows")
    refused(k, [key, value] + views[:6], views[:4], "expected 9..=9 inputs")
    k.execute([E.TensorView(None, E.F16, (0, 128)), NONE] + [NONE] * 7, [NONE] * 4)
    k.release()


def test_attention_refusals(provider):
    at = Places()
    views, q, y = cache_views(at), at(E.F16, (6, 256)), at(E.F16, (6, 256))
    k = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAttention")
    k.execute([at(E.F16, (6, 512))] + views, [y])                               # packed rows
    refused(k, [at(E.F16, (6, 384))] + views, [y], "query must have shape [T, 256], or packed [T, 512]")
    refused(k, [at(E.F16, (2, 3, 256))] + views, [y], "query must have shape [T, 256]")
    refused(k, [at(E.F32, (6, 256))] + views, [y], "query must have dtype Float16 or BFloat16")
    refused(k, [q] + views, [at(E.BF16, (6, 256))], "output must have dtype Float16")
    refused(k, [q] + views, [at(E.F16, (6, 512))], "output must have shape [6, 256]")
    refused(k, [q] + views, [q], "output overlaps query")
    refused(k, [q] + views, [], "expected 1..=1 outputs")
    refused(k, [q] + views[:5], [y], "expected 8..=8 inputs")
    for rows in (1 << 27, 1 << 28):
        refused(k, [E.TensorView(q.data, E.F16, (rows, 256))] + views, [y], "too many rows")
    k.execute([E.TensorView(None, E.F16, (0, 256))] + [NONE] * 7, [NONE])
    k.release()


def test_pages_refusals(provider):
    at = Places()
    table, lengths, parents, new = at(E.I32, (3, 5)), at(E.I32, (3,)), at(E.I32, (3,)), at(E.I32, (3,))
    pools = [at(E.I8, (2, 9, 16)), at(E.F32, (2, 9))]
    outs = [at(E.I32, (3, 5)), at(E.I32, (3,)), at(E.I32, (3, 2)), at(E.I32, (2,))]
    k = provider.get_kernel({"page_size": 16}, op_type="CachePages")
    k.execute([table, lengths, parents, new] + pools, outs + pools)
    k.execute([table, lengths, NONE, NONE] + pools, outs + pools)
    refused(k, [NONE, lengths, parents, new] + pools, outs + pools, "block_table is required")
    refused(k, [at(E.I64, (3, 5)), lengths, parents, new] + pools, outs + pools, "block_table must have dtype Int32")
    refused(k, [at(E.I32, (3, 0)), lengths, parents, new] + pools, outs + pools, "block_table must have shape [S, W]")
    refused(k, [table, NONE, parents, new] + pools, outs + pools, "lengths is required")
    refused(k, [table, at(E.I32, (4,)), parents, new] + pools, outs + pools, "lengths must have shape [3]")
    refused(k, [table, lengths, at(E.I64, (3,)), new] + pools, outs + pools, "parents must have dtype Int32")
    refused(k, [table, lengths, parents, at(E.I32, (3, 1))] + pools, outs + pools, "new_tokens must have shape [3]")
    refused(k, [table, lengths, parents, new, pools[0], at(E.F32, (2, 8))], outs + pools, "all pools must have P=9 pages")
    refused(k, [table, lengths, parents, new, at(E.F32, (9,))], outs + pools[:1], "a pool must have shape [L, P, ..]")
    refused(k, [table, lengths, parents, new, NONE], outs + pools[:1], "pool is required")
    refused(k, [table, lengths, parents, new] + pools, outs + [pools[0], at(E.F32, (2, 9))], "pool is changed where it is")
    refused(k, [table, lengths, parents, new] + pools, outs + pools[:1], "pool is required and absent")
    refused(k, [table, lengths, parents, new] + pools[:1], outs + pools, "expected as many outputs as inputs")
    refused(k, [table, lengths, parents, new] + pools, swapped(outs, 0, table) + pools, "next_table overlaps block_table")
    refused(k, [table, lengths, parents, new] + pools, swapped(outs, 1, lengths) + pools, "next_lengths overlaps lengths")
    refused(k, [table, lengths, parents, new] + pools, swapped(outs, 2, at(E.I32, (4, 2))) + pools, "moves must have shape [3, 2]")
    refused(k, [table, lengths, parents, new] + pools, swapped(outs, 3, at(E.I32, (1,))) + pools, "counts must have shape [2]")
    refused(k, [table, lengths, parents, new, pools[0], pools[0]], outs + [pools[0]] * 2, "overlaps")
    big = E.TensorView(pools[0].data, E.I8, (1, (1 << 18) + 1, 1))
    refused(k, [table, lengths, parents, new, big], outs + [big], "a pool may have 1..=262144 pages")
    many = E.TensorView(HOLD.ctypes.data // 16 * 16 + 16, E.I32, (1025, 5))
    refused(k, [many, lengths, parents, new] + pools, outs + pools, "up to 1024 sequences")
    refused(k, [E.TensorView(many.data, E.I32, (1000, 3000000)), lengths, parents, new] + pools, outs + pools, "fewer than 2^31 entries")
    refused(k, [E.TensorView(many.data, E.I32, (2, 1 << 27)), lengths, parents, new] + pools, outs + pools, "fewer than 2^30 tokens a sequence")
    k.execute([E.TensorView(None, E.I32, (0, 5)), NONE, NONE, NONE, NONE], [NONE])
    k.release()
    k = provider.get_kernel({"page_size": 16, "compact": 1}, op_type="CachePages")
    moves = at(E.I32, (4, 2))
    k.execute([table, lengths, NONE, NONE] + pools, swapped(outs, 2, moves) + pools)
    refused(k, [table, lengths, parents, NONE] + pools, swapped(outs, 2, moves) + pools, "do not go with compact=1")
    refused(k, [table, lengths, NONE, new] + pools, swapped(outs, 2, moves) + pools, "do not go with compact=1")
    refused(k, [table, lengths, NONE, NONE] + pools, outs + pools, "moves must have shape [4, 2]")
    k.release()


def test_steps_and_reasons(provider):
    """A call of a node is one step, whatever it launches; no old text is the reason where a node is supported."""
    at = Places()
    views, q, y = cache_views(at), at(E.F16, (6, 256)), at(E.F16, (6, 256))
    k = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAttention")
    before = provider.kernel_launch_count()
    k.execute([q] + views, [y])
    assert provider.kernel_launch_count() == before + 1
    k.release()
    for op_type, attrs in (("RotaryEmbedding", {"head_size": 64}), ("CacheAppend", {"kv_num_heads": 1, "head_size": 64}), ("CacheAttention", {"num_heads": 1, "kv_num_heads": 1, "head_size": 64}),
                           ("CachePages", {"page_size": 16})):
        a = E.make_node_attrs(op_type, attrs)
        reason = C.create_string_buffer(b"left from before", 64)
        assert getattr(provider.lib, f"nxrt_rocm_ep_supports_{E._NODE_OPS[op_type][1]}")(provider.handle, C.byref(a), None, 0, reason, 64) == 1 and reason.value == b""


def test_workspace_requests(provider):
    descs = [((6, 256), E.F16)] + [(s, d) for s, d in CACHE]
    k = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAttention")
    k.workspace_requirement(descs)
    for bad, message in ((descs[:7], "needs the shapes"), (swapped(descs, 7, ((3, 1 << 26), E.I32)), "shapes that no call takes"), (swapped(descs, 0, ((1 << 28, 256), E.F16)), "shapes that no call takes"),
                         (swapped(descs, 7, ((1 << 19, 1), E.I32)), "shapes that no call takes")):
        with pytest.raises(E.EpError, match=message):
            k.workspace_requirement(bad)
    k.release()
    k = provider.get_kernel({"page_size": 16}, op_type="CachePages")
    with pytest.raises(E.EpError, match="needs the shape of a pool"):
        k.workspace_requirement([((3, 5), E.I32), ((3,), E.I32)])
    k.release()


class Cache(C.Structure):
    """RocmCache of csrc/hip_ffi.h."""
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "ends", "past", "table")] + [("pages", C.c_int64)] + \
               [(n, C.c_int) for n in ("sequences", "width", "page", "kv_heads", "head_size", "code_dtype")]


class AttentionArgs(C.Structure):
    """RocmCacheAttentionArgs of csrc/hip_ffi.h."""
    _fields_ = [("cache", Cache), ("q", C.c_void_p), ("y", C.c_void_p), ("rows", C.c_int64), ("q_step", C.c_int64), ("heads", C.c_int), ("dtype", C.c_int), ("window", C.c_int),
                ("scale", C.c_float), ("softcap", C.c_float)]


@pytest.mark.parametrize("rows,sequences,heads,kv_heads,width", [(1, 1, 32, 8, 2048), (64, 64, 32, 8, 256), (1, 1, 28, 4, 16), (8192, 1, 32, 8, 128), (1111, 3, 14, 2, 257), (4, 1, 128, 1, 4096)])
def test_the_built_library_plans_scratch(rows, sequences, heads, kv_heads, width):
    """What joins pieces of long contexts takes stays within some tens of MB, and nothing where no call splits."""
    lib = C.CDLL(build.LIB)
    lib.rocm_cache_attention_workspace_bytes.restype = C.c_uint64
    a = AttentionArgs()
    a.rows, a.heads = rows, heads
    a.cache.sequences, a.cache.width, a.cache.page, a.cache.kv_heads, a.cache.head_size = sequences, width, 64, kv_heads, 128
    assert lib.rocm_cache_attention_workspace_bytes(C.byref(a)) <= 256 << 20
    a.rows = 0
    assert lib.rocm_cache_attention_workspace_bytes(C.byref(a)) == 0
    a.rows, a.cache.width = rows, 1
    a.cache.page = 16
    assert lib.rocm_cache_attention_workspace_bytes(C.byref(a)) == 0
