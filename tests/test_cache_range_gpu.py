"""CacheAttention over the whole range of scores, scales and values, with an allowance that goes by what a row sees."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from . import cache_helpers
from .cache_helpers import Cache, decode, floats
from .node_helpers import as64
from .test_cache_attention_gpu import attend, near

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["short_table", "long_table"])
def table(request, monkeypatch):
    monkeypatch.setattr(cache_helpers, "LEAST_SLOTS", [(1 << 20) * (request.param == "long_table")])
    return request.param


def attention_seen(cache, q, heads, *, window=0, softcap=0.0):
    """attention64, with an allowance that goes by what a row sees: weights are rounded to 11 bits, and to 2^-36 of the row's largest product of a weight and its page's scale."""
    d, group = cache.head, heads // cache.kv_heads
    y, slack = np.zeros((cache.rows, heads, d)), np.zeros((cache.rows, heads, d))
    for i, n in enumerate(cache.new):
        if not n:
            continue
        k, v = cache.tokens(i, cache.past[i] + n)
        slot = np.arange(cache.past[i] + n)
        page, place = cache.table[i, slot // cache.page], slot % cache.page
        codes, scales = decode(cache.v[page, :, :, place], cache.code), cache.vs[page].astype(np.float64)
        for r in range(n):
            own, row = cache.past[i] + r, cache.ends[i] + r
            seen = (slot <= own) & ((slot > own - window) if window else True)
            for h in range(heads):
                g = h // group
                kk, vv, qq = k[seen, g], v[seen, g], q[row, h]
                z = (kk @ qq) / np.sqrt(d)
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                w = np.exp(z - z.max())
                w /= w.sum()
                y[row, h] = w @ vv
                # as in attention64; softcap: a few f32 roundings of the score, each 2^-24 of it
                off = (np.abs(kk).sum(-1) * np.abs(qq).max() * 2.0 ** -22 + np.abs(kk) @ np.abs(qq) * (d + 8) * 2.0 ** -24).max() / np.sqrt(d) + 2.0 ** -20 + np.abs(z).max() * 2.0 ** -20 * bool(softcap)
                slack[row, h] = (w * (2.0 ** -11 + 2 * off)) @ np.abs(vv) + 2.0 ** -36 * (w * scales[seen, g]).max() * np.abs(codes[seen, g]).sum(0)
    return y, slack


def check_seen(ep, cache, heads, dtype, seed, *, sd=1.0, window=0, softcap=0.0):
    q = floats(np.random.default_rng(seed), (cache.rows, heads * cache.head), dtype, sd)
    got, variant = attend(ep, cache, q, dtype, heads, local_window_size=window or -1, softcap=softcap)
    with np.errstate(invalid="ignore", over="ignore"):
        want, slack = attention_seen(cache, as64(q, dtype).reshape(-1, heads, cache.head), heads, window=window, softcap=softcap)
    near(got, want, slack, dtype)
    return variant


@pytest.mark.parametrize("softcap", [1e-46, 1e-39, 1e-20, 1e-3, 0.3, 3.0, 30.0, 1e3, 1e4, 1e6, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("new", [[1, 1], [150, 7]])
def test_softcaps_of_every_size(ep, table, new, softcap):
    """From caps that make attention even to caps that are none."""
    cache = Cache(np.random.default_rng(31), new, [200, 30], E.I8, 1, 64, 64)
    check_seen(ep, cache, 4, E.F16, 32, sd=3.0, softcap=softcap)


KINDS = [([1, 1], [200, 30]), ([150, 7], [200, 30]), ([300], [10]), ([1], [5000]), ([70], [3000])]          # few rows, more, two teams of waves, pieces of either


def check_values_of_size(ep, new, past, size):
    cache = Cache(np.random.default_rng(38), new, past, E.I8, 1, 64, 64)
    cache.vs[:] = np.where(np.isnan(cache.vs), cache.vs, np.float32(size))
    q = floats(np.random.default_rng(39), (cache.rows, 2 * 64), E.BF16)
    got, _ = attend(ep, cache, q, E.BF16, 2)
    want, slack = attention_seen(cache, as64(q, E.BF16).reshape(-1, 2, 64), 2)
    near(got, want, slack + 2.0 ** -133 * (1 + 2.0 ** -3), E.BF16)           # half a step of bf16's smallest numbers is 2^-134, of f32's on the way 2^-150 each


@pytest.mark.parametrize("size", [1e-36, 1e33, 2.4e36])
@pytest.mark.parametrize("new,past", KINDS)
def test_values_as_large_as_they_can_be(ep, table, new, past, size):
    """Values up to the largest that bf16 has are no infinities on the way, nor are small ones nothing."""
    check_values_of_size(ep, new, past, size)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,bits", [([1, 1], 30), ([150, 70], 30), ([150, 70], 60), ([150, 70], 100)])
def test_scales_of_pages_that_a_row_does_not_see(ep, table, new, bits, page, code):
    """Every third page of values has a scale far above the others': rows in front of the first, or with a window behind the last, are as without it."""
    cache = Cache(np.random.default_rng(33), new, [40, 100], code, 1, 64, page)
    for i in range(2):
        live = -(-(cache.past[i] + new[i]) // page)
        cache.vs[cache.table[i, 2:live:3]] *= np.float32(2.0 ** bits)
    check_seen(ep, cache, 4, E.BF16, 34)
    check_seen(ep, cache, 4, E.BF16, 35, window=20)


@pytest.mark.parametrize("new", [[1, 1], [150, 7]])
@pytest.mark.parametrize("bits", [12, 20, 30, 60, 90])
def test_small_pages_that_take_all(ep, table, new, bits):
    """The page that takes nearly all of the weight has by far the smallest scale: its values come out with their digits."""
    cache = Cache(np.random.default_rng(36), new, [200, 96], E.I8, 1, 64, 16)
    # keys: the first page's stand out in element 0
    cache.k[:, :, :, 0] = 0
    for i in range(2):
        cache.k[cache.table[i, 0], :, :, 0] = 100
        cache.ks[cache.table[i, 0]] = 0.02
        cache.vs[cache.table[i, 0]] *= np.float32(2.0 ** -bits)
    q = np.zeros((cache.rows, 2, 64), np.float32)
    q[:, :, 0] = 4 * bits                                        # scores of the first page: bits nats
    q[:, :, 1:] = np.random.default_rng(37).standard_normal((cache.rows, 2, 63)) * 0.1
    q = synth.to_dtype(q.reshape(cache.rows, -1), E.BF16)
    got, _ = attend(ep, cache, q, E.BF16, 2)
    want, slack = attention_seen(cache, as64(q, E.BF16).reshape(-1, 2, 64), 2)
    near(got, want, slack, E.BF16)


@pytest.mark.parametrize("size", [1e-43, 1e-39])
@pytest.mark.parametrize("new,past", KINDS)
def test_scales_below_the_normal_numbers(ep, table, new, past, size):
    """Pages of values whose scale is one of f32's subnormal numbers."""
    check_values_of_size(ep, new, past, size)


@pytest.mark.parametrize("sequences", [65, 100, 130])
def test_pieces_among_many_sequences(ep, sequences):
    """More sequences than a wave looks at at once, some of them long enough to be cut."""
    rng = np.random.default_rng(sequences)
    past = rng.integers(0, 60, sequences)
    past[[3, 64, sequences - 1]] = [4000, 2600, 5100]
    cache = Cache(rng, rng.integers(0, 3, sequences).clip(0, 2) | (past > 1000), past, E.I8, 1, 64, 32)
    assert check_seen(ep, cache, 2, E.F16, 40) == "cache_attention_pieces"
