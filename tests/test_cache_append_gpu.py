"""CacheAppend against its definition, bit for bit: fresh and begun pages, both code types, what it leaves alone."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .cache_helpers import Cache, append32, floats, same_values
from .node_helpers import Device

pytestmark = pytest.mark.gpu


def check(got, want, code):
    for name, g, w in zip(("k", "v"), got, (want.k, want.v)):
        assert same_values(g, w, code), name
    for name, g, w in zip(("k_scale", "v_scale"), got[2:], (want.ks, want.vs)):
        assert np.array_equal(g, w, equal_nan=True), name


def append(ep, cache, key, value, dtype, *, heads=0, packed=False, offset=0, past=None, table=None, ends=None):
    """Runs the node on a copy of the cache on the GPU; keys and values [T, kv_heads * head] as stored."""
    dev = Device(ep)
    try:
        kernel = ep.get_kernel({"num_heads": heads, "kv_num_heads": cache.kv_heads, "head_size": cache.head}, op_type="CacheAppend")
        views = cache.views(dev)
        for at, other in ((4, ends), (5, past), (6, table)):
            if other is not None:
                views[at] = dev.view(np.asarray(other, np.int32), E.I32)
        if packed:
            queries = np.full((key.shape[0], heads * cache.head), 7, key.dtype)
            rows = [dev.view(np.concatenate([queries, key, value], -1), dtype, offset=offset), E.TensorView.absent()]
        else:
            rows = [dev.view(key, dtype, offset=offset), dev.view(value, dtype, offset=offset)]
        kernel.execute(rows + views, views[:4])
        got = cache.read(ep, views)
        assert kernel.last_variant() == ("cache_append_int8" if cache.code == E.I8 else "cache_append_e4m3")
        kernel.release()
        return got
    finally:
        dev.free()


def rows_of(rng, cache, dtype, extra=0):
    return [floats(rng, (cache.rows + extra, cache.kv_heads * cache.head), dtype, sd) for sd in (1.0, 0.3)]


def as_heads(x, cache, dtype):
    return synth.to_f32(x, dtype).reshape(-1, cache.kv_heads, cache.head)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("page,head,kv_heads", [(16, 64, 2), (32, 80, 1), (64, 128, 4), (128, 256, 2), (64, 16, 3), (128, 96, 1)])
def test_ragged(ep, page, head, kv_heads, dtype, code):
    """None, one or many new tokens; pages that are new, begun, filled to the end or run over; rows behind the last sequence."""
    rng = np.random.default_rng(page + head)
    cache = Cache(rng, [1, 0, 3, page, 5 * page + 7, 1, page - 1], [0, 5, page - 1, 2 * page, 13, 3 * page - 1, 1], code, kv_heads, head, page, width=12, fill=False)
    key, value = rows_of(rng, cache, dtype, extra=3)
    got = append(ep, cache, key, value, dtype, offset=1)
    append32(cache, as_heads(key, cache, dtype), as_heads(value, cache, dtype))
    check(got, cache, code)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
def test_token_by_token(ep, code):
    """One token at a time into a page: scales grow now and then, and the tokens before stay within half a step of each scale they went through."""
    rng = np.random.default_rng(5)
    page, head = 32, 64
    start = Cache(rng, [page], [0], code, 1, head, page, fill=False)
    key, value = rows_of(rng, start, E.F16)
    grown = 0
    allowed = np.zeros(page)
    for t in range(page):
        step = start
        step.new, step.past, step.ends, step.past_lengths = [1], [t], np.array([0, 1], np.int32), np.array([t], np.int32)
        before = step.ks.copy()
        got = append(ep, step, key[t:t + 1], value[t:t + 1], E.F16)
        append32(step, as_heads(key[t:t + 1], step, E.F16), as_heads(value[t:t + 1], step, E.F16))
        check(got, step, code)
        p = step.table[0, 0]
        if t == 0 or step.ks[p, 0] != before[p, 0]:
            grown += 1
            allowed[:t] += step.ks[p, 0] / 2
            allowed[t] += step.ks[p, 0] / 2
        else:
            allowed[t] = step.ks[p, 0] / 2
    assert 1 < grown < page
    if code == E.I8:
        k, _ = start.tokens(0, page)
        assert (np.abs(k[:, 0] - as_heads(key, start, E.F16)[:, 0]) <= allowed[:, None] * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
def test_packed_rows(ep, code):
    rng = np.random.default_rng(6)
    cache = Cache(rng, [70, 1], [10, 64], code, 2, 64, 64, fill=False)
    key, value = rows_of(rng, cache, E.BF16)
    got = append(ep, cache, key, value, E.BF16, heads=6, packed=True, offset=3)
    append32(cache, as_heads(key, cache, E.BF16), as_heads(value, cache, E.BF16))
    check(got, cache, code)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinities_and_nan(ep, bad, code):
    """They take the scale of their page and head, keys or values, and no other's; the page stays so until it begins again."""
    rng = np.random.default_rng(7)
    cache = Cache(rng, [4, 70], [10, 0], code, 2, 64, 64, fill=False)
    key, value = rows_of(rng, cache, E.F32)
    key[2, 64 + 5] = bad                       # sequence 0, head 1
    value[4 + 66, 3] = bad                     # sequence 1, second page, head 0
    got = append(ep, cache, key, value, E.F32)
    append32(cache, as_heads(key, cache, E.F32), as_heads(value, cache, E.F32))
    check(got, cache, code)
    first, second = cache.table[0, 0], cache.table[1, 1]
    assert np.isnan(got[2][first]).tolist() == [False, True] and not np.isnan(got[3][first]).any() and np.isnan(got[3][second]).tolist() == [True, False]
    # more tokens: still NaN; a page that begins again: not
    cache.new, cache.past, cache.ends, cache.past_lengths = [1, 1], [14, 64], np.array([0, 1, 2], np.int32), np.array([14, 64], np.int32)
    key, value = rows_of(rng, cache, E.F32)
    got = append(ep, cache, key, value, E.F32)
    append32(cache, as_heads(key, cache, E.F32), as_heads(value, cache, E.F32))
    check(got, cache, code)
    assert np.isnan(got[2][first, 1]) and not np.isnan(got[3][second, 0])


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("size", [0.0, 1e-45, 3e-39, 1e-30, 1e30, 3e38])
def test_scales_from_zero_to_the_largest(ep, size, code):
    rng = np.random.default_rng(8)
    cache = Cache(rng, [20, 1], [0, 5], code, 1, 64, 16, fill=False)
    key, value = ((rng.uniform(-1, 1, (cache.rows, 64)) * size).astype(np.float32) for _ in range(2))
    got = append(ep, cache, key, value, E.F32)
    with np.errstate(all="ignore"):
        append32(cache, key.reshape(-1, 1, 64), value.reshape(-1, 1, 64))
    check(got, cache, code)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
def test_half_way_values(ep, code):
    """Quotients half-way between codes, and next to it."""
    cache = Cache(np.random.default_rng(0), [64], [0], code, 1, 256, 64, fill=False)
    top = 127.0 if code == E.I8 else 448.0
    for scale in (1.0, 0.1, 3.7e-3):
        if code == E.I8:
            steps = np.concatenate([np.arange(-126.5, 127), np.nextafter(np.arange(-126.5, 127), 0)])
        else:
            v = np.unique(np.abs(np.nan_to_num(np.array([decoded for decoded in np.unique(same_table())]))))
            middle = (v[1:] + v[:-1]) / 2
            steps = np.concatenate([middle, -middle, np.nextafter(middle.astype(np.float32), np.float32(0)), v])
        x = np.resize(steps, 64 * 256).astype(np.float32) * np.float32(scale)
        x[0] = top * np.float32(scale)
        key = np.clip(x, -top * scale, top * scale).astype(np.float32).reshape(64, 256)
        got = append(ep, cache, key, -key, E.F32)
        want = Cache(np.random.default_rng(0), [64], [0], code, 1, 256, 64, fill=False)
        append32(want, key.reshape(-1, 1, 256), -key.reshape(-1, 1, 256))
        check(got, want, code)


def same_table():
    from .cache_helpers import E4M3
    return E4M3[:127]


def test_tables_that_lead_nowhere(ep):
    """Pages outside the pool, past lengths and ends out of range: those tokens are dropped, and nothing else is touched."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [2, 2, 2, 2], [0, 0, 0, 0], E.I8, 1, 64, 16, fill=False)
    before = [x.copy() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    key, value = rows_of(rng, cache, E.F16)
    table = cache.table.copy()
    table[:, 0] = [-1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31]
    got = append(ep, cache, key, value, E.F16, table=table)
    for g, b in zip(got, before):
        assert np.array_equal(g.view(np.uint8), b.view(np.uint8))
    got = append(ep, cache, key, value, E.F16, past=[16, 2 ** 31 - 1, 16, 99])             # behind the table's width
    for g, b in zip(got, before):
        assert np.array_equal(g.view(np.uint8), b.view(np.uint8))
    got = append(ep, cache, key, value, E.F16, ends=[-5, -3, 0, -9, -2 ** 31])             # no row for anyone
    for g, b in zip(got, before):
        assert np.array_equal(g.view(np.uint8), b.view(np.uint8))
    # ends beyond the rows are the rows; falling ones are empty sequences
    got = append(ep, cache, key, value, E.F16, ends=[0, 2, 1, 99, 99], past=[-3, 0, 0, 0])
    want = Cache(np.random.default_rng(9), [2, 2, 2, 2], [0, 0, 0, 0], E.I8, 1, 64, 16, fill=False)
    want.new, want.ends = [2, 0, 7, 0], np.array([0, 2, 1, 8, 8], np.int32)
    append32(want, as_heads(key, want, E.F16), as_heads(value, want, E.F16))
    check(got, want, E.I8)


@pytest.mark.parametrize("sequences", [65, 130, 1000])
def test_many_sequences(ep, sequences):
    """More than a wave looks at once, some without tokens."""
    rng = np.random.default_rng(sequences)
    new = rng.integers(0, 3, sequences)
    cache = Cache(rng, new, rng.integers(0, 33, sequences), E.I8, 1, 16, 16, width=4, fill=False)
    key, value = rows_of(rng, cache, E.F16)
    got = append(ep, cache, key, value, E.F16)
    append32(cache, as_heads(key, cache, E.F16), as_heads(value, cache, E.F16))
    check(got, cache, E.I8)
