"""CacheAttention against its definition in 64 bits: head layouts, lengths, pages, windows, what masks leave, and pieces of long contexts."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E

from . import cache_helpers
from .cache_helpers import Cache, attention64, floats
from .node_helpers import EPS, Device, as64

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["short_table", "long_table"])
def table(request, monkeypatch):
    """Few rows in all go in small tiles where the table is short, and prompts of 65 rows and more in large ones where it has room for a million tokens."""
    monkeypatch.setattr(cache_helpers, "LEAST_SLOTS", [(1 << 20) * (request.param == "long_table")])
    return request.param


def attend(ep, cache, q, dtype, heads, *, offset=0, packed=False, extra=0, views=None, dev=None, **attrs):
    own = dev is None
    dev = dev or Device(ep)
    try:
        kernel = ep.get_kernel({"num_heads": heads, "kv_num_heads": cache.kv_heads, "head_size": cache.head, **attrs}, op_type="CacheAttention")
        rows, wide = q.shape
        source = q
        if packed:
            source = np.concatenate([q, np.full((rows, 2 * cache.kv_heads * cache.head), 0x7E00 if dtype == E.F16 else 0x7FC0, np.uint16).view(q.dtype)], -1)
        y, read = dev.output((rows, wide), dtype, offset)
        fill = read().copy()
        kernel.execute([dev.view(source, dtype, offset=offset)] + (views or cache.views(dev)), [y])
        ep.sync()
        got, variant = read().copy(), kernel.last_variant()
        kernel.release()
        used = rows - extra
        assert np.array_equal(got[used:].view(np.uint16), fill[used:].view(np.uint16)), "rows of no sequence are written"
        return got[:used].reshape(used, heads, cache.head), variant
    finally:
        if own:
            dev.free()


def near(got, want, slack, dtype):
    error = np.abs(as64(got, dtype) - want)
    allowed = EPS[dtype] / 2 * np.abs(want) * (1 + 2.0 ** -8) + slack + (2.0 ** -24 if dtype == E.F16 else 0)
    assert (error <= allowed).all(), (float((error / allowed).max()), np.argwhere(error > allowed)[:5].tolist())


def check(ep, cache, heads, dtype, seed, *, sd=1.0, extra=0, packed=False, offset=0, window=0, softcap=0.0, scale=0.0):
    rng = np.random.default_rng(seed)
    q = floats(rng, (cache.rows + extra, heads * cache.head), dtype, sd)
    attrs = {"local_window_size": window or -1, "softcap": softcap, "scale": scale}
    got, variant = attend(ep, cache, q, dtype, heads, extra=extra, packed=packed, offset=offset, **attrs)
    with np.errstate(invalid="ignore"):
        want, slack = attention64(cache, as64(q, dtype).reshape(-1, heads, cache.head), heads, window=window, softcap=softcap, scale=scale)
    near(got, want, slack, dtype)
    return variant


@pytest.mark.parametrize("dtype", [E.F16, E.BF16])
@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("head,page,kv_heads,group", [(64, 16, 2, 7), (80, 32, 1, 1), (96, 64, 2, 4), (128, 64, 4, 7), (128, 16, 1, 16), (128, 128, 2, 3), (256, 32, 1, 2), (64, 128, 3, 17), (80, 16, 2, 5)])
def test_single_tokens(ep, head, page, kv_heads, group, code, dtype):
    """The next token of sequences from no past at all to several steps of 64 tokens, a sequence without one, rows behind the last."""
    rng = np.random.default_rng(head + page + group)
    cache = Cache(rng, [1, 1, 0, 1, 1, 1, 1], [0, 1, 9, 63, 64, 331, 15], code, kv_heads, head, page, width=31)
    check(ep, cache, kv_heads * group, dtype, 1, extra=2)


@pytest.mark.parametrize("dtype", [E.F16, E.BF16])
@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("head,page,kv_heads,group", [(64, 16, 2, 7), (128, 64, 2, 4), (80, 32, 1, 1), (96, 128, 1, 3), (256, 64, 1, 2), (128, 32, 1, 48)])
def test_chunks(ep, table, head, page, kv_heads, group, code, dtype):
    """Prompts and chunks behind a past, ragged, with tiles that begin inside a token's heads."""
    rng = np.random.default_rng(head + page)
    cache = Cache(rng, [70, 1, 0, 33, 5], [0, 100, 3, 129, 64], code, kv_heads, head, page, width=20)
    check(ep, cache, kv_heads * group, dtype, 2, extra=1, packed=True, offset=1)


KINDS = {
    # (new tokens of the sequences, past, heads, key heads): what the call's size makes of it on 256 CUs
    "few_rows_four_waves": ([1] * 139 + [2], [17 * i % 300 for i in range(140)], 8, 2),
    "tiles_of_128": ([900, 0, 203], [70, 5, 333], 64, 2),
    "tiles_of_256": ([1500, 1, 650], [0, 900, 129], 64, 2),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("head,page,code,window", [(64, 16, E.I8, 0), (64, 64, E.F8E4M3, 0), (80, 32, E.I8, 100), (80, 128, E.F8E4M3, 0), (96, 64, E.I8, 0), (96, 16, E.F8E4M3, 0), (128, 16, E.F8E4M3, 77),
                                                   (128, 64, E.I8, 0), (128, 128, E.F8E4M3, 500), (128, 32, E.I8, 0), (256, 16, E.I8, 0), (256, 64, E.F8E4M3, 0)])
def test_tiles_of_every_kind(ep, kind, head, page, code, window):
    """Calls large enough for the kernels of many tiles; some rows of every sequence, its first and last among them, against the definition."""
    new, past, heads, kv_heads = KINDS[kind]
    rng = np.random.default_rng(head + page)
    cache = Cache(rng, new, past, code, kv_heads, head, page)
    q = floats(rng, (cache.rows + 1, heads * head), E.F16)
    got, variant = attend(ep, cache, q, E.F16, heads, extra=1, local_window_size=window or -1)
    assert variant.startswith("cache_attention_rows") == (kind != "few_rows_four_waves")
    rows = set(rng.integers(0, cache.rows, 12).tolist()) | {int(e) for e in cache.ends[:-1] if e < cache.rows} | {int(e) - 1 for e in cache.ends[1:]} if len(new) < 9 else set(range(0, cache.rows, 5))
    of_heads = [0, heads // kv_heads - 1, heads - 1]
    want, slack = attention64(cache, as64(q, E.F16).reshape(-1, heads, head), heads, window=window, rows=rows, of_heads=of_heads)
    at = np.ix_(sorted(rows), of_heads)
    near(got[at], want[at], slack[at], E.F16)


@pytest.mark.parametrize("rows", [1, 2, 64, 65, 127, 128, 129, 200, 257])
@pytest.mark.parametrize("group", [1, 4])
def test_prompt_lengths(ep, table, rows, group):
    rng = np.random.default_rng(rows)
    cache = Cache(rng, [rows], [0], E.I8, 1, 64, 16)
    variant = check(ep, cache, group, E.F16, 3)
    assert variant.startswith("cache_attention_rows") == (table == "long_table" and rows * group > 64)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("new,heads", [([1, 1, 1], 6), ([40, 1, 90], 6), ([40, 1, 90], 132)])
def test_windows(ep, new, heads, window):
    rng = np.random.default_rng(window)
    cache = Cache(rng, new, [200, 0, 65], E.F8E4M3, 2, 64, 32)
    assert check(ep, cache, heads, E.BF16, 4, window=window).startswith("cache_attention_rows") == (heads == 132)


@pytest.mark.parametrize("new", [[1, 1], [150, 7]])
def test_softcap_and_scale(ep, table, new):
    rng = np.random.default_rng(11)
    cache = Cache(rng, new, [200, 30], E.I8, 2, 128, 64)
    check(ep, cache, 8, E.F16, 5, sd=4.0, softcap=5.0)
    check(ep, cache, 8, E.F16, 6, softcap=50.0, scale=0.3)
    check(ep, cache, 8, E.BF16, 7, scale=2.0 ** -10)


@pytest.mark.parametrize("new", [[1, 1], [150, 7]])
@pytest.mark.parametrize("sd", [0.0, 1e-30, 1e-6, 30.0, 1e4])
def test_sizes_of_queries(ep, table, sd, new):
    """From queries of zeros (even attention) to scores of thousands (one token takes all)."""
    rng = np.random.default_rng(12)
    cache = Cache(rng, new, [100, 30], E.I8, 1, 64, 16)
    check(ep, cache, 4, E.BF16, 8, sd=sd)


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("new", [[1, 1], [150, 3]])
def test_scales_of_pages(ep, table, new, code):
    """Pages whose scales differ by orders of magnitude, some zero: keys of zeros, values of zeros, both."""
    rng = np.random.default_rng(13)
    cache = Cache(rng, new, [300, 70], code, 2, 64, 16)
    live = ~np.isnan(cache.ks)
    cache.ks[live] *= 10.0 ** rng.uniform(-3, 0.5, live.sum()).astype(np.float32)
    cache.vs[live] *= 10.0 ** rng.uniform(-6, 3, live.sum()).astype(np.float32)
    for zero in (cache.ks, cache.vs):
        zero[live & (rng.random(live.shape) < 0.2)] = 0
    check(ep, cache, 4, E.BF16, 9)
    cache.vs[live] = 0
    check(ep, cache, 4, E.BF16, 10)


@pytest.mark.parametrize("new,heads", [([1, 1, 1], 4), ([90, 3, 40], 4), ([90, 3, 40], 132)])
def test_nan_stays_with_the_rows_that_see_it(ep, new, heads):
    """A page of scale NaN, keys or values: rows that see it are NaN, others (before it, outside their window, of other heads and sequences) are as without it."""
    rng = np.random.default_rng(14)
    for which in ("ks", "vs"):
        cache = Cache(rng, new, [100, 70, 30], E.I8, 2, 64, 16)
        q = floats(rng, (cache.rows, heads * 64), E.F16)
        want, slack = attention64(cache, as64(q, E.F16).reshape(-1, heads, 64), heads, window=40)
        bad = 6 if new[0] == 1 else 8                     # a page of the first sequence: all of its queries see page 6; some are before page 8, others are past it
        getattr(cache, which)[cache.table[0, bad], 0] = np.nan
        got, _ = attend(ep, cache, q, E.F16, heads, local_window_size=40)
        own = 100 + np.arange(new[0])
        sees = np.zeros(got.shape[:2], bool)
        sees[:new[0], :heads // 2] = ((own >= 16 * bad) & (own - 40 < 16 * bad + 15))[:, None]
        assert sees.any() and not sees.all()
        assert np.isnan(as64(got, E.F16)[sees]).all()
        near(got[~sees], want[~sees], slack[~sees], E.F16)


@pytest.mark.parametrize("new", [[1], [90]])
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_nothing_but_nan_pages(ep, table, which, new):
    """Every page of one head has a scale of NaN: its rows are NaN, the other head's are as without it. And a scale of 0 is no NaN."""
    rng = np.random.default_rng(24)
    cache = Cache(rng, new, [700], E.I8, 2, 64, 16)
    q = floats(rng, (cache.rows, 2 * 64), E.F16)
    want, slack = attention64(cache, as64(q, E.F16).reshape(-1, 2, 64), 2)
    getattr(cache, which)[:, 0] = np.nan
    got, _ = attend(ep, cache, q, E.F16, 2)
    assert np.isnan(as64(got[:, 0], E.F16)).all()
    near(got[:, 1], want[:, 1], slack[:, 1], E.F16)
    cache.ks[:, 0] = 0.02
    cache.vs[:, 0] = 0.0
    got, _ = attend(ep, cache, q, E.F16, 2)
    assert not as64(got[:, 0], E.F16).any()


@pytest.mark.parametrize("new", [[1, 1], [90, 3]])
def test_the_widest_windows(ep, new):
    """A window as long as anything can be, or longer, is none."""
    rng = np.random.default_rng(25)
    cache = Cache(rng, new, [130, 7], E.I8, 1, 64, 16)
    q = floats(rng, (cache.rows, 2 * 64), E.F16)
    plain, _ = attend(ep, cache, q, E.F16, 2)
    for window in (1 << 29, (1 << 30) - 1, 1 << 30, (1 << 31) - 1):
        got, _ = attend(ep, cache, q, E.F16, 2, local_window_size=window)
        assert np.array_equal(got, plain), window


def test_nan_and_infinite_queries(ep, table):
    rng = np.random.default_rng(15)
    for new in ([1, 1, 1, 1], [40, 9, 3, 1]):
        cache = Cache(rng, new, [100, 70, 30, 0], E.I8, 1, 64, 16)
        q = floats(rng, (cache.rows, 2 * 64), E.BF16)
        want, slack = attention64(cache, as64(q, E.BF16).reshape(-1, 2, 64), 2)
        q[0, 3] = 0x7FC0
        q[1, 64 + 5] = 0x7F80
        got, _ = attend(ep, cache, q, E.BF16, 2)
        assert np.isnan(as64(got[0, 0], E.BF16)).all() and np.isnan(as64(got[1, 1], E.BF16)).all()
        keep = np.ones(got.shape[:2], bool)
        keep[0, 0] = keep[1, 1] = False
        near(got[keep], want[keep], slack[keep], E.BF16)


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 40, 40]])
def test_pages_that_are_not_there(ep, table, new):
    """Entries outside the pool hold no tokens: the rest of the context is what a row sees; a row that sees none is zero. Past lengths beyond the table end with it."""
    rng = np.random.default_rng(16)
    cache = Cache(rng, new, [160, 160, 160], E.F8E4M3, 1, 64, 16)
    q = floats(rng, (cache.rows, 2 * 64), E.F16)
    views_of = lambda dev, entries, past: cache.views(dev)[:5] + [dev.view(np.asarray(past, np.int32), E.I32), dev.view(entries, E.I32)]  # noqa: E731
    entries = cache.table.copy()
    odd = entries[0, 1:15:2]
    odd[:] = [-1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31, -5, -1, -1][:len(odd)]
    entries[1] = -1
    dev = Device(ep)
    try:
        got, _ = attend(ep, cache, q, E.F16, 2, views=views_of(dev, entries, cache.past_lengths), dev=dev)
    finally:
        dev.free()
    # the definition over the tokens that are there
    q64 = as64(q, E.F16).reshape(-1, 2, 64)
    assert not got[cache.ends[1]:cache.ends[2]].any()
    for i in (0, 2):
        k, v = cache.tokens(i, 160 + new[i])
        there = np.ones(len(k), bool) if i == 2 else (np.arange(len(k)) // 16) % 2 == 0
        for r in range(new[i]):
            seen = there & (np.arange(len(k)) <= 160 + r)
            for h in range(2):
                z = k[seen, 0] @ q64[cache.ends[i] + r, h] / 8
                w = np.exp(z - z.max())
                w /= w.sum()
                assert np.abs(as64(got[cache.ends[i] + r, h], E.F16) - w @ v[seen, 0]).max() <= 2.0 ** -9 * (w @ np.abs(v[seen, 0])).max()
    # a past beyond the table: every query sees all that the table has, and so the NaN codes of slots without tokens; one below 0 is 0
    dev = Device(ep)
    try:
        got, _ = attend(ep, cache, q, E.F16, 2, views=views_of(dev, cache.table, [2 ** 31 - 1, 2 ** 30, -4]), dev=dev)
    finally:
        dev.free()
    assert np.isnan(as64(got[:cache.ends[2]], E.F16)).all() and np.isfinite(as64(got[cache.ends[2]:], E.F16)).all()


@pytest.mark.parametrize("sequences", [64, 65, 200])
def test_many_sequences(ep, sequences):
    rng = np.random.default_rng(sequences)
    cache = Cache(rng, rng.integers(0, 3, sequences), rng.integers(0, 40, sequences), E.I8, 1, 64, 16, width=5)
    check(ep, cache, 2, E.F16, 17)


@pytest.mark.parametrize("new,past", [([1], [5000]), ([1, 1, 1], [3000, 17, 700]), ([3, 1], [2049, 4095]), ([60], [2500]), ([130], [1900])])
@pytest.mark.parametrize("window", [0, 1500, 2500])
def test_pieces_of_long_contexts(ep, new, past, window):
    """Few rows over a long context: several workgroups share it, and their results are joined. (A window below 2048 tokens leaves nothing to share.)"""
    rng = np.random.default_rng(past[0])
    cache = Cache(rng, new, past, E.I8, 1, 64, 32)
    assert check(ep, cache, 4, E.F16, 18, window=window).endswith("pieces") == (window != 1500)


@pytest.mark.parametrize("new,past,heads,kv_heads,page,variant", [([3, 9], [5000, 2500], 30, 10, 64, "cache_attention_pieces"), ([1, 0, 30, 2], [2300, 9, 4100, 40], 12, 3, 16, "cache_attention_pieces"),
                                                                  ([300], [9000], 12, 3, 64, "cache_attention_rows_pieces"), ([290, 3, 1], [6500, 7000, 1], 30, 10, 32, "cache_attention_rows_pieces")])
def test_pieces_of_several_tiles_and_heads(ep, new, past, heads, kv_heads, page, variant):
    """Tiles, pieces and key heads in numbers that no power of two divides; some rows against the definition."""
    rng = np.random.default_rng(heads + past[0])
    cache = Cache(rng, new, past, E.I8, kv_heads, 64, page)
    q = floats(rng, (cache.rows, heads * 64), E.F16)
    got, used = attend(ep, cache, q, E.F16, heads)
    assert used == variant
    rows = set(rng.integers(0, cache.rows, 10).tolist()) | {int(e) - 1 for e in cache.ends[1:]}
    want, slack = attention64(cache, as64(q, E.F16).reshape(-1, heads, 64), heads, rows=rows)
    near(got[sorted(rows)], want[sorted(rows)], slack[sorted(rows)], E.F16)


def test_weights_far_below_the_largest(ep):
    """One token at the top and thousands far below it, whose weights together count: none of them is lost to f16."""
    rng = np.random.default_rng(19)
    past = 8191
    cache = Cache(rng, [1], [past], E.I8, 1, 64, 64)
    cache.k[:] = 0
    cache.k[cache.table[0, 3], 0, 5, 0] = 127
    cache.v[:] = np.abs(cache.v)
    cache.vs[:] = 0.01
    cache.ks[:] = 1.0
    for nats in (5.0, 9.0, 13.0, 17.0):
        q = np.zeros((1, 64), np.float16)
        q[0, 0] = nats * 8 / 127
        want, slack = attention64(cache, as64(q, E.F16).reshape(1, 1, 64), 1)
        got, _ = attend(ep, cache, q, E.F16, 1)
        near(got, want, slack, E.F16)


@pytest.mark.parametrize("new", [[1, 1], [150, 7]])
def test_shared_pages(ep, table, new):
    """Two sequences over the same prompt's pages."""
    rng = np.random.default_rng(20)
    cache = Cache(rng, new, [128, 128], E.I8, 1, 64, 64)
    cache.table[1, :2] = cache.table[0, :2]
    check(ep, cache, 4, E.F16, 21)


def test_a_cache_beyond_32_bits(ep):
    """Pages whose bytes begin beyond 4 GiB."""
    heads, head, page, pages = 8, 128, 128, 34000                   # 4.46 GB of keys, as much of values
    rng = np.random.default_rng(22)
    small = Cache(rng, [1], [300], E.I8, heads, head, page)
    each = heads * head * page
    bufs = [ep.allocate(pages * each) for _ in range(2)] + [ep.allocate(pages * heads * 4) for _ in range(2)]
    dev = Device(ep)
    try:
        table = np.array([[pages - 1, 5, pages - 2]], np.int32)
        for j, p in enumerate(table[0]):
            src = small.table[0, j]
            for buf, x in zip(bufs, (small.k, small.v)):
                ep.copy_from_host(buf, x[src], offset=int(p) * each)
            for buf, x in zip(bufs[2:], (small.ks, small.vs)):
                ep.copy_from_host(buf, x[src], offset=int(p) * heads * 4)
        shapes = [(pages, heads, page, head), (pages, heads, head, page), (pages, heads), (pages, heads)]
        views = [E.TensorView(b.ptr, dt, s) for b, dt, s in zip(bufs, (E.I8, E.I8, E.F32, E.F32), shapes)]
        views += [dev.view(small.ends, E.I32), dev.view(small.past_lengths, E.I32), dev.view(table, E.I32)]
        q = floats(rng, (1, 8 * head), E.F16)
        got, _ = attend(ep, small, q, E.F16, 8, views=views, dev=dev)
        want, slack = attention64(small, as64(q, E.F16).reshape(1, 8, head), 8)
        near(got, want, slack, E.F16)
    finally:
        dev.free()
        for b in bufs:
            ep.deallocate(b)
