"""The paged 8-bit cache on the host: codes, pages, and 64-bit references of the operators around it."""
from __future__ import annotations

import numpy as np

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import as64

TOP = {E.I8: 127.0, E.F8E4M3: 448.0}


def _e4m3_values():
    bits = np.arange(256)
    exponent, mantissa = (bits >> 3) & 15, bits & 7
    v = np.where(exponent == 0, mantissa / 8 * 2.0 ** -6, (1 + mantissa / 8) * 2.0 ** (exponent - 7.0))
    v[(bits & 127) == 127] = np.nan
    return np.where(bits & 128, -v, v)


E4M3 = _e4m3_values()


def decode(codes, code):
    return codes.astype(np.float64) if code == E.I8 else E4M3[codes]


def encode(x, code):
    """f32 quotients (or products) to codes, to the nearest, ties to even; within the type's range."""
    if code == E.I8:
        return np.rint(x).astype(np.int8)
    x = np.clip(np.asarray(x, np.float64), -448, 448)
    at = np.clip(np.searchsorted(E4M3[:127], np.abs(x)), 1, 126)
    low, high = E4M3[at - 1], E4M3[at]
    up = (np.abs(x) - low > high - np.abs(x)) | ((np.abs(x) - low == high - np.abs(x)) & (at % 2 == 0))
    bits = np.where(up, at, at - 1).astype(np.uint8)
    return bits | np.where(np.signbit(x), 128, 0).astype(np.uint8)


def same_values(got, want, code):
    """Codes that stand for the same numbers: -0 is 0."""
    return np.array_equal(decode(got, code), decode(want, code), equal_nan=True)


LEAST_SLOTS = [0]                   # that a sequence's table has, beyond what it needs: entries without a page


class Cache:
    """A cache with pages at random places of the pool, one more than needed; slots and pages without tokens hold what would show (NaN codes, NaN scales)."""

    def __init__(self, rng, new, past, code, kv_heads, head, page, *, width=None, fill=True):
        self.new, self.past, self.code, self.kv_heads, self.head, self.page = list(new), list(past), code, kv_heads, head, page
        need = [-(-(a + b) // page) for a, b in zip(new, past)]
        pages = sum(need) + 1
        self.table = np.full((len(new), max(width or max(max(need, default=1), 1), LEAST_SLOTS[0] // page)), -7, np.int32)
        order = rng.permutation(pages)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        np_type, bad = (np.int8, -128) if code == E.I8 else (np.uint8, 127)
        self.k, self.v = np.full((pages, kv_heads, page, head), bad, np_type), np.full((pages, kv_heads, head, page), bad, np_type)
        self.ks, self.vs = np.full((pages, kv_heads), np.nan, np.float32), np.full((pages, kv_heads), np.nan, np.float32)
        spread = 40.0 if code == E.I8 else 120.0
        for i, n in enumerate(need):
            # tokens that are there: all of them, or those of the past
            for t in range((past[i] + new[i]) if fill else past[i]):
                p, s = self.table[i, t // page], t % page
                self.k[p, :, s], self.v[p, :, :, s] = (encode(np.clip(rng.standard_normal((kv_heads, head)) * spread, -TOP[code], TOP[code]).astype(np.float32), code) for _ in range(2))
            for j in range(-(-((past[i] + new[i]) if fill else past[i]) // page)):
                self.ks[self.table[i, j]], self.vs[self.table[i, j]] = (rng.uniform(0.4, 1.6, kv_heads) / spread for _ in range(2))
        self.ends = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.past_lengths = np.asarray(past, np.int32)

    @property
    def rows(self):
        return int(self.ends[-1])

    def tokens(self, i, length):
        """Keys and values of a sequence's first tokens in 64 bits: [length, kv_heads, head]."""
        t = np.arange(length)
        p, s = self.table[i, t // self.page], t % self.page
        k = decode(self.k[p, :, s], self.code) * self.ks[p].astype(np.float64)[..., None]
        v = decode(self.v[p, :, :, s], self.code) * self.vs[p].astype(np.float64)[..., None]
        return k, v

    def views(self, dev):
        """k_cache, v_cache, k_scale, v_scale, cumulative_lengths, past_lengths, block_table."""
        return [dev.view(self.k, self.code), dev.view(self.v, self.code), dev.view(self.ks, E.F32), dev.view(self.vs, E.F32), dev.view(self.ends, E.I32),
                dev.view(self.past_lengths, E.I32), dev.view(self.table, E.I32)]

    def read(self, ep, views):
        ep.sync()
        return [ep.download(E.DeviceBuffer(v.data, 0), x.shape, x.dtype) for v, x in zip(views[:4], (self.k, self.v, self.ks, self.vs))]


def append32(cache, key, value):
    """What CacheAppend makes of a cache, in the arithmetic that it is defined in; keys and values f32 [T, kv_heads, head]. The cache is changed."""
    top = np.float32(TOP[cache.code])
    for i, n in enumerate(cache.new):
        t = 0
        while t < n:
            position = cache.past[i] + t
            p, slot = cache.table[i, position // cache.page], position % cache.page
            count = min(cache.page - slot, n - t)
            for h in range(cache.kv_heads):
                for x, codes, scales in ((key, cache.k[p, h], cache.ks), (value, cache.v[p, h].T, cache.vs)):
                    x = x[cache.ends[i] + t:cache.ends[i] + t + count, h]
                    new = np.float32(np.abs(x).max() / top)
                    old = scales[p, h] if slot else np.float32(0)
                    bad = not np.isfinite(x).all() or np.isnan(old)
                    scale = np.float32(np.nan) if bad else max(old, new)
                    if slot and (bad or scale != old):
                        ratio = np.float32(0) if bad or scale == 0 else np.float32(old / scale)
                        codes[:slot] = encode((decode(codes[:slot], cache.code).astype(np.float32) * ratio).astype(np.float32), cache.code) if ratio > 0 else 0
                    codes[slot:slot + count] = encode((x / scale).astype(np.float32), cache.code) if not bad and scale > 0 else 0
                    scales[p, h] = scale
            t += count


def attention64(cache, q, heads, *, scale=None, window=0, softcap=0.0, rows=None, of_heads=None):
    """[T, heads, head] in 64 bits (of some rows and heads, if they are given), zero where nothing is seen; and how far off the kernel may be beside its last rounding: per element, from the roundings that it makes."""
    d, group = cache.head, heads // cache.kv_heads
    scale = scale or 1 / np.sqrt(d)
    y, slack = np.zeros((cache.rows, heads, d)), np.zeros((cache.rows, heads, d))
    for i, n in enumerate(cache.new):
        if not n:
            continue
        k, v = cache.tokens(i, cache.past[i] + n)
        slot = np.arange(cache.past[i] + n)
        page, place = cache.table[i, slot // cache.page], slot % cache.page
        codes, top = decode(cache.v[page, :, :, place], cache.code), np.nanmax(cache.vs[page], 0)
        for r in range(n):
            own, row = cache.past[i] + r, cache.ends[i] + r
            if rows is not None and row not in rows:
                continue
            seen = (slot <= own) & ((slot > own - window) if window else True)
            for h in of_heads or range(heads):
                kk, vv, qq = k[seen, h // group], v[seen, h // group], q[row, h]
                z = scale * (kk @ qq)
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                w = np.exp(z - z.max())
                w /= w.sum()
                y[row, h] = w @ vv
                # scores: products of f16 operands (a query's bits reach 2^-22 of its row's largest) summed in f32, then a few f32 steps; weights: a rounding to 11 bits,
                # those of f32 and of the exponential; and half of f16's smallest step, 2^-25, of weights that are held times 2^11 or more (relative to the row's largest) and times
                # their page's scale over the largest such scale: 2^-36 of a value whose page had that scale
                off = scale * (np.abs(kk).sum(-1) * np.abs(qq).max() * 2.0 ** -22 + np.abs(kk) @ np.abs(qq) * (d + 8) * 2.0 ** -24).max() + 2.0 ** -20
                slack[row, h] = (w * (2.0 ** -11 + 2 * off)) @ np.abs(vv) + 2.0 ** -36 * top[h // group] * np.abs(codes[seen, h // group]).sum(0)
    return y, slack


def floats(rng, shape, dtype, sd=1.0):
    return synth.to_dtype((rng.standard_normal(shape) * sd).astype(np.float32), dtype)


def pages_step(table, lengths, parents, grow, page, pages):
    """next table, next lengths, moves, counts by the definition, one slot after the other."""
    slots, width = table.shape
    new_lengths = [int(np.clip(lengths[p], 0, width * page)) if 0 <= p < slots else 0 for p in parents]
    valid = lambda p: int(p) if 0 <= p < pages else -1  # noqa: E731
    next_table = np.full_like(table, -1)
    held, missing = set(), 0
    for i, n in enumerate(new_lengths):
        for j in range(n // page):
            p = valid(table[parents[i], j])
            next_table[i, j] = p
            if p < 0:
                missing += 1
            else:
                held.add(p)
    begun = [valid(table[parents[i], n // page]) if n % page else None for i, n in enumerate(new_lengths)]
    keeps = [b is not None and b >= 0 and b not in held and b not in begun[:i] for i, b in enumerate(begun)]
    held |= {b for b, keep in zip(begun, keeps) if keep}
    free = [p for p in range(pages) if p not in held]
    used, moves = 0, np.full((slots, 2), -1, np.int32)

    def fresh():
        nonlocal used, missing
        used += 1
        if used > len(free):
            missing += 1
            return -1
        return free[used - 1]

    for i, n in enumerate(new_lengths):
        if begun[i] is not None:
            if begun[i] < 0:
                missing += 1
            elif keeps[i]:
                next_table[i, n // page] = begun[i]
            else:
                next_table[i, n // page] = fresh()
                if next_table[i, n // page] >= 0:
                    moves[i] = begun[i], next_table[i, n // page]
        end = min(n + max(0, int(grow[i])), width * page) if 0 <= parents[i] < slots else 0
        for j in range(-(-n // page), -(-end // page)):
            next_table[i, j] = fresh()
    return next_table, np.asarray(new_lengths, np.int32), moves, np.asarray([len(held) + min(used, len(free)), missing], np.int32)


def pages_compact(table, lengths, page, pages):
    slots, width = table.shape
    lengths = np.clip(lengths, 0, width * page)
    used = [[(int(p) if 0 <= p < pages else -1) for p in table[i, :-(-int(n) // page)]] for i, n in enumerate(lengths)]
    live = sorted({p for row in used for p in row if p >= 0})
    n = len(live)
    sources, holes = [p for p in live if p >= n], [p for p in range(n) if p not in set(live)]
    to = dict(zip(sources, holes))
    next_table = np.full_like(table, -1)
    for i, row in enumerate(used):
        for j, p in enumerate(row):
            next_table[i, j] = to.get(p, p)
    moves = np.full((pages // 2, 2), -1, np.int32)
    for i, (a, b) in enumerate(zip(sources, holes)):
        moves[i] = a, b
    return next_table, lengths.astype(np.int32), moves, np.asarray([n, sum(p < 0 for row in used for p in row)], np.int32)
