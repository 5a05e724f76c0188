"""CacheAppend where a page's scale is a few of f32's smallest steps."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .cache_helpers import Cache, encode, same_values
from .test_cache_append_gpu import append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
@pytest.mark.parametrize("largest", [1, 63, 64, 100, 130, 190, 191, 300, 1000, 5000, 40000, 10 ** 6])
def test_scales_of_a_few_steps(ep, largest, code):
    """f32 inputs so small that their page's scale has few bits: quotients end at the largest code and keep their sign."""
    cache = Cache(np.random.default_rng(41), [20, 1], [0, 5], code, 1, 64, 16, fill=False)
    rng = np.random.default_rng(42)
    key, value = ((rng.integers(-largest, largest + 1, (cache.rows, 64)).astype(np.int32)) for _ in range(2))
    for x in (key, value):
        x[0, 3], x[1, 4], x[20, 5] = largest, -largest, -largest
    key, value = (np.where(x < 0, np.abs(x).view(np.uint32) | 0x80000000, x.view(np.uint32)).astype(np.uint32).view(np.float32) for x in (key, value))     # multiples of 2^-149
    cache.ks[cache.table[1, 0]], cache.vs[cache.table[1, 0]] = 0.0, 0.0
    cache.k[cache.table[1, 0], :, :5], cache.v[cache.table[1, 0], :, :, :5] = 0, 0
    got = append(ep, cache, key, value, E.F32)
    top = 127 if code == E.I8 else 448
    for i, n in enumerate(cache.new):
        for t in range(n):
            position = cache.past[i] + t
            p, slot = cache.table[i, position // 16], position % 16
            first = max(cache.past[i], position // 16 * 16) - cache.past[i] + int(cache.ends[i])
            last = min(int(cache.ends[i]) + n, int(cache.ends[i]) + (position // 16 + 1) * 16 - cache.past[i])
            for x, codes, scales in ((key, got[0][p, 0, slot], got[2]), (value, got[1][p, 0, :, slot], got[3])):
                scale = np.float32(np.abs(x[first:last]).max() / np.float32(top))
                assert scales[p, 0] == scale
                quotient = np.clip(x[cache.ends[i] + t].astype(np.float64) / scale, -top, top) if scale > 0 else np.zeros(64)
                assert same_values(codes, encode(quotient.astype(np.float32), code), code)
