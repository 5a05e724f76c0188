"""RotaryEmbedding against its definition in 64 bits: layouts, positions, scalings, caches."""
import math

import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, as64

pytestmark = pytest.mark.gpu


def frequencies(part, theta=10000.0, scaling=0, factor=1.0, original=8192, low=1.0, high=4.0, fast=32.0, slow=1.0):
    f = theta ** (-np.arange(0, part, 2) / part)
    if scaling == 1:
        return f / factor, 1.0
    if scaling == 2:
        wavelength = 2 * np.pi / f
        smooth = (original / wavelength - low) / (high - low)
        blend = (1 - smooth) * f / factor + smooth * f
        return np.where(wavelength > original / low, f / factor, np.where(wavelength < original / high, f, blend)), 1.0
    if scaling == 3:
        pair = lambda turns: part * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), part - 1)
        slower = np.clip((np.arange(part // 2) - first) / max(last - first, 0.001), 0, 1)
        return f / factor * slower + f * (1 - slower), 0.1 * math.log(factor) + 1
    return f, 1.0


def turned(x, cos, sin, part, interleaved):
    """x [rows, heads, d]; cos, sin [rows, part / 2]"""
    y = x.copy()
    a, b = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    y[..., a] = x[..., a] * cos[:, None] - x[..., b] * sin[:, None]
    y[..., b] = x[..., b] * cos[:, None] + x[..., a] * sin[:, None]
    return y


def near(got, want, size, dtype):
    """One rounding to the type, and what f32 does to two products of cosines rounded to f32: 2^-24 each for the cosine, the product and the sum."""
    assert (np.abs(as64(got, dtype) - want) <= EPS[dtype] / 2 * np.abs(want) + 4 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == E.F16 else 0)).all()


def run(ep, x, dtype, positions, attrs, *, caches=(), cache_dtype=E.F32, shape=None, offset=0, position_dtype=E.I64, in_place=False):
    dev = Device(ep)
    try:
        kernel = ep.get_kernel(attrs, op_type="RotaryEmbedding")
        shape = shape or x.shape
        y, read = dev.output(shape, dtype, offset)
        source = dev.view(x, dtype, shape, offset)
        if in_place:
            ep.sync()
            ep.copy_from_host(y.data + offset * E._ITEM[dtype], x)
            source = y
        inputs = [source, dev.view(np.asarray(positions, E._NP[position_dtype]), position_dtype)] + [dev.view(synth.to_dtype(c, cache_dtype), cache_dtype) for c in caches]
        kernel.execute(inputs, [y])
        ep.sync()
        got = read().copy()
        variant = kernel.last_variant()
        kernel.release()
        return got, variant
    finally:
        dev.free()


@pytest.mark.parametrize("dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("rows,heads,d,part,behind", [(1, 36, 128, 0, 512), (3, 5, 80, 32, 0), (7, 2, 64, 26, 3), (300, 3, 30, 10, 0), (2, 1, 256, 256, 8), (1, 1, 2, 2, 1), (517, 9, 64, 0, 64), (1, 2, 600, 512, 0)])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_layouts(ep, rows, heads, d, part, behind, interleaved, dtype):
    rng = np.random.default_rng(rows * 7 + d)
    x = synth.to_dtype(rng.standard_normal((rows, heads * d + behind)).astype(np.float32), dtype)
    positions = rng.integers(0, 5000, rows)
    attrs = {"head_size": d, "num_heads": heads, "rotary_embedding_dim": part, "interleaved": interleaved}
    f, _ = frequencies(part or d)
    angle = positions[:, None] * f
    x64 = as64(x, dtype)
    cos, sin = np.cos(angle), np.sin(angle)
    want = x64.copy()
    want[:, :heads * d] = turned(x64[:, :heads * d].reshape(rows, heads, d), cos, sin, part or d, interleaved).reshape(rows, -1)
    size = x64.copy()
    size[:, :heads * d] = turned(np.abs(x64[:, :heads * d]).reshape(rows, heads, d), np.abs(cos) + np.abs(sin), -np.abs(cos) - np.abs(sin), part or d, interleaved).reshape(rows, -1)
    size = np.abs(size) + np.abs(x64)
    for in_place in (False, True):
        got, variant = run(ep, x, dtype, positions, attrs, offset=1, in_place=in_place)
        assert variant == "rotary"
        near(got, want, size, dtype)
        # what does not turn passes through bit for bit
        assert np.array_equal(got[:, heads * d:], x[:, heads * d:])


@pytest.mark.parametrize("scaling", [dict(), dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0), dict(scaling=2, factor=32.0, original=4096), dict(scaling=3, factor=16.0, original=4096),
                                     dict(scaling=3, factor=40.0, original=4096, theta=1e6)])
@pytest.mark.parametrize("start", [0, 131071, 2 ** 31 + 11, -5])
def test_far_positions_and_scalings(ep, start, scaling):
    """f32 rows, where a wrong angle shows: the reference takes the angle in integers of a turn's 2^-60, without floating point's loss at far positions."""
    from fractions import Fraction
    rng = np.random.default_rng(abs(start) % 1000)
    rows, heads, d = 5, 2, 64
    x = rng.standard_normal((rows, heads * d)).astype(np.float32)
    positions = start + np.arange(rows)
    f, magnitude = frequencies(d, **scaling)
    whole = 2 ** 200
    two_pi = Fraction(6283185307179586476925286766559, 10 ** 30)
    angle = np.empty((rows, d // 2))
    for r, p in enumerate(positions):
        for i, v in enumerate(f):
            turns = Fraction(int(p)) * Fraction(float(v)) / two_pi
            angle[r, i] = float((turns - round(turns)) * two_pi)
    assert whole > 0
    cos, sin = magnitude * np.cos(angle), magnitude * np.sin(angle)
    names = {"original": "original_max_position", "theta": "rope_theta"}
    got, _ = run(ep, x, E.F32, positions, {"head_size": d, **{names.get(k, k): v for k, v in scaling.items()}})
    x64 = x.reshape(rows, heads, d).astype(np.float64)
    want = turned(x64, cos, sin, d, False)
    size = np.abs(x64) + np.abs(np.roll(x64, d // 2, -1))
    # the frequency itself has 53 bits: position * f is off by up to |angle before the turns come off| * 2^-51
    frequency_slack = (np.abs(positions)[:, None] * f * 2.0 ** -51)
    slack = np.concatenate([frequency_slack, frequency_slack], -1)[:, None]
    assert (np.abs(got.reshape(rows, heads, d) - want) <= 2.0 ** -24 * np.abs(want) + magnitude * (4 * 2.0 ** -24 + slack) * size).all()


@pytest.mark.parametrize("cache_dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_caches(ep, cache_dtype, interleaved):
    """Cosines and sines as inputs; a position that they do not have gives NaN where the row turns, and nowhere else."""
    rng = np.random.default_rng(3)
    heads, d, part, most = 3, 48, 32, 40
    x = rng.standard_normal((6, heads * d)).astype(np.float32)
    angle = np.arange(most)[:, None] * frequencies(part)[0]
    caches = [np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)]
    positions = np.array([0, 39, 40, -1, 2 ** 40, 7])
    attrs = {"head_size": d, "rotary_embedding_dim": part, "interleaved": interleaved}
    got, variant = run(ep, x, E.F32, positions, attrs, caches=caches, cache_dtype=cache_dtype)
    assert variant == "rotary_cached"
    there = (positions >= 0) & (positions < most)
    cos, sin = (as64(synth.to_dtype(c, cache_dtype), cache_dtype)[np.where(there, positions, 0)] for c in caches)
    x64 = x.reshape(6, heads, d).astype(np.float64)
    want = turned(x64, cos, sin, part, interleaved)
    got = got.reshape(6, heads, d)
    assert np.isnan(got[~there][..., :part]).all() and np.array_equal(got[..., part:], x.reshape(6, heads, d)[..., part:])
    assert np.allclose(got[there], want[there], rtol=0, atol=4 * 2.0 ** -24 * 2 * np.abs(x).max())


@pytest.mark.parametrize("position_dtype", [E.I64, E.I32])
def test_batches(ep, position_dtype):
    """Rank 3 with a position for each row or one for all sequences; rank 4 with the heads in front of the tokens."""
    rng = np.random.default_rng(4)
    n, s, heads, d = 3, 5, 4, 32
    x = rng.standard_normal((n, s, heads, d)).astype(np.float32)
    positions = rng.integers(0, 900, (n, s))
    f, _ = frequencies(d)

    def want(p):
        angle = p.reshape(-1, 1) * f
        return turned(x.reshape(n * s, heads, d).astype(np.float64), np.cos(angle), np.sin(angle), d, False).reshape(x.shape)

    close = lambda got, w: np.allclose(got, w, rtol=0, atol=4 * 2.0 ** -24 * 2 * np.abs(x).max())  # noqa: E731
    got, _ = run(ep, x.reshape(n, s, heads * d), E.F32, positions, {"head_size": d}, position_dtype=position_dtype)
    assert close(got.reshape(x.shape), want(positions))
    got, _ = run(ep, x.reshape(n, s, heads * d), E.F32, [17], {"head_size": d}, position_dtype=position_dtype)
    assert close(got.reshape(x.shape), want(np.tile(17 + np.arange(s), (n, 1))))
    for p, w in ((positions, want(positions)), ([17], want(np.tile(17 + np.arange(s), (n, 1))))):
        for in_place in (False, True):
            got, _ = run(ep, np.ascontiguousarray(x.transpose(0, 2, 1, 3)), E.F32, p, {"head_size": d}, position_dtype=position_dtype, in_place=in_place)
            assert close(got.transpose(0, 2, 1, 3), w)


def test_no_rows(ep):
    kernel = ep.get_kernel({"head_size": 8}, op_type="RotaryEmbedding")
    kernel.execute([E.TensorView(None, E.F16, (0, 16)), E.TensorView(None, E.I64, (0,))], [E.TensorView(None, E.F16, (0, 16))])
    kernel.release()
