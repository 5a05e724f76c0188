"""RotaryEmbedding's scalings at the ends of what their attributes may be."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import as64
from .test_rotary_gpu import frequencies, near, run, turned

pytestmark = pytest.mark.gpu


def check(ep, f, magnitude, attrs):
    """Rows of two heads of 64 whose pairs turn by f a position."""
    x = synth.to_dtype(np.random.default_rng(51).standard_normal((9, 128)).astype(np.float32), E.F32)
    positions = np.array([0, 1, 2, 3, 17, 100, 4095, 4096, 70000])
    angle = positions[:, None] * f
    cos, sin = magnitude * np.cos(angle), magnitude * np.sin(angle)
    got, _ = run(ep, x, E.F32, positions, {"head_size": 64, "scaling": 3, **attrs})
    x64 = as64(x, E.F32).reshape(9, 2, 64)
    want = turned(x64, cos, sin, 64, 0).reshape(9, -1)
    # an element is a c - b s or b c + a s: of its terms, cosines and sines are off by 2^-24 of theirs, products and their sum by as much again
    pair = np.abs(x64) + np.abs(np.roll(x64, 32, -1))
    size = (pair * np.tile(np.abs(cos) + np.abs(sin), 2)[:, None]).reshape(9, -1)
    near(got, want, size, E.F32)


@pytest.mark.parametrize("factor", [1e-5, 0.5, 1.0, 1.5, 40.0])
def test_magnitude_of_yarn(ep, factor):
    """0.1 ln(factor) + 1 for contexts that are stretched; nothing is amplified or turned round where they are not."""
    f, _ = frequencies(64, scaling=3, factor=factor, original=4096)
    check(ep, f, 0.1 * np.log(factor) + 1 if factor > 1 else 1.0, {"factor": factor, "original_max_position": 4096})


@pytest.mark.parametrize("original", [1, 3, 4])
def test_yarn_where_no_pair_turns_once(ep, original):
    """Within so short a context every pair makes fewer than beta_slow turns: all of them are slowed, the first one too."""
    check(ep, 10000.0 ** (-np.arange(0, 64, 2) / 64) / 8, 0.1 * np.log(8) + 1, {"factor": 8.0, "original_max_position": original})
