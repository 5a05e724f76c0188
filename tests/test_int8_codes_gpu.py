"""Codes of rows whose scale is near the end of f32's normal numbers: the quotients that lie half way between two codes, and next to it."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .node_helpers import Device, codes32

pytestmark = pytest.mark.gpu


def rows_at_borders(exponent, k):
    """A row of scale s = 2^exponent m: its largest value 127 s, the others the f32 values nearest to (j + 1/2) s, and one step to either side."""
    rng = np.random.default_rng(abs(exponent))
    rows = []
    while len(rows) < 40:
        top = (np.float32(127) * np.ldexp(np.float32(1) + rng.integers(0, 1 << 23) / np.float32(1 << 23), exponent)).astype(np.float32)
        scale = np.float32(top / np.float32(127))
        j = rng.integers(0, 8, k)
        middle = ((j + 0.5) * np.float64(scale)).astype(np.float32)
        row = (middle.view(np.int32) + rng.integers(-1, 2, k).astype(np.int32)).view(np.float32) * rng.choice([-1, 1], k).astype(np.float32)
        row[rng.integers(k)] = top
        rows.append(row)
    return np.stack(rows)


@pytest.mark.parametrize("exponent", [-126, -125, -124, -122, -118, -110, -101, -60, 0, 100])
def test_codes_are_the_nearest(ep, exponent):
    """B is the identity and b_scale a power of two, so that each result is a code times the row's scale, exactly up to the scale's rounding into y."""
    k = 128
    a = rows_at_borders(exponent, k)
    want, scale = codes32(a)
    up = np.float32(2.0 ** min(-exponent, 126))
    dev = Device(ep)
    kernel = ep.get_kernel({"K": k, "N": k}, op_type="MatMulInt8")
    try:
        y, read = dev.output(a.shape, E.F32)
        kernel.execute([dev.view(a, E.F32), dev.view(np.eye(k, dtype=np.int8), E.I8), dev.view(np.full(k, up), E.F32)], [y])
        got = np.rint(read().astype(np.float64) / (scale.astype(np.float64) * float(up))[:, None]).astype(np.int64)
    finally:
        dev.free()
        kernel.release()
    assert np.array_equal(got, want), (exponent, (got != want).sum())
