"""MatMulInt8 against integer sums in 64 bits: heights on either side of each kernel, widths and depths that divide nothing, every type, extreme codes."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, as64, codes32

pytestmark = pytest.mark.gpu


def run(ep, m, n, k, dtype, *, y_dtype=None, bias=None, codes=False, scale_dtype=E.F32, seed=0, a=None, b=None, offset=0, workspace=False, shape=None):
    rng = np.random.default_rng(seed + m * 7 + n * 3 + k)
    y_dtype = y_dtype or (dtype if not codes else E.F16)
    b = rng.integers(-128, 128, (n, k)).astype(np.int8) if b is None else b
    sb = synth.to_dtype((rng.uniform(0.5, 1.5, n) / (73 * np.sqrt(k))).astype(np.float32), scale_dtype)
    if codes:
        q = rng.integers(-127, 128, (m, k)).astype(np.int8) if a is None else a
        sa = rng.uniform(0.01, 0.03, m).astype(np.float32)
        a_stored, a_dtype = q, E.I8
    else:
        a = synth.to_dtype((rng.standard_normal((m, k)) * np.where(rng.random(k) < 0.02, 8.0, 1.0)).astype(np.float32), dtype) if a is None else a
        q, sa = codes32(synth.to_f32(a, dtype))
        a_stored, a_dtype = a, dtype
    bias_np = None
    if bias is not None:
        bias_np = synth.to_dtype(rng.standard_normal(n if bias == "column" else (m, n)).astype(np.float32), y_dtype)
    product = (q.astype(np.float64) @ b.astype(np.float64).T) * sa.astype(np.float64)[:, None] * as64(sb, scale_dtype)
    want = product + (as64(bias_np, y_dtype) if bias_np is not None else 0)
    dev = Device(ep)
    kernel = ep.get_kernel({"K": k, "N": n}, op_type="MatMulInt8")
    lead = shape or (m,)
    try:
        inputs = [dev.view(a_stored, a_dtype, (*lead, k), offset), dev.view(b, E.I8, None, offset if k % 16 else 0), dev.view(sb, scale_dtype, None, offset)]
        if codes or bias:
            inputs.append(dev.view(sa, E.F32, lead, offset) if codes else E.TensorView.absent())
        if bias:
            inputs.append(dev.view(bias_np, y_dtype, (n,) if bias == "column" else (*lead, n), offset))
        y, read = dev.output((*lead, n), y_dtype, offset)
        ws = None
        if workspace:
            need, align = kernel.workspace_requirement([(v.shape if v.data else None, v.dtype) for v in inputs])
            ws = ep.allocate(max(need, 1), align)
            dev.bufs.append(ws)
        kernel.execute(inputs, [y], workspace=ws)
        got = as64(read().reshape(m, n), y_dtype)
        variant = kernel.last_variant()
    finally:
        dev.free()
        kernel.release()
    # the sum's way into f32, two products and the bias: four roundings of 2^-24, then the one to the result's type
    bound = EPS[y_dtype] / 2 * np.abs(want) * (1 + 2 ** -10) + 4 * 2.0 ** -24 * (np.abs(product) + np.abs(want)) + (2.0 ** -25 if y_dtype == E.F16 else 0)
    err = np.abs(got - want)
    assert (err <= bound).all(), (variant, (err / np.maximum(bound, 1e-300)).max(), np.argwhere(err > bound)[:4])
    return variant


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 300])
def test_rows(ep, m):
    run(ep, m, 272, 512, E.BF16)
    run(ep, m, 100, 384, E.F16, bias="column")


@pytest.mark.parametrize("k", [1, 15, 16, 17, 64, 100, 112, 127, 128, 129, 144, 1000, 4099, 18944])
@pytest.mark.parametrize("m", [1, 7, 40, 130])
def test_depths(ep, m, k):
    run(ep, m, 80, k, E.F16)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 33, 127, 128, 130, 255, 256, 257, 1000, 2311])
@pytest.mark.parametrize("m", [1, 24, 140, 520])
def test_widths(ep, m, n):
    run(ep, m, n, 256, E.BF16, bias="column")


@pytest.mark.parametrize("dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("y_dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("m", [1, 3, 20, 150])
def test_types(ep, m, dtype, y_dtype):
    run(ep, m, 136, 320, dtype, y_dtype=y_dtype, bias="row", scale_dtype=dtype)


@pytest.mark.parametrize("m,k", [(1, 512), (3, 500), (18, 384), (18, 400), (150, 256), (150, 77)])
def test_given_codes(ep, m, k):
    run(ep, m, 200, k, E.F16, codes=True)
    run(ep, m, 200, k, E.F16, codes=True, bias="row", y_dtype=E.F32)


@pytest.mark.parametrize("m", [1, 2, 20, 150])
@pytest.mark.parametrize("k", [100, 256, 331])
def test_elements_anywhere(ep, m, k):
    run(ep, m, 50, k, E.F16, offset=3, bias="column")
    run(ep, m, 50, k, E.F16, offset=1, codes=True)


@pytest.mark.parametrize("m", [1, 40, 140])
def test_the_largest_sums(ep, m):
    """Codes of 127 and -128 throughout: the sums reach 127 * 128 * K, close to the end of an int32 at K = 131071."""
    k, n = 131071, 17
    a = np.full((m, k), 127, np.int8)
    a[:, 1::2] = -127
    b = np.full((n, k), -128, np.int8)
    b[:, 1::2] = 127
    b[3] = -b[3].clip(-127, 127)
    run(ep, m, n, k, E.F16, codes=True, y_dtype=E.F32, a=a, b=b)


@pytest.mark.parametrize("m,n,k", [(500, 512, 18944), (300, 384, 4096), (1000, 3584, 1024), (600, 2000, 896)])
def test_tall(ep, m, n, k):
    run(ep, m, n, k, E.BF16, bias="column", workspace=True)


@pytest.mark.parametrize("k", [64, 65, 128, 192, 208, 256, 320, 1040])
def test_tiles_of_256(ep, k):
    """Enough tiles for the largest ones, their last rows and columns partial, from one step of K to many."""
    assert run(ep, 2050, 6200, k, E.F16, bias="column") == "int8_tile_256"


@pytest.mark.parametrize("y_dtype,bias,n", [(E.F32, "row", 6200), (E.BF16, "row", 6200), (E.BF16, "column", 6201), (E.F32, None, 6203)])
def test_results_of_tiles_of_256(ep, y_dtype, bias, n):
    assert run(ep, 2050, n, 128, E.BF16, y_dtype=y_dtype, bias=bias) == "int8_tile_256"


@pytest.mark.parametrize("m", [1, 5, 20, 150])
def test_callers_workspace(ep, m):
    for k in (384, 333):
        run(ep, m, 90, k, E.BF16, workspace=True)


def test_leading_dimensions(ep):
    run(ep, 12, 64, 128, E.F16, shape=(3, 2, 2), bias="row")


def test_ties_and_zero_rows(ep):
    """Quotients that lie half way between two codes go to the even one; a row of zeros gives the bias."""
    k = 256
    a = np.zeros((4, k), np.float32)
    a[0] = np.arange(k) * 0.5 - 63.5          # the largest is 64: scale 64 / 127
    a[1, 0] = 127.0                           # scale 1: the quotients are the values
    a[1, 1:] = np.resize([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5], k - 1)
    a[3, 5] = 1e-42                           # a scale below the normal numbers
    for m in (4, 70):
        run(ep, m, 48, k, E.F32, a=np.resize(a, (m, k)), bias="column")


@pytest.mark.parametrize("m", [2, 30, 140])
def test_rows_that_are_not_finite_leave_the_others_alone(ep, m):
    rng = np.random.default_rng(3)
    n, k = 40, 200
    a = rng.standard_normal((m, k)).astype(np.float32)
    b = rng.integers(-127, 128, (n, k)).astype(np.int8)
    results = []
    for dirty in (False, True):
        x = a.copy()
        if dirty:
            x[m - 1, 3] = np.inf if m == 30 else np.nan
        dev = Device(ep)
        kernel = ep.get_kernel({"K": k, "N": n}, op_type="MatMulInt8")
        y, read = dev.output((m, n), E.F32)
        kernel.execute([dev.view(x, E.F32), dev.view(b, E.I8), dev.view(np.ones(n, np.float32), E.F32)], [y])
        results.append(read())
        dev.free()
        kernel.release()
    assert np.array_equal(results[0][:-1], results[1][:-1]) and np.isnan(results[1][-1]).all()


@pytest.mark.parametrize("m,k", [(1, 384), (40, 333), (500, 4096)])
def test_graph_replays(ep, m, k):
    rng = np.random.default_rng(m)
    n = 256
    dev = Device(ep)
    kernel = ep.get_kernel({"K": k, "N": n}, op_type="MatMulInt8")
    data = [rng.standard_normal((m, k)).astype(np.float16) for _ in range(3)]
    try:
        a = dev.view(data[0], E.F16)
        rest = [dev.view(rng.integers(-127, 128, (n, k)).astype(np.int8), E.I8), dev.view(np.full(n, 0.001, np.float32), E.F32)]
        y, read = dev.output((m, n), E.F16)
        want = []
        for d in data:
            ep.copy_from_host(dev.bufs[0], d)
            kernel.execute([a] + rest, [y])
            want.append(read().copy())
        ep.capture_begin()
        kernel.execute([a] + rest, [y])
        graph = ep.capture_end()
        for d, w in zip(data, want):
            ep.copy_from_host(dev.bufs[0], d)
            graph.replay()
            ep.sync()
            assert np.array_equal(read(), w)
            kernel.execute([a] + rest, [y])
            assert np.array_equal(read(), w)
        graph.release()
    finally:
        dev.free()
        kernel.release()


def test_more_rows_than_one_launch_quantizes(ep):
    run(ep, 2 ** 21 + 3, 1, 16, E.F16)
