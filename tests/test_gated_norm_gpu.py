"""GatedResidualNorm against its definition in 64 bits: widths that divide nothing, every type, every part present and absent, in place, and as codes."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, as64, gated_norm64

pytestmark = pytest.mark.gpu

# A row's sums are taken over at most 32 elements a lane, 6 steps over a wave and 16 waves: 54 roundings of 2^-24 in a sum of squares, half of that in its root,
# and fewer than ten more on the way to an output: under 2^-18 of the terms' magnitudes. Centring adds the mean's own error, 54 roundings of the largest element.
F32_ERROR = 2.0 ** -18


def run(ep, rows, h, dtype, *, layer=False, post=True, gates=1, pre=True, betas=False, block=True, outputs="zn", epsilon=1e-6, residual_scale=1.0, block_scale=1.0, weight_dtype=None,
        offset=0, in_place=False, seed=0, scale=1.0, shape=None):
    rng = np.random.default_rng(seed + rows * 131 + h)
    wd = weight_dtype or dtype
    make = lambda n, dt, mean=0.0, sd=1.0: synth.to_dtype((rng.standard_normal(n) * sd + mean).astype(np.float32), dt)  # noqa: E731
    residual, y = make((rows, h), dtype, 0.2, 3.0 * scale), make((rows, h), dtype, 0.1, scale) if block else None
    post_gamma, gate = make(h, wd, 1.0, 0.2) if post else None, make((gates, h), wd, 0.0, 0.5) if gates else None
    pre_gamma, pre_beta = make(h, wd, 1.0, 0.2) if pre else None, make(h, wd, 0.0, 0.3) if betas else None
    post_beta = make(h, wd, 0.0, 0.3) if betas and post else None
    of = lambda x, dt: None if x is None else as64(x, dt)  # noqa: E731
    z64, n64, size = gated_norm64(as64(residual, dtype), of(y, dtype), of(post_gamma, wd), of(gate, wd), of(pre_gamma, wd), of(pre_beta, wd), of(post_beta, wd), epsilon=epsilon,
                                  residual_scale=residual_scale, block_scale=block_scale, layer=layer)
    dev = Device(ep)
    kernel = ep.get_kernel({"epsilon": epsilon, "residual_scale": residual_scale, "block_scale": block_scale, "layer_norm": int(layer)}, op_type="GatedResidualNorm")
    shape = shape or (rows, h)
    gate_shape = None if gate is None else (h,) if gates == 1 else (gates, h)
    try:
        res_view, blk_view = dev.view(residual, dtype, shape, offset), dev.view(y, dtype, shape, offset)
        inputs = [res_view, blk_view, dev.view(post_gamma, wd, None, offset), dev.view(gate, wd, gate_shape, offset), dev.view(pre_gamma, wd, None, offset), dev.view(pre_beta, wd, None, offset),
                  dev.view(post_beta, wd, None, offset)]
        z_view, z_read = dev.output(shape, dtype, offset)
        n_view, n_read = dev.output(shape, E.I8 if "c" in outputs else dtype, offset)
        s_view, s_read = dev.output((rows,), E.F32)
        if in_place:
            z_view, n_view = res_view, blk_view
            z_read = lambda: ep.download(dev.bufs[0], (offset + rows * h,), E._NP[dtype])[offset:].reshape(shape)  # noqa: E731
            n_read = lambda: ep.download(dev.bufs[1], (offset + rows * h,), E._NP[dtype])[offset:].reshape(shape)  # noqa: E731
        out = [z_view if "z" in outputs else E.TensorView.absent(), n_view if "n" in outputs or "c" in outputs else E.TensorView.absent()]
        if "c" in outputs:
            out.append(s_view)
        kernel.execute(inputs, out)
        got = {"z": z_read().reshape(rows, h) if "z" in outputs else None, "n": n_read().reshape(rows, h) if "n" in outputs or "c" in outputs else None, "s": s_read() if "c" in outputs else None}
    finally:
        dev.free()
        kernel.release()
    half = EPS[dtype] / 2
    if got["z"] is not None:
        err = np.abs(as64(got["z"], dtype) - z64)
        bound = half * np.abs(z64) * (1 + 2 ** -10) + F32_ERROR * size + (2.0 ** -25 if dtype == E.F16 else 0)        # (an f16 below 2^-14 is rounded to a step of 2^-24)
        assert (err <= bound).all(), (err / bound).max()
    spread = 1 / np.sqrt(((z64 - (z64.mean(-1, keepdims=True) if layer else 0)) ** 2).mean(-1, keepdims=True) + epsilon)
    weight = np.abs(of(pre_gamma, wd)) if pre_gamma is not None else 1.0
    n_size = spread * weight * (size + (np.abs(size).max(-1, keepdims=True) if layer else 0)) + np.abs(n64)
    if "n" in outputs:
        err = np.abs(as64(got["n"], dtype) - n64)
        bound = half * np.abs(n64) * (1 + 2 ** -10) + 2 * F32_ERROR * n_size + (2.0 ** -25 if dtype == E.F16 else 0)
        assert (err <= bound).all(), (err / bound).max()
    if "c" in outputs:
        top = np.abs(n64).max(-1)
        assert (np.abs(got["s"] - top / 127) <= 2 * F32_ERROR * n_size.max(-1) / 127 + top * 2.0 ** -23).all()
        off = np.abs(got["n"].astype(np.float64) * got["s"][:, None].astype(np.float64) - n64)
        assert (off <= 0.5 * got["s"][:, None] * (1 + 2 ** -14) + 2 * F32_ERROR * n_size).all()
        assert (np.abs(got["n"].astype(int)).max(-1) == 127)[top > 0].all()
    return got


@pytest.mark.parametrize("dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("h", [1, 7, 8, 9, 64, 511, 512, 513, 896, 2881, 4096, 8192, 8193, 18944, 32768])
def test_widths(ep, h, dtype):
    run(ep, 3, h, dtype, outputs="zn")


@pytest.mark.parametrize("rows,gates", [(1, 1), (2, 2), (5, 1), (12, 3), (333, 3), (70, 70)])
@pytest.mark.parametrize("layer", [False, True])
def test_rows_and_gates(ep, rows, gates, layer):
    for h, dtype in ((200, E.F16), (1031, E.BF16)):
        run(ep, rows, h, dtype, gates=gates, layer=layer, betas=layer, residual_scale=0.7071, block_scale=1.5)


@pytest.mark.parametrize("parts", [dict(post=False), dict(gates=0), dict(pre=False), dict(post=False, gates=0, pre=False), dict(block=False, post=False, gates=0), dict(betas=True),
                                   dict(outputs="z"), dict(outputs="n"), dict(weight_dtype=E.F32, betas=True, layer=True)])
@pytest.mark.parametrize("h", [72, 3585])
def test_parts(ep, parts, h):
    run(ep, 9, h, E.BF16, **parts)


@pytest.mark.parametrize("dtype", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("h", [5, 128, 1000, 3584, 9001, 20000])
def test_codes(ep, h, dtype):
    run(ep, 6, h, dtype, outputs="zc")
    run(ep, 6, h, dtype, outputs="c", layer=True, betas=True)


@pytest.mark.parametrize("offset", [1, 3, 5])
def test_elements_anywhere(ep, offset):
    run(ep, 7, 264, E.F16, offset=offset)
    run(ep, 7, 4096, E.F32, offset=offset, outputs="zc")


@pytest.mark.parametrize("h", [40, 2881])
def test_in_place(ep, h):
    """The new stream over the old one, the normalized rows over the block's: the same bits as beside them."""
    beside, over = run(ep, 17, h, E.BF16), run(ep, 17, h, E.BF16, in_place=True)
    assert np.array_equal(beside["z"], over["z"]) and np.array_equal(beside["n"], over["n"])


def test_leading_dimensions(ep):
    run(ep, 12, 320, E.F16, gates=3, shape=(3, 2, 2, 320))


def test_small_and_large_values(ep):
    """Rows whose squares would leave f16, and rows far below epsilon."""
    run(ep, 3, 512, E.F16, scale=3000.0, epsilon=1e-5)
    run(ep, 3, 512, E.BF16, scale=1e-6, epsilon=1e-5)
    run(ep, 3, 512, E.F32, scale=1e12)


def _plain(ep, residual, dtype, codes=False):
    dev = Device(ep)
    kernel = ep.get_kernel({"epsilon": 0.0}, op_type="GatedResidualNorm")
    try:
        n_view, n_read = dev.output(residual.shape, E.I8 if codes else dtype)
        s_view, s_read = dev.output((residual.shape[0],), E.F32)
        kernel.execute([dev.view(residual, dtype)], [E.TensorView.absent(), n_view] + ([s_view] if codes else []))
        return n_read(), s_read() if codes else None
    finally:
        dev.free()
        kernel.release()


def test_rows_that_are_not_finite_leave_the_others_alone(ep):
    rng = np.random.default_rng(5)
    clean = rng.standard_normal((6, 300)).astype(np.float32)
    dirty = clean.copy()
    dirty[1, 7], dirty[4, 299] = np.nan, np.inf
    want, got = _plain(ep, clean, E.F32)[0], _plain(ep, dirty, E.F32)[0]
    fine = [0, 2, 3, 5]
    assert np.array_equal(want[fine], got[fine]) and np.isnan(got[1]).all()
    assert np.isnan(got[4, 299]) and (got[4, :299] == 0).all()              # the others over an infinite root
    codes, scale = _plain(ep, dirty, E.F32, codes=True)
    assert np.isnan(scale[[1, 4]]).all() and (codes[[1, 4]] == 0).all() and np.isfinite(scale[fine]).all()


def test_graph_replays(ep):
    """Recorded once and replayed with new inputs, eager calls in between: every replay as the eager call."""
    rng = np.random.default_rng(9)
    rows, h = 4, 1000
    dev = Device(ep)
    kernel = ep.get_kernel({"epsilon": 1e-6}, op_type="GatedResidualNorm")
    data = [rng.standard_normal((2, rows, h)).astype(np.float16) for _ in range(4)]
    try:
        r, b = dev.view(data[0][0], E.F16), dev.view(data[0][1], E.F16)
        z, z_read = dev.output((rows, h), E.F16)
        n, n_read = dev.output((rows, h), E.F16)
        want = []
        for d in data:
            ep.copy_from_host(dev.bufs[0], d[0])
            ep.copy_from_host(dev.bufs[1], d[1])
            kernel.execute([r, b], [z, n])
            want.append((z_read().copy(), n_read().copy()))
        ep.capture_begin()
        kernel.execute([r, b], [z, n])
        graph = ep.capture_end()
        for d, (zw, nw) in zip(data, want):
            ep.copy_from_host(dev.bufs[0], d[0])
            ep.copy_from_host(dev.bufs[1], d[1])
            graph.replay()
            ep.sync()
            assert np.array_equal(z_read(), zw) and np.array_equal(n_read(), nw)
        graph.release()
    finally:
        dev.free()
        kernel.release()


@pytest.mark.parametrize("rows,h,gates,outputs", [(2 ** 21 + 5, 8, 1, "zn"), (2 * (2 ** 21 + 3), 4, 2, "zc")])
def test_more_rows_than_one_launch_takes(ep, rows, h, gates, outputs):
    run(ep, rows, h, E.F16, gates=gates, outputs=outputs)
