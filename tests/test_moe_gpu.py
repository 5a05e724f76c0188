"""QMoE against its definition in 64 bits: from one token to prompts, sizes that divide nothing, each layout and option, padding rows, ties."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, Experts, as64, moe64

pytestmark = pytest.mark.gpu


def check(got, want, noise, dtype, what):
    """Two roundings to the type lie between input and result, of h and of y. A rounding of a value v is off by at most half a step of its binade: evenly spread,
    at most eps / 2 |v| / sqrt(3) in the mean square. h's roundings are independent, so that they are off in y by that times sqrt(noise), noise = sum w^2 h^2 W2^2
    (not by that times |y|: what the experts add may cancel). So each row's error has a mean square of at most (eps / 2)^2 / 3 times |y|^2 + noise; it is
    held to three times that (sqrt(3) in the norm), one element to y's half step and six deviations. The f32 sums before h are off by 2^-16 of their terms' size."""
    half = EPS[dtype] / 2
    nan = np.isnan(want).any(-1)
    assert np.isnan(got[nan]).all(), what
    got, want, noise = got[~nan], want[~nan], noise[~nan]
    assert np.isfinite(got).all(), what
    if not want.size:
        return
    assert (got[np.abs(want).sum(-1) == 0] == 0).all(), what
    err = np.abs(got - want)
    spread = np.sqrt(noise)
    if want.shape[-1] >= 64:
        size = np.sqrt((want ** 2 + noise).sum(-1))
        off = np.linalg.norm(err, axis=-1)
        assert (off <= (half + 2.0 ** -13) * size).all(), (what, (off / np.maximum(size, 1e-300)).max(), half)
    bound = half * np.abs(want) * (1 + 2 ** -8) + (6 / np.sqrt(3) * half + 2.0 ** -12) * spread
    assert (err <= bound).all(), (what, (err / np.maximum(bound, 1e-300)).max())


def run(ep, rows, experts, k, hidden, inter, block, dtype, *, fusion=1, zero_points=False, bias=False, normalize=True, clamped=False, logits=None, logits_dtype=None, scale_dtype=None,
        bias_dtype=None, x=None, seed=0, offset=0, workspace=False, flat=False, fc3=False, shape=None, again=False):
    rng = np.random.default_rng(seed + rows * 11 + experts * 5 + hidden + inter)
    logits_dtype = logits_dtype or E.F32
    make = lambda n, d: Experts(rng, experts, n, d, block, dtype, zero_points=zero_points, bias=bias, scale_dtype=scale_dtype, bias_dtype=bias_dtype)  # noqa: E731
    fc1, fc2 = make(inter if fusion == 0 else 2 * inter, hidden), make(hidden, inter)
    third = make(inter, hidden) if fusion == 0 else None
    x = synth.to_dtype(rng.standard_normal((rows, hidden)).astype(np.float32), dtype) if x is None else x
    logits = synth.to_dtype((rng.standard_normal((rows, experts)) * 1.5).astype(np.float32) if logits is None else np.asarray(logits, np.float32), logits_dtype)
    attrs = {"k": k, "block_size": block, "swiglu_fusion": fusion, "normalize_routing_weights": int(normalize)}
    extra = {"alpha": 1.702, "beta": 1.0, "limit": 1.5} if clamped else {}
    if clamped:
        attrs.update(activation_alpha=1.702, activation_beta=1.0, swiglu_limit=1.5)
    want, noise = moe64(as64(x, dtype), as64(logits, logits_dtype), fc1, fc2, third, k=k, normalize=normalize, fusion=fusion, **extra)
    dev = Device(ep)
    kernel = ep.get_kernel(attrs, op_type="QMoE")
    lead = shape or (rows,)
    try:
        inputs = [dev.view(x, dtype, (*lead, hidden), offset), dev.view(logits, logits_dtype, (*lead, experts), offset)]
        packed = lambda p: dev.view(p.b, E.U8, (*p.b.shape[:2], p.b.shape[2] * p.b.shape[3]) if flat else None)  # noqa: E731
        for p in (fc1, fc2, third):
            inputs += [packed(p), dev.view(p.scales, p.scale_dtype, None, offset), dev.view(p.bias, p.bias_dtype, None, offset)] if p is not None else [E.TensorView.absent()] * 3
        inputs += [dev.view(p.zp, E.U8, None, offset) if p is not None else E.TensorView.absent() for p in (fc1, fc2, third)]
        y, read = dev.output((*lead, hidden), dtype, offset)
        ws = None
        if workspace:
            need, align = kernel.workspace_requirement([(v.shape if v.data else None, v.dtype) for v in inputs])
            ws = ep.allocate(need, align)
            dev.bufs.append(ws)
        kernel.execute(inputs, [y], workspace=ws)
        got = read().reshape(rows, hidden)
        variant = kernel.last_variant()
        if again:                                     # the same bits each time, though atomics order an expert's rows
            for _ in range(3):
                kernel.execute(inputs, [y], workspace=ws)
                assert np.array_equal(read().reshape(rows, hidden).view(np.uint16), got.view(np.uint16))
    finally:
        dev.free()
        kernel.release()
    check(as64(got, dtype), want, noise, dtype, (variant, rows, experts, k, hidden, inter, block))
    return got, variant


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 33, 48, 64, 65, 100, 150])
@pytest.mark.parametrize("dtype", [E.F16, E.BF16])
def test_rows(ep, rows, dtype):
    run(ep, rows, 8, 2, 256, 128, 32, dtype, again=True)


@pytest.mark.parametrize("block", [32, 64, 128, 256])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows", [1, 6, 20, 70, 300])
def test_blocks(ep, rows, block, zero_points):
    run(ep, rows, 4, 2, 512, 384, block, E.F16, zero_points=zero_points)
    run(ep, rows, 4, 2, 512, 384, block, E.BF16, zero_points=zero_points, bias=True)


@pytest.mark.parametrize("hidden,inter", [(64, 64), (72, 40), (96, 33), (100, 17), (101, 50), (288, 288), (130, 1000), (1000, 90), (520, 264), (257, 129)])
@pytest.mark.parametrize("rows", [1, 3, 18, 80])
def test_sizes(ep, rows, hidden, inter):
    run(ep, rows, 4, 2, hidden, inter, 32, E.F16, bias=True)
    run(ep, rows, 4, 2, hidden, inter, 64, E.BF16, zero_points=True)


@pytest.mark.parametrize("fusion", [0, 1, 2])
@pytest.mark.parametrize("rows", [1, 7, 40, 200])
def test_layouts(ep, rows, fusion):
    run(ep, rows, 8, 3, 256, 160, 32, E.F16, fusion=fusion, bias=True, zero_points=True)
    run(ep, rows, 8, 3, 256, 160, 128, E.BF16, fusion=fusion, flat=True)


@pytest.mark.parametrize("experts,k", [(1, 1), (2, 2), (5, 5), (64, 8), (65, 6), (128, 8), (200, 3), (257, 7), (1024, 4), (64, 64)])
@pytest.mark.parametrize("rows", [1, 4, 21, 130])
def test_experts(ep, rows, experts, k):
    run(ep, rows, experts, k, 64, 32, 32, E.F16, again=experts == 64)


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("clamped", [False, True])
@pytest.mark.parametrize("rows", [1, 12, 90])
def test_options(ep, rows, normalize, clamped):
    run(ep, rows, 8, 4, 128, 96, 32, E.BF16, normalize=normalize, clamped=clamped, bias=True)


@pytest.mark.parametrize("dtype,logits_dtype,scale_dtype,bias_dtype", [(E.F16, E.F16, E.F32, E.F32), (E.BF16, E.BF16, E.F32, E.F32), (E.BF16, E.F32, E.BF16, E.F32), (E.F16, E.F32, E.F32, E.F16)])
@pytest.mark.parametrize("rows", [1, 10, 100])
def test_types(ep, rows, dtype, logits_dtype, scale_dtype, bias_dtype):
    run(ep, rows, 8, 2, 128, 64, 32, dtype, logits_dtype=logits_dtype, scale_dtype=scale_dtype, bias_dtype=bias_dtype, bias=True)


@pytest.mark.parametrize("rows", [1, 5, 40, 150])
def test_ties_go_to_the_lowest_index(ep, rows):
    rng = np.random.default_rng(2)
    logits = rng.integers(0, 3, (rows, 70)).astype(np.float32)             # many equal ones at every border
    logits[0, :] = 0.0
    logits[0, 40:] = -0.0                                                  # equal to 0
    run(ep, rows, 70, 6, 64, 32, 32, E.F16, logits=logits)


@pytest.mark.parametrize("rows", [1, 4, 16, 33, 200])
def test_padding_rows_and_masked_experts(ep, rows):
    rng = np.random.default_rng(rows)
    logits = rng.standard_normal((rows, 16)).astype(np.float32)
    logits[rows // 2:] = -np.inf                                           # rows of no sequence
    logits[: rows // 2, 3:14] = -np.inf                                    # fewer experts than k are left
    run(ep, rows, 16, 6, 64, 64, 32, E.BF16, logits=logits, normalize=False)
    got, _ = run(ep, rows, 16, 6, 64, 64, 32, E.BF16, logits=np.full((rows, 16), -np.inf), bias=True)
    assert not got.any()


@pytest.mark.parametrize("rows", [1, 3, 20, 120])
def test_logits_that_are_not_numbers(ep, rows):
    rng = np.random.default_rng(rows)
    logits = rng.standard_normal((rows, 8)).astype(np.float32)
    logits[rows - 1, 5] = np.nan if rows % 2 else np.inf
    run(ep, rows, 8, 2, 64, 32, 32, E.F16, logits=logits)
    logits[rows - 1] = [np.float32(-3.4e38)] * 7 + [np.float32(3.4e38)]    # the lowest numbers there are: one expert is left
    run(ep, rows, 8, 2, 64, 32, 32, E.F16, logits=logits)
    logits[rows - 1] = np.float32(-3.4e38)                                 # and equal ones
    run(ep, rows, 8, 2, 64, 32, 32, E.F16, logits=logits)


@pytest.mark.parametrize("rows", [2, 18, 130])
def test_inputs_that_are_not_finite_leave_the_other_rows_alone(ep, rows):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, 64)).astype(np.float16)
    logits = rng.standard_normal((rows, 4)).astype(np.float32)
    clean, _ = run(ep, rows, 4, 2, 64, 32, 32, E.F16, x=x, logits=logits)
    for value in (np.inf, np.nan):
        dirty = x.copy()
        dirty[1, 9] = value
        dev = Device(ep)
        kernel = ep.get_kernel({"k": 2, "block_size": 32, "swiglu_fusion": 1, "normalize_routing_weights": 1}, op_type="QMoE")
        g = np.random.default_rng(rows * 11 + 4 * 5 + 64 + 32)
        fc1, fc2 = Experts(g, 4, 64, 64, 32, E.F16), Experts(g, 4, 64, 32, 32, E.F16)
        y, read = dev.output((rows, 64), E.F16)
        none = E.TensorView.absent()
        kernel.execute([dev.view(dirty, E.F16), dev.view(logits, E.F32), dev.view(fc1.b, E.U8), dev.view(fc1.scales, E.F16), none, dev.view(fc2.b, E.U8), dev.view(fc2.scales, E.F16)], [y])
        got = read()
        dev.free()
        kernel.release()
        others = [r for r in range(rows) if r != 1]
        assert np.array_equal(got[others], clean[others]) and not np.isfinite(got[1]).any()


@pytest.mark.parametrize("rows", [1, 9, 90])
def test_every_token_to_one_expert(ep, rows):
    logits = np.zeros((rows, 32), np.float32)
    logits[:, 17] = 5.0
    logits[:, 4] = 4.0
    run(ep, rows, 32, 2, 128, 64, 32, E.F16, logits=logits)


@pytest.mark.parametrize("rows", [1, 5, 30, 140])
def test_elements_anywhere_and_callers_workspace(ep, rows):
    run(ep, rows, 4, 2, 136, 72, 32, E.F16, offset=3, bias=True, zero_points=True, workspace=True)


@pytest.mark.parametrize("block,inter", [(32, 2176), (64, 4224), (128, 3000), (256, 2049)])
@pytest.mark.parametrize("rows", [5, 17, 90])
def test_down_in_slices_of_its_k(ep, rows, block, inter):
    run(ep, rows, 4, 2, 200, inter, block, E.BF16, zero_points=True, again=True)
    run(ep, rows, 4, 2, 200, inter, block, E.F16, scale_dtype=E.F32, bias=True)


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("dtype,scale_dtype", [(E.F16, E.F32), (E.BF16, E.F32), (E.BF16, E.BF16), (E.F16, E.F16)])
def test_tiles_of_128_pairs(ep, block, dtype, scale_dtype):
    _, variant = run(ep, 333, 3, 2, 192, 160, block, dtype, scale_dtype=scale_dtype, zero_points=block == 64, bias=True)
    assert variant == "moe_tiles_128"


def test_leading_dimensions(ep):
    run(ep, 12, 4, 2, 64, 32, 32, E.F16, shape=(2, 3, 2))


@pytest.mark.parametrize("rows,experts,k,hidden,inter,block,dtype", [(1, 32, 8, 2048, 1024, 32, E.BF16), (3, 4, 2, 1024, 3584, 32, E.F16), (48, 16, 8, 1024, 512, 64, E.BF16),
                                                                    (777, 8, 4, 720, 720, 32, E.F16), (1000, 16, 8, 512, 256, 128, E.BF16)])
def test_real_sizes(ep, rows, experts, k, hidden, inter, block, dtype):
    run(ep, rows, experts, k, hidden, inter, block, dtype, bias=rows == 777, clamped=rows == 777)


@pytest.mark.parametrize("rows", [1, 12, 150])
def test_graphs_that_share_a_node(ep, rows):
    """Two graphs of one node, hence of one scratch, replayed in turn with eager calls of another height between them."""
    rng = np.random.default_rng(rows)
    e, k, h, i = 8, 2, 128, 64
    fc1, fc2 = Experts(rng, e, 2 * i, h, 32, E.F16), Experts(rng, e, h, i, 32, E.F16)
    dev = Device(ep)
    kernel = ep.get_kernel({"k": k, "block_size": 32, "swiglu_fusion": 1}, op_type="QMoE")
    none = E.TensorView.absent()
    try:
        weights = [dev.view(fc1.b, E.U8), dev.view(fc1.scales, E.F16), none, dev.view(fc2.b, E.U8), dev.view(fc2.scales, E.F16)]
        calls = []
        for m in (rows, rows, 2 * rows):
            x, l = rng.standard_normal((m, h)).astype(np.float16), rng.standard_normal((m, e)).astype(np.float32)
            y, read = dev.output((m, h), E.F16)
            calls.append(([dev.view(x, E.F16), dev.view(l, E.F32)] + weights, [y], read))
        want = []
        for inputs, outputs, read in calls:
            kernel.execute(inputs, outputs)
            want.append(read().copy())
        graphs = []
        for inputs, outputs, _ in calls[:2]:
            ep.capture_begin()
            kernel.execute(inputs, outputs)
            graphs.append(ep.capture_end())
        for _ in range(3):
            for i_graph, graph in enumerate(graphs):
                graph.replay()
                ep.sync()
                assert np.array_equal(calls[i_graph][2](), want[i_graph])
                kernel.execute(*calls[2][:2])
                assert np.array_equal(calls[2][2](), want[2])
        for graph in graphs:
            graph.release()
    finally:
        dev.free()
        kernel.release()
