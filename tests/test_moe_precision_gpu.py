"""QMoE where its precision can go wrong: up to four tokens, whose h is not rounded, values far larger than the rest at weights that are zero, values below the
normal numbers of f16."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, Experts, as64, moe64

pytestmark = pytest.mark.gpu


def silence(p, k, block):
    """Element k of every row of every expert gets its zero point as weight."""
    at, low = (k // block, k % block // 2), k % 2 == 0
    zero = np.full(p.b.shape[:2], 8, np.uint8) if p.zp is None else (p.zp[..., at[0] // 2] >> (4 * (at[0] % 2))) & 15
    byte = p.b[:, :, at[0], at[1]]
    p.b[:, :, at[0], at[1]] = (byte & 0xf0) | zero if low else (byte & 0x0f) | (zero << 4)
    p.w[..., k] = 0


def call(ep, x, logits, fc1, fc2, dtype, block):
    dev = Device(ep)
    kernel = ep.get_kernel({"k": 2, "block_size": block, "swiglu_fusion": 2, "normalize_routing_weights": 1}, op_type="QMoE")
    none = E.TensorView.absent()
    try:
        inputs = [dev.view(x, dtype), dev.view(logits, E.F32)]
        for p in (fc1, fc2):
            inputs += [dev.view(p.b, E.U8), dev.view(p.scales, p.scale_dtype), dev.view(p.bias, p.bias_dtype)]
        inputs += [none] * 3 + [dev.view(p.zp, E.U8) for p in (fc1, fc2)]
        y, read = dev.output(x.shape, dtype)
        kernel.execute(inputs, [y])
        return as64(read(), dtype), kernel.last_variant()
    finally:
        dev.free()
        kernel.release()


def check(got, want, noise, dtype, variant, below_normal=0.0):
    """Half a step of y, and what f32 sums and h's two parts leave in front of it. A lane's 16 products of two, four chains of them and six sums over lanes are some ten
    roundings of 2^-24, each of a part of the sum: 2^-20 of the size of g and u, and again of y's; exp and the quotient 2^-21; the parts of h 2^-22 (f16) or 2^-18 (bf16)
    of it. All are independent over the columns of h, which makes them that much of sqrt(noise) in y: 2^-13 of it is eight times 2^-16, a row's largest.
    Tiles (five tokens and more) round h once: another half step, evenly spread and independent, six deviations of it.
    below_normal: the mean square of what h's fixed step of 2^-24 below the normal numbers leaves in y."""
    half = EPS[dtype] / 2
    rounded = 0.0 if variant == "moe_few" else 6 / np.sqrt(3) * half
    bound = half * np.abs(want) * (1 + 2 ** -8) + (2.0 ** -13 + rounded) * np.sqrt(noise) + 6 * np.sqrt(below_normal) + (2.0 ** -25 if dtype == E.F16 else 0)
    off = np.abs(got - want)
    assert (off <= bound).all(), (variant, (off / bound).max(), (off > bound).mean())


def operands(rows, dtype, zero_points, bias=False, scale_dtype=None, block=32, hidden=1024, inter=256):
    rng = np.random.default_rng(rows * 7 + block + 2 * zero_points)
    options = dict(zero_points=zero_points, bias=bias, scale_dtype=scale_dtype, bias_dtype=E.F32)
    fc1, fc2 = Experts(rng, 4, 2 * inter, hidden, block, dtype, **options), Experts(rng, 4, hidden, inter, block, dtype, **options)
    return rng.standard_normal((rows, hidden)).astype(np.float32), (rng.standard_normal((rows, 4)) * 1.5).astype(np.float32), fc1, fc2


def compare(ep, x, logits, fc1, fc2, dtype, block=32, below_normal=None):
    want, noise = moe64(as64(x, dtype), logits.astype(np.float64), fc1, fc2, None, k=2, normalize=True, fusion=2)
    got, variant = call(ep, x, logits, fc1, fc2, dtype, block)
    assert (variant == "moe_few") == (x.shape[0] <= 4)
    extra = 0.0
    if below_normal is not None:
        # two experts a token, weights at most 1: sum of (2^-24)^2 / 12 over the columns of h, of the experts that have the largest weights
        extra = 2 * (2.0 ** -48 / 12) * (fc2.w ** 2).sum(-1).max(0)
    check(got, want, noise, dtype, variant, extra)


@pytest.mark.parametrize("dtype", [E.F16, E.BF16])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 4])
def test_h_of_few_tokens_is_not_rounded(ep, rows, dtype, zero_points):
    for block in (32, 128):
        x, logits, fc1, fc2 = operands(rows, dtype, zero_points, bias=True, block=block)
        compare(ep, synth.to_dtype(x, dtype), logits, fc1, fc2, dtype, block)


@pytest.mark.parametrize("dtype,size", [(E.F16, 4000.0), (E.F16, 60000.0), (E.BF16, 2.0 ** 17), (E.BF16, 2.0 ** 30)])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 4, 9, 300])
def test_large_values_at_weights_of_zero_add_nothing(ep, rows, dtype, size, zero_points):
    x, logits, fc1, fc2 = operands(rows, dtype, zero_points)
    for k in (0, 37, 1023):
        x[:, k] = size if k != 37 else -size
        for p in (fc1,):
            silence(p, k, 32)
    compare(ep, synth.to_dtype(x, dtype), logits, fc1, fc2, dtype)


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 4, 9])
@pytest.mark.parametrize("dtype,gate,up", [(E.F16, 200.0, 150.0), (E.BF16, 1000.0, 1000.0)])
def test_large_h_at_weights_of_zero_adds_nothing(ep, rows, dtype, gate, up, zero_points):
    x, logits, fc1, fc2 = operands(rows, dtype, zero_points, bias=True)
    for j in (0, 77, 255):
        fc1.bias[:, j], fc1.bias[:, 256 + j] = gate, up
        fc1.bias64[:, j], fc1.bias64[:, 256 + j] = gate, up
        silence(fc2, j, 32)
    compare(ep, synth.to_dtype(x, dtype), logits, fc1, fc2, dtype)


@pytest.mark.parametrize("rows", [1, 3, 9, 300])
def test_x_below_the_normal_numbers_of_f16(ep, rows):
    x, logits, fc1, fc2 = operands(rows, E.F16, False, scale_dtype=E.F32)
    fc1.scales, fc1.w = fc1.scales * np.float32(2 ** 17), fc1.w * 2.0 ** 17
    compare(ep, (x * 2.0 ** -17).astype(np.float16), logits, fc1, fc2, E.F16)


@pytest.mark.parametrize("rows", [1, 3, 9, 300])
def test_h_below_the_normal_numbers_of_f16(ep, rows):
    x, logits, fc1, fc2 = operands(rows, E.F16, False, scale_dtype=E.F32)
    fc1.scales, fc1.w = fc1.scales * np.float32(2 ** -8), fc1.w * 2.0 ** -8
    fc2.scales, fc2.w = fc2.scales * np.float32(2 ** 16), fc2.w * 2.0 ** 16
    compare(ep, x.astype(np.float16), logits, fc1, fc2, E.F16, below_normal=True)
