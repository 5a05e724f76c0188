"""Operators beside MatMulNBits on the host: attributes, refusals with their reasons, scratch, and what supports_op says. The GPU's functions are stood for."""
import ctypes as C

import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .test_allocation_failure_cpu import host_only  # noqa: F401  (the fixture: the library's host sources without a GPU)

HOLD = np.zeros(1 << 16, np.uint8)


def view(dtype, shape, **kw):
    base = HOLD.ctypes.data
    return E.TensorView((base + 255) // 256 * 256 + kw.pop("at", 0), dtype, shape, **kw)


NONE = E.TensorView.absent()


@pytest.fixture
def provider(host_only):  # noqa: F811
    p = E.RocmExecutionProvider(0)
    yield p
    p.shutdown()


def refused(kernel, inputs, outputs, message, **kw):
    with pytest.raises(E.EpError) as e:
        kernel.execute(inputs, outputs, **kw)
    assert e.value.code == 3 and message in e.value.message, e.value.message


@pytest.mark.parametrize("op_type,attrs,message", [
    ("MatMulInt8", dict(N=8), "missing required integer attribute 'K'"),
    ("MatMulInt8", dict(K=8), "missing required integer attribute 'N'"),
    ("MatMulInt8", dict(K=0, N=8), "'K' must be 1..=131071"),
    ("MatMulInt8", dict(K=131072, N=8), "'K' must be 1..=131071"),
    ("MatMulInt8", dict(K=8, N=-1), "'N' must be"),
    ("QMoE", dict(k=2), "missing required integer attribute 'block_size'"),
    ("QMoE", dict(k=0, block_size=32), "'k' must be 1..=64"),
    ("QMoE", dict(k=65, block_size=32), "'k' must be 1..=64"),
    ("QMoE", dict(k=2, block_size=48), "block_size must be a power of two and at least 32"),
    ("QMoE", dict(k=2, block_size=16), "block_size must be a power of two and at least 32"),
    ("QMoE", dict(k=2, block_size=32, expert_weight_bits=8), "expert_weight_bits must be 4"),
    ("QMoE", dict(k=2, block_size=32, swiglu_fusion=3), "swiglu_fusion must be 0, 1 or 2"),
    ("QMoE", dict(k=2, block_size=32, normalize_routing_weights=2), "normalize_routing_weights must be 0 or 1"),
    ("QMoE", dict(k=2, block_size=32, swiglu_limit=0.0), "swiglu_limit must be positive"),
    ("QMoE", dict(k=2, block_size=32, activation_alpha=float("nan")), "must be finite"),
    ("GatedResidualNorm", dict(epsilon=-1.0), "epsilon must be finite and not negative"),
    ("GatedResidualNorm", dict(epsilon=float("nan")), "epsilon must be finite and not negative"),
    ("GatedResidualNorm", dict(residual_scale=float("inf")), "must be finite"),
    ("GatedResidualNorm", dict(layer_norm=2), "layer_norm must be 0 or 1"),
])
def test_attributes(provider, op_type, attrs, message):
    with pytest.raises(E.EpError) as e:
        provider.get_kernel(attrs, op_type=op_type)
    assert message in e.value.message and e.value.message.startswith(op_type + ": ")
    ok, reason = provider.supports_op(attrs, op_type=op_type)
    assert not ok and message in reason


def test_names_that_are_not_there(provider):
    with pytest.raises(ValueError, match="unknown operator"):
        provider.get_kernel({}, op_type="Conv")
    with pytest.raises(ValueError, match="no attribute"):
        provider.get_kernel({"K": 8, "N": 8, "bits": 4}, op_type="MatMulInt8")


def test_a_shorter_struct_reads_as_absent(provider):
    """A caller built against fewer attributes: those past its struct are at their defaults, whatever `present` says."""
    a = E.make_node_attrs("QMoE", {"k": 2, "block_size": 32, "swiglu_limit": -1.0})
    h = C.c_void_p()
    assert provider.lib.nxrt_rocm_qmoe_create(provider.handle, C.byref(a), C.byref(h)).code == 3
    a.struct_size = E.QMoEAttrs.swiglu_limit.offset
    assert provider.lib.nxrt_rocm_qmoe_create(provider.handle, C.byref(a), C.byref(h)).code == 0
    provider.lib.nxrt_rocm_node_release(h)
    for create in (provider.lib.nxrt_rocm_qmoe_create, provider.lib.nxrt_rocm_matmul_int8_create, provider.lib.nxrt_rocm_gated_residual_norm_create):
        assert create(provider.handle, None, C.byref(h)).code == 3 and not h.value


@pytest.mark.parametrize("op_type,attrs,inputs,message", [
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.F16), ((8, 8), E.I8), ((8,), E.F32)], ""),
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.I8), ((8, 8), E.I8), ((8,), E.F32), ((1,), E.F32)], ""),
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.I8), ((8, 8), E.I8), ((8,), E.F32)], "a_scale goes with Int8 A"),
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.U8), ((8, 8), E.I8), ((8,), E.F32)], "A must have a float dtype or Int8"),
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.F16), ((8, 8), E.U8), ((8,), E.F32)], "B must have dtype Int8"),
    ("MatMulInt8", dict(K=8, N=8), [((1, 8), E.F16), ((8, 8), E.I8)], "expected 3..=5 inputs"),
    ("GatedResidualNorm", {}, [((1, 8), E.F16), ((1, 8), E.F16)], ""),
    ("GatedResidualNorm", {}, [((1, 8), E.F16), ((1, 8), E.F32)], "block must have the residual's dtype"),
    ("GatedResidualNorm", {}, [((1, 8), E.I32)], "residual must have a float dtype"),
    ("QMoE", dict(block_size=32, swiglu_fusion=1), [((1, 64), E.F16), ((1, 4), E.F32), ((4, 64, 32), E.U8), ((4, 64, 2), E.F16), (None, 0), ((4, 64, 16), E.U8), ((4, 64, 1), E.F16)], ""),
    ("QMoE", dict(block_size=32), [((1, 64), E.F16), ((1, 4), E.F32), ((4, 64, 32), E.U8), ((4, 64, 2), E.F16), (None, 0), ((4, 64, 16), E.U8), ((4, 64, 1), E.F16)], "fc3 goes with swiglu_fusion=0"),
    ("QMoE", dict(block_size=32, swiglu_fusion=1), [((1, 64), E.F32), ((1, 4), E.F32), ((4, 64, 32), E.U8), ((4, 64, 2), E.F16), (None, 0), ((4, 64, 16), E.U8), ((4, 64, 1), E.F16)],
     "input must have dtype Float16 or BFloat16"),
])
def test_supports(provider, op_type, attrs, inputs, message):
    ok, reason = provider.supports_op(attrs, inputs, op_type=op_type)
    assert ok == (not message) and message in reason


def test_gated_norm_refusals(provider):
    k = provider.get_kernel({}, op_type="GatedResidualNorm")
    r, b, w, z = view(E.F16, (4, 8)), view(E.F16, (4, 8), at=256), view(E.F16, (8,), at=512), view(E.F16, (4, 8), at=1024)
    k.execute([r, b, w], [z])
    refused(k, [], [z], "expected 1..=7 inputs")
    refused(k, [r, b], [], "expected 1..=3 outputs")
    refused(k, [NONE, b], [z], "residual is required")
    refused(k, [view(E.I32, (4, 8))], [z], "residual must have dtype")
    refused(k, [view(E.F16, ())], [z], "residual must have rank >= 1")
    refused(k, [view(E.F16, (1, 32769))], [view(E.F16, (1, 32769))], "the last dimension must be 1..=32768")
    refused(k, [view(E.F16, (4, 0))], [view(E.F16, (4, 0))], "the last dimension must be 1..=32768")
    refused(k, [view(E.F16, (2 ** 32, 8))], [z], "is too large")
    refused(k, [r, view(E.F16, (3, 8), at=256)], [z], "block must have shape [4, 8], got [3, 8]")
    refused(k, [r, view(E.BF16, (4, 8), at=256)], [z], "block must have dtype Float16")
    refused(k, [r, b, view(E.F16, (7,), at=512)], [z], "post_gamma must have shape [8]")
    refused(k, [r, b, view(E.BF16, (8,), at=512)], [z], "post_gamma must have dtype Float16 or Float32")
    refused(k, [r, b, NONE, view(E.F16, (3, 8), at=512)], [z], "G dividing the 4 rows")
    refused(k, [r, b, NONE, view(E.F16, (0, 8), at=512)], [z], "G dividing the 4 rows")
    refused(k, [r, NONE, w], [z], "need a block")
    refused(k, [r, b, NONE, NONE, NONE, NONE, w], [z], "post_beta needs a post_gamma")
    refused(k, [r, b], [NONE, NONE], "neither Z nor N")
    refused(k, [r, b], [z, view(E.I8, (4, 8), at=2048)], "n_scale goes with Int8 N")
    refused(k, [r, b], [z, view(E.F16, (4, 8), at=2048), view(E.F32, (4,), at=4096)], "n_scale goes with Int8 N")
    refused(k, [r, b], [z, view(E.I8, (4, 8), at=2048), view(E.F32, (5,), at=4096)], "n_scale must have one element for each of the 4 rows")
    refused(k, [r, b], [view(E.F16, (4, 8), at=16)], "Z overlaps residual")
    refused(k, [r, b], [z, z], "N overlaps Z")
    refused(k, [r, b], [NONE, view(E.I8, (4, 8)), view(E.F32, (4,), at=4096)], "N overlaps residual")
    refused(k, [r, b, w], [view(E.F16, (1, 8), at=512)], "Z must have shape")
    refused(k, [view(E.F16, (4, 8), strides=(16, 1))], [z], "residual must be contiguous")
    refused(k, [view(E.F16, (4, 8), device_index=1)], [z], "must live on ROCm device 0")
    refused(k, [view(E.F16, (4, 8), device_type=0)], [z], "must live on ROCm device 0")
    refused(k, [view(E.F16, (4, 8), at=1)], [z], "not aligned to its elements")
    k.execute([r, b], [r, b])                                              # over its own inputs
    k.execute([E.TensorView(None, E.F16, (0, 8))], [E.TensorView(None, E.F16, (0, 8))])
    k.release()


def test_int8_refusals(provider):
    k = provider.get_kernel({"K": 32, "N": 8}, op_type="MatMulInt8")
    a, b, s, y = view(E.F16, (3, 32)), view(E.I8, (8, 32), at=256), view(E.F32, (8,), at=1024), view(E.F16, (3, 8), at=2048)
    codes, sa = view(E.I8, (3, 32)), view(E.F32, (3,), at=4096)
    k.execute([a, b, s], [y])
    k.execute([codes, b, s, sa], [y])
    refused(k, [a, b], [y], "expected 3..=5 inputs")
    refused(k, [a, NONE, s], [y], "B is required")
    refused(k, [view(E.F16, (3, 31)), b, s], [y], "A must have last dimension K=32")
    refused(k, [a, view(E.I8, (8, 31), at=256), s], [y], "B must have shape [8, 32]")
    refused(k, [a, view(E.U8, (8, 32), at=256), s], [y], "B must have dtype Int8")
    refused(k, [a, view(E.I8, (8, 32), at=260), s], [y], "B must start at a multiple of 16 bytes")
    refused(k, [a, b, view(E.F32, (7,), at=1024)], [y], "b_scale must have shape [8]")
    refused(k, [a, b, s, sa], [y], "a_scale goes with Int8 A")
    refused(k, [codes, b, s], [y], "a_scale goes with Int8 A")
    refused(k, [codes, b, s, view(E.F32, (2,), at=4096)], [y], "a_scale must have one element")
    refused(k, [a, b, s, NONE, view(E.F16, (2, 8), at=4096)], [y], "bias must have shape [3, 8]")
    refused(k, [a, b, s], [view(E.F16, (3, 7), at=2048)], "Y must have shape [3, 8]")
    refused(k, [a, b, s], [NONE], "Y is required")
    refused(k, [a, b, s], [a], "Y must have shape")
    refused(k, [a, b, s], [view(E.F16, (3, 8), at=128)], "Y overlaps A")
    refused(k, [a, b, s], [view(E.I8, (3, 8), at=2048)], "Y must have dtype")
    k.execute([E.TensorView(None, E.F16, (0, 32)), b, s], [E.TensorView(None, E.F16, (0, 8))])
    k.release()


def test_moe_refusals(provider):
    k = provider.get_kernel({"k": 2, "block_size": 32, "swiglu_fusion": 1}, op_type="QMoE")
    e, h, i = 4, 64, 32
    x, l, y = view(E.F16, (3, h)), view(E.F32, (3, e), at=512), view(E.F16, (3, h), at=1024)
    w1, s1 = view(E.U8, (e, 2 * i, 2, 16), at=2048), view(E.F16, (e, 2 * i, 2), at=16384)
    w2, s2 = view(E.U8, (e, h, 1, 16), at=20480), view(E.F16, (e, h, 1), at=32768)
    base = [x, l, w1, s1, NONE, w2, s2]
    far = dict(at=40960)

    def but(i, v):
        return base[:i] + [v] + base[i + 1:]

    k.execute(base, [y])
    k.execute(but(2, view(E.U8, (e, 2 * i, 32), at=2048)), [y])
    refused(k, base[:6], [y], "expected 7..=14 inputs")
    refused(k, but(0, view(E.F32, (3, h))), [y], "input must have dtype Float16 or BFloat16")
    refused(k, but(1, view(E.F32, (2, e), at=512)), [y], "router_probs must have as many rows")
    refused(k, but(1, view(E.F32, (3, 1), at=512)), [y], "k=2 is more than the 1 experts")
    refused(k, but(1, view(E.F32, (3, 1025), at=512)), [y], "1..=1024 experts")
    refused(k, but(1, view(E.F32, (3, 5), at=512)), [y], "fc1_experts_weights must have shape [5, 64, 2, 16]")
    refused(k, but(2, view(E.U8, (e, 2 * i), at=2048)), [y], "fc1_experts_weights must have rank 3 or 4")
    refused(k, but(2, view(E.U8, (e, 2 * i + 1, 2, 16), at=2048)), [y], "an even number")
    refused(k, but(2, view(E.U8, (e, 2 * i, 2, 16), at=2056)), [y], "must start at a multiple of 16 bytes")
    refused(k, but(3, view(E.BF16, (e, 2 * i, 2), at=16384)), [y], "fc1_scales must have dtype Float16 or Float32")
    refused(k, but(3, view(E.F32, (e, 2 * i, 2), at=16384)), [y], "all scales must have one dtype")
    refused(k, but(3, view(E.F16, (e, 2 * i, 3), at=16384)), [y], "fc1_scales must have shape [4, 64, 2]")
    refused(k, but(4, view(E.F16, (e, i), **far)), [y], "fc1_experts_bias must have shape [4, 64]")
    refused(k, but(5, view(E.U8, (e, h, 2, 16), at=20480)), [y], "fc2_experts_weights must have shape [4, 64, 1, 16]")
    refused(k, base + [NONE, w1], [y], "fc3 goes with swiglu_fusion=0 only")
    refused(k, base + [NONE] * 4 + [view(E.U8, (e, 2 * i, 2), **far)], [y], "fc1_zero_points must have shape [4, 64, 1]")
    refused(k, base, [view(E.BF16, (3, h), at=1024)], "output must have dtype Float16")
    refused(k, base, [view(E.F16, (3, h), at=128)], "output overlaps input")
    refused(k, base, [view(E.F16, (3, h), at=2048)], "output overlaps fc1_experts_weights")
    split = provider.get_kernel({"k": 2, "block_size": 32}, op_type="QMoE")
    refused(split, base, [y], "fc2_experts_weights must have shape [4, 64, 2, 16]")           # (the gate alone is in fc1: I = 64)
    refused(split, base[:5] + [view(E.U8, (e, h, 2, 16), at=20480), view(E.F16, (e, h, 2), at=32768)], [y], "fc3_experts_weights is required")
    big = E.TensorView(x.data, E.F16, (2 ** 23, h)), E.TensorView(x.data, E.F32, (2 ** 23, e)), E.TensorView(x.data, E.F16, (2 ** 23, h))
    refused(k, [big[0], big[1]] + base[2:], [big[2]], "rows times k must be below 2^24")
    k.execute([E.TensorView(None, E.F16, (0, h)), E.TensorView(None, E.F32, (0, e))] + base[2:], [E.TensorView(None, E.F16, (0, h))])
    k.release()
    split.release()


def test_scratch(host_only, provider):  # noqa: F811
    """A call's scratch: the caller's, refused where it is short or not aligned, else the node's own, kept when it is outgrown and never made under capture."""
    k = provider.get_kernel({"K": 32, "N": 8}, op_type="MatMulInt8")
    call = lambda m: ([view(E.F16, (m, 32)), view(E.I8, (8, 32), at=8192), view(E.F32, (8,), at=16384)], [view(E.F16, (m, 8), at=20480)])  # noqa: E731
    need, align = k.workspace_requirement([((3, 32), E.F16), ((8, 32), E.I8), ((8,), E.F32)])
    assert need >= 3 * 128 + 12 and align == 256
    at = view(E.U8, (1,), at=32768).data
    k.execute(*call(3), workspace=E.DeviceBuffer(at, need))
    refused(k, *call(3), "is smaller than the required", workspace=E.DeviceBuffer(at, need - 1))
    refused(k, *call(3), "workspace must be aligned to 256 bytes", workspace=E.DeviceBuffer(at + 16, need))
    provider.capture_begin()
    refused(k, *call(3), "a call under graph capture needs a workspace, or one eager call")
    provider.capture_end()
    failures = C.c_int.in_dll(host_only, "failures_due")
    failures.value = 1
    with pytest.raises(E.EpError) as err:
        k.execute(*call(3))
    assert err.value.code == 7
    k.execute(*call(3))
    assert k.retired_buffers() == 0
    k.execute(*call(60))
    assert k.retired_buffers() == 1
    provider.capture_begin()
    k.execute(*call(40))
    provider.capture_end()
    with pytest.raises(E.EpError):
        k.workspace_requirement([((-1, 32), E.F16)])
    k.release()


@pytest.mark.parametrize("x,logits,w1", [((3, 0), (3, 4), (4, 64, 1, 16)), ((3, 32), (3, 0), (0, 64, 1, 16)), ((3, 32), (3, 4), (4, 0, 1, 16)), ((3, 32), (3, 4), (4, 1, 1, 16)),
                                         ((3, 32), (3, 2048), (2048, 64, 1, 16)), ((2 ** 23, 32), (2 ** 23, 4), (4, 64, 1, 16))])
def test_scratch_of_shapes_that_no_call_takes(provider, x, logits, w1):
    k = provider.get_kernel({"k": 2, "block_size": 32, "swiglu_fusion": 1}, op_type="QMoE")
    with pytest.raises(E.EpError) as err:
        k.workspace_requirement([(x, E.F16), (logits, E.F32), (w1, E.U8)])
    assert err.value.code == 3 and "shapes that no call takes" in err.value.message
    assert k.workspace_requirement([((0, 32), E.F16), ((0, 4), E.F32), ((4, 64, 1, 16), E.U8)])[1] == 256
    k.release()
