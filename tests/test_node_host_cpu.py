"""What the operators beside MatMulNBits keep to on the host: counted steps, scratch, reasons. The GPU's functions are stood for."""
import ctypes as C

import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .test_allocation_failure_cpu import host_only  # noqa: F401  (the fixture: the library's host sources without a GPU)

HOLD = np.zeros(1 << 20, np.uint8)
NONE = E.TensorView.absent()


def view(dtype, shape, at=0):
    return E.TensorView((HOLD.ctypes.data + 255) // 256 * 256 + at, dtype, shape)


@pytest.fixture
def provider(host_only):  # noqa: F811
    p = E.RocmExecutionProvider(0)
    yield p
    p.shutdown()


def int8_call(rows, dtype=E.F16, k=32):
    scale = [view(E.F32, (rows,), 1 << 17)] if dtype == E.I8 else []
    return [view(dtype, (rows, k)), view(E.I8, (8, k), 1 << 18), view(E.F32, (8,), 1 << 19)] + scale, [view(E.F16, (rows, 8), 3 << 18)]


@pytest.mark.parametrize("dtype", [E.F16, E.F32, E.I8])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 33), (40, 32), (500, 33)])
def test_a_product_is_one_step(provider, rows, k, dtype):
    """One for a product with all that it takes: quantized rows, padded rows, slices of K."""
    kernel = provider.get_kernel({"K": k, "N": 8}, op_type="MatMulInt8")
    before = provider.kernel_launch_count()
    kernel.execute(*int8_call(rows, dtype, k))
    assert provider.kernel_launch_count() == before + 1
    kernel.release()


def test_outgrown_scratch_is_freed_until_a_capture_was_opened(provider):
    """Calls of growing length, as prompts are: while no graph can name the scratch, a node has one."""
    kernel = provider.get_kernel({"K": 32, "N": 8}, op_type="MatMulInt8")
    for rows in (4, 40, 400, 1000):
        kernel.execute(*int8_call(rows))
        assert kernel.retired_buffers() == 0
    provider.capture_begin()
    kernel.execute(*int8_call(1000))
    provider.capture_end()
    kernel.execute(*int8_call(2000))
    assert kernel.retired_buffers() == 1                     # what the recorded call names
    kernel.release()


@pytest.mark.parametrize("op_type,attrs", [("QMoE", {"k": 2, "block_size": 32}), ("MatMulInt8", {"K": 32, "N": 8}), ("GatedResidualNorm", {})])
def test_no_reason_where_a_node_is_supported(provider, op_type, attrs):
    """What the caller's buffer held before is no reason."""
    a = E.make_node_attrs(op_type, attrs)
    supports = getattr(provider.lib, f"nxrt_rocm_ep_supports_{E._NODE_OPS[op_type][1]}")
    reason = C.create_string_buffer(b"left from before", 64)
    assert supports(provider.handle, C.byref(a), None, 0, reason, 64) == 1 and reason.value == b""
    assert supports(provider.handle, C.byref(a), None, 0, None, 0) == 1
