"""The plans of the operators beside MatMulNBits as the built library makes them, without a GPU: what scratch a call of given extents takes."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from onnx_genai_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class MoeWeights(C.Structure):
    _fields_ = [("b", C.c_void_p), ("scales", C.c_void_p), ("zp", C.c_void_p), ("bias", C.c_void_p)]


class MoeArgs(C.Structure):
    """RocmMoeArgs of csrc/hip_ffi.h."""
    _fields_ = [("x", C.c_void_p), ("logits", C.c_void_p), ("y", C.c_void_p), ("gate", MoeWeights), ("up", MoeWeights), ("down", MoeWeights), ("up_expert_step", C.c_int64),
                ("up_row_step", C.c_int), ("rows", C.c_int64), ("hidden", C.c_int64), ("inter", C.c_int64), ("experts", C.c_int), ("k", C.c_int), ("block_size", C.c_int),
                ("normalize", C.c_int), ("dtype", C.c_int), ("logits_dtype", C.c_int), ("scale_dtype", C.c_int), ("bias_dtype", C.c_int), ("alpha", C.c_float), ("beta", C.c_float),
                ("limit", C.c_float)]


def moe_workspace(rows, experts, k=2, hidden=64, inter=32, block=32):
    a = MoeArgs()
    a.rows, a.experts, a.k, a.hidden, a.inter, a.block_size = rows, experts, k, hidden, inter, block
    lib = C.CDLL(build.LIB)
    lib.rocm_moe_workspace_bytes.restype = C.c_uint64
    return lib.rocm_moe_workspace_bytes(C.byref(a))


@pytest.mark.parametrize("experts", [4, 256, 257, 512, 1024])
def test_no_rows_take_no_scratch(experts):
    """Asked in a process of its own: a division by an empty grid would end the process that asks."""
    asked = subprocess.run([sys.executable, "-c", f"from tests.test_node_plans_cpu import moe_workspace; print(moe_workspace(0, {experts}))"], cwd=ROOT, capture_output=True, text=True)
    assert asked.returncode == 0, (asked.returncode, asked.stderr)
    assert int(asked.stdout) == 0
    assert moe_workspace(1, experts) > 0
