"""Calls of the cache's operators at the limits of what they take, on the host: what is empty and what is refused. The GPU's functions are stood for."""
import pytest

from onnx_genai_amd import ep as E

from .test_allocation_failure_cpu import host_only  # noqa: F401  (the fixture: the library's host sources without a GPU)
from .test_cache_nodes_cpu import NONE, Places, cache_views, provider, refused  # noqa: F401  (provider: a fixture)


@pytest.mark.parametrize("compact", [0, 1])
def test_pages_without_slots(provider, compact):  # noqa: F811
    """Counts and moves are checked and written where they are there; nothing else has to be."""
    at = Places()
    table, pool, counts, moves = E.TensorView(None, E.I32, (0, 5)), at(E.U8, (2, 9, 5)), at(E.I32, (2,)), at(E.I32, (4, 2))
    k = provider.get_kernel({"page_size": 16, "compact": compact}, op_type="CachePages")
    before = provider.kernel_launch_count()
    k.execute([table] + [NONE] * 4, [NONE])
    assert provider.kernel_launch_count() == before
    k.execute([table] + [NONE] * 3 + [pool], [NONE, NONE, moves, counts, pool])
    assert provider.kernel_launch_count() == before + 1
    refused(k, [table] + [NONE] * 4, [NONE, NONE, moves, at(E.I64, (2,))], "counts must have dtype Int32")
    refused(k, [table] + [NONE] * 4, [NONE, NONE, moves, at(E.I32, (3,))], "counts must have shape [2]")
    if compact:
        refused(k, [table] + [NONE] * 4, [NONE, NONE, at(E.I32, (4, 3)), counts], "moves must have shape [4, 2]")
        refused(k, [table] + [NONE] * 4, [NONE, NONE, at(E.I32, (8,)), counts], "moves must have shape [P / 2, 2]")
        refused(k, [table] + [NONE] * 4, [NONE, NONE, E.TensorView(counts.data, E.I32, (4, 2)), counts], "counts overlaps moves")
    k.release()


def test_rows_without_sequences(provider):  # noqa: F811
    """A padded batch in which no sequence is left: nothing to do, and the empty table and lengths have no memory."""
    at = Places()
    views = cache_views(at)[:4] + [at(E.I32, (1,)), E.TensorView(None, E.I32, (0,)), E.TensorView(None, E.I32, (0, 5))]
    before = provider.kernel_launch_count()
    k = provider.get_kernel({"kv_num_heads": 2, "head_size": 64}, op_type="CacheAppend")
    k.execute([at(E.F16, (6, 128)), at(E.F16, (6, 128))] + views, views[:4])
    refused(k, [at(E.F16, (6, 128)), at(E.F16, (6, 128))] + views[:6] + [E.TensorView(None, E.I32, (5,))], views[:4], "past_lengths is required")
    k.release()
    k = provider.get_kernel({"num_heads": 4, "kv_num_heads": 2, "head_size": 64}, op_type="CacheAttention")
    k.execute([at(E.F16, (6, 256))] + views, [at(E.F16, (6, 256))])
    k.release()
    assert provider.kernel_launch_count() == before
