"""CachePages against its definition: tables, moves and counts, and every byte of the pools."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .cache_helpers import pages_compact, pages_step
from .node_helpers import Device

pytestmark = pytest.mark.gpu


def run(ep, table, lengths, parents, grow, page, pages, pools, compact=False):
    """pools: host arrays [L, P, ..] with their types. -> next table, lengths, moves, counts, pools"""
    dev = Device(ep)
    try:
        kernel = ep.get_kernel({"page_size": page, "compact": int(compact)}, op_type="CachePages")
        i32 = lambda x: dev.view(np.asarray(x, np.int32), E.I32) if x is not None else E.TensorView.absent()  # noqa: E731
        views = [dev.view(x, dt) for x, dt in pools]
        outs = [dev.output(table.shape, E.I32), dev.output((table.shape[0],), E.I32), dev.output((pages // 2 if compact else table.shape[0], 2), E.I32), dev.output((2,), E.I32)]
        kernel.execute([i32(table), i32(lengths), i32(parents), i32(grow)] + views, [o for o, _ in outs] + views)
        ep.sync()
        got = [read().copy() for _, read in outs]
        after = [ep.download(E.DeviceBuffer(v.data, 0), x.shape, x.dtype) for v, (x, _) in zip(views, pools)]
        kernel.release()
        return got, after
    finally:
        dev.free()


def some_pools(rng, pages, layers=2):
    return [(rng.integers(-127, 128, (layers, pages, 2, 16, 40), dtype=np.int8), E.I8), (rng.integers(0, 255, (layers, pages, 10004), dtype=np.uint8), E.U8),
            (rng.standard_normal((layers, pages, 3)).astype(np.float32), E.F32), (rng.integers(0, 255, (1, pages, 5), dtype=np.uint8), E.U8)]


def check(ep, table, lengths, parents, grow, page, pages, *, compact=False, layers=2):
    rng = np.random.default_rng(pages)
    pools = some_pools(rng, pages, layers)
    got, after = run(ep, table, lengths, parents, grow, page, pages, pools, compact)
    p = np.arange(table.shape[0]) if parents is None else np.asarray(parents)
    want = pages_compact(table, lengths, page, pages) if compact else pages_step(table, lengths, p, np.zeros(len(p)) if grow is None else grow, page, pages)
    for name, g, w in zip(("table", "lengths", "moves", "counts"), got, want):
        assert np.array_equal(g, w), name
    for (x, _), a in zip(pools, after):
        expected = x.copy()
        for source, to in want[2]:
            if to >= 0:
                expected[:, to] = x[:, source]
        assert np.array_equal(a, expected)
    return want


def tables(rng, slots, width, page, pages, longest, share=False):
    order, at = rng.permutation(pages), 0
    table, lengths = np.full((slots, width), -1, np.int32), np.zeros(slots, np.int32)
    for i in range(slots):
        lengths[i] = rng.integers(0, longest + 1)
        n = -(-lengths[i] // page)
        for j in range(n):
            if share and i and rng.random() < 0.5 and j < lengths[i - 1] // page:
                table[i, j] = table[i - 1, j]
            else:
                table[i, j] = order[at]
                at += 1
    return table, lengths


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("slots,page,pages", [(1, 16, 40), (8, 16, 300), (33, 64, 700), (5, 1, 900), (100, 48, 4000)])
def test_steps(ep, slots, page, pages, seed):
    """Beams that continue one another, end, and grow by none, one or many tokens."""
    rng = np.random.default_rng(100 * seed + slots)
    table, lengths = tables(rng, slots, 14, page, pages, min(10 * page, 300), share=seed % 2 == 1)
    parents = rng.integers(-1, slots, slots) if seed < 6 else None
    grow = [None, np.ones(slots, int), rng.integers(0, 4 * page, slots)][seed % 3]
    check(ep, table, lengths, parents, grow, page, pages)


def test_a_page_begun_here_and_whole_there(ep):
    """A sequence that was cut back into a page that another one has filled: it gets a copy, whatever its place."""
    table = np.array([[3, 4, -1], [3, 5, -1], [3, 6, -1]], np.int32)
    want = check(ep, table, [32, 10, 16], None, [1, 1, 1], 16, 12)
    assert want[2].tolist() == [[-1, -1], [3, 1], [-1, -1]]          # (page 0, the lowest free one, goes to the first sequence's 33rd token)
    assert check(ep, table, [10, 10, 10], None, [1, 1, 1], 16, 12)[2].tolist() == [[-1, -1], [3, 0], [3, 1]]


def test_all_ended(ep):
    table, lengths = tables(np.random.default_rng(1), 6, 8, 16, 60, 100)
    want = check(ep, table, lengths, [-1] * 6, [5] * 6, 16, 60)
    assert want[3].tolist() == [0, 0] and (want[0] == -1).all()


def test_too_few_pages(ep):
    """Entries that get no page are -1 and counted, and the table of before still stands."""
    table, lengths = tables(np.random.default_rng(2), 4, 8, 16, 20, 70)
    want = check(ep, table, lengths, [0, 0, 0, 0], [100, 100, 100, 100], 16, 20)
    assert want[3][1] > 0


def test_values_out_of_range(ep):
    """Parents, lengths, entries and growth that are none."""
    table = np.array([[1, 2, 99], [-1, 2, 0], [2 ** 31 - 1, -2 ** 31, 1]], np.int32)
    for lengths in ([20, 40, 2 ** 31 - 1], [-5, 48, 33]):
        for parents in ([0, 1, 2], [7, 2, 2], [-2 ** 31, 2 ** 31 - 1, 1]):
            check(ep, table, lengths, parents, [2 ** 31 - 1, -3, 1], 16, 10)
        check(ep, table, lengths, None, None, 16, 10, compact=True)


@pytest.mark.parametrize("slots,page,pages,longest", [(1, 16, 1, 16), (1, 16, 2, 16), (3, 16, 31, 80), (20, 64, 333, 500), (60, 16, 1500, 300), (8, 16, 100, 0), (1000, 16, 5000, 60), (30, 16, 8192 + 5, 900)])
@pytest.mark.parametrize("share", [False, True])
def test_compact(ep, slots, page, pages, longest, share):
    rng = np.random.default_rng(pages)
    table, lengths = tables(rng, slots, max(1, -(-longest // page)), page, pages, longest, share)
    check(ep, table, lengths, None, None, page, pages, compact=True, layers=1)


def test_the_most_slots(ep):
    rng = np.random.default_rng(3)
    table, lengths = tables(rng, 1024, 4, 16, 6000, 60)
    check(ep, table, lengths, rng.integers(-1, 1024, 1024), np.ones(1024, int), 16, 6000, layers=1)


def test_the_most_pages(ep):
    """Ids up to 2^18 in both modes."""
    rng = np.random.default_rng(4)
    pages = 1 << 18
    table = rng.choice(pages, (64, 40), replace=False).astype(np.int32)
    table[0, 0], table[1, 1] = pages - 1, 0
    table[63, 39] = pages - 2
    lengths = np.full(64, 39 * 16 + 3, np.int32)
    pools = [(rng.integers(0, 255, (1, pages, 16), dtype=np.uint8), E.U8)]
    for compact in (False, True):
        got, after = run(ep, table, lengths, None if compact else np.arange(64) // 2, None if compact else np.full(64, 20), 16, pages, pools, compact)
        want = pages_compact(table, lengths, 16, pages) if compact else pages_step(table, lengths, np.arange(64) // 2, np.full(64, 20), 16, pages)
        for g, w in zip(got, want):
            assert np.array_equal(g, w)
        expected = pools[0][0].copy()
        moved = want[2][want[2][:, 1] >= 0]
        expected[:, moved[:, 1]] = pools[0][0][:, moved[:, 0]]
        assert np.array_equal(after[0], expected)


def test_no_slots(ep):
    kernel = ep.get_kernel({"page_size": 16}, op_type="CachePages")
    none = E.TensorView.absent()
    kernel.execute([E.TensorView(None, E.I32, (0, 4)), none, none, none, none], [none])
    kernel.release()
