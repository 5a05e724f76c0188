"""The operators of the cache where something runs out or grows large: pages, the range of scales and scores, what a caller's workspace has room for."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E

from .cache_helpers import pages_step
from .node_helpers import Device

pytestmark = pytest.mark.gpu

BEHIND = 8192                       # bytes behind a workspace that no call may touch


def step_pages(ep, table, lengths, parents, grow, page, pool, compact=False):
    """CachePages in a workspace of exactly the size that it asks for. -> next table, lengths, moves, counts, the pool after it"""
    dev = Device(ep)
    try:
        kernel = ep.get_kernel({"page_size": page, "compact": int(compact)}, op_type="CachePages")
        i32 = lambda x: dev.view(np.asarray(x, np.int32), E.I32) if x is not None else E.TensorView.absent()  # noqa: E731
        inputs = [i32(table), i32(lengths), i32(parents), i32(grow), dev.view(pool, E.U8)]
        outs = [dev.output(table.shape, E.I32), dev.output((table.shape[0],), E.I32), dev.output((table.shape[0], 2), E.I32), dev.output((2,), E.I32)]
        need, _ = kernel.workspace_requirement([(v.shape, v.dtype) for v in inputs])
        fill = np.full(need + BEHIND, 0xA5, np.uint8)
        ws = dev.view(fill, E.U8)
        kernel.execute(inputs, [o for o, _ in outs] + inputs[4:], workspace=E.DeviceBuffer(ws.data, need))
        ep.sync()
        assert np.array_equal(ep.download(E.DeviceBuffer(ws.data, 0), fill.shape, np.uint8)[need:], fill[need:]), "written behind the workspace"
        kernel.release()
        return [read().copy() for _, read in outs], ep.download(E.DeviceBuffer(inputs[4].data, 0), pool.shape, np.uint8)
    finally:
        dev.free()


@pytest.mark.parametrize("slots,pages,longer", [(4, 20, 0), (128, 64, 0), (200, 64, 1), (256, 16, 0), (1024, 300, 0), (1024, 1022, 1), (1024, 1030, 0), (130, 2, 0)])
def test_more_copies_than_pages(ep, slots, pages, longer):
    """Two prompts that many slots continue, in a pool with a page for some of them: copies that get a page are made, and nothing else."""
    rng = np.random.default_rng(slots + pages)
    table = np.full((slots, 3), -1, np.int32)
    table[:, 0] = np.where(np.arange(slots) < slots // 2, 0, 1)
    lengths, grow = np.full(slots, 5), np.full(slots, 16 * longer)
    pool = rng.integers(0, 256, (2, pages, 48), dtype=np.uint8)
    got, after = step_pages(ep, table, lengths, None, grow, 16, pool)
    want = pages_step(table, lengths, np.arange(slots), grow, 16, pages)
    made = want[2][want[2][:, 1] >= 0]
    assert len(made) == min(slots - 2, pages - 2) if not longer else len(made) <= pages - 2
    for name, g, w in zip(("table", "lengths", "moves", "counts"), got, want):
        assert np.array_equal(g, w), name
    expected = pool.copy()
    expected[:, made[:, 1]] = pool[:, made[:, 0]]
    assert np.array_equal(after, expected)


def held_by(table, lengths, page):
    return {int(p) for row, n in zip(table, lengths) for p in row[:-(-int(n) // page)]}


def without_the_old(want, table, lengths, parents, page):
    """A step that runs out of pages, by the definition: copies into pages that the inputs' table has are not made."""
    next_table, next_lengths, moves, counts = (x.copy() for x in want)
    old = held_by(table, lengths, page)
    for i, (_, to) in enumerate(moves):
        if to >= 0 and int(to) in old:
            next_table[i, next_lengths[i] // page] = -1
            moves[i] = -1
            counts += [-1, 1]
    return next_table, next_lengths, moves, counts


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("slots,width,pages", [(6, 5, 22), (40, 6, 150), (300, 3, 500)])
def test_the_table_of_before_stands_where_pages_run_out(ep, slots, width, pages, seed):
    rng = np.random.default_rng(seed)
    page, order, at = 16, rng.permutation(pages), 0
    table, lengths = np.full((slots, width), -1, np.int32), np.zeros(slots, np.int32)
    for i in range(slots):                                     # sequences until the pool is all but full
        n = int(min(rng.integers(0, width), pages - 2 - at))
        table[i, :n] = order[at:at + n]
        lengths[i] = max(0, n * page - int(rng.integers(0, page)))
        at += n
    parents, grow = rng.integers(0, max(1, slots // 3), slots), np.full(slots, 3 * page)
    pool = rng.integers(0, 256, (3, pages, 52), dtype=np.uint8)
    got, after = step_pages(ep, table, lengths, parents, grow, page, pool)
    plain = pages_step(table, lengths, parents, grow, page, pages)
    want = plain
    if plain[3][1]:                                            # (some of the smaller tables have pages enough)
        want = without_the_old(plain, table, lengths, parents, page)
        old = sorted(held_by(table, lengths, page))
        assert np.array_equal(after[:, old], pool[:, old]), "bytes of the table of before"
    for name, g, w in zip(("table", "lengths", "moves", "counts"), got, want):
        assert np.array_equal(g, w), name
    expected = pool.copy()
    made = want[2][want[2][:, 1] >= 0]
    expected[:, made[:, 1]] = pool[:, made[:, 0]]
    assert np.array_equal(after, expected)
    # other parents, and no growth, from the same table
    again = np.where(np.arange(slots) < 2, np.arange(slots), -1)
    got, last = step_pages(ep, table, lengths, again, None, page, after)
    want = pages_step(table, lengths, again, np.zeros(slots), page, pages)
    for name, g, w in zip(("table", "lengths", "moves", "counts"), got, want):
        assert np.array_equal(g, w), name


@pytest.mark.parametrize("compact", [0, 1])
def test_counts_of_no_slots(ep, compact):
    dev = Device(ep)
    try:
        kernel = ep.get_kernel({"page_size": 16, "compact": compact}, op_type="CachePages")
        none = E.TensorView.absent()
        pool = dev.view(np.arange(2 * 9 * 5, dtype=np.uint8).reshape(2, 9, 5), E.U8)
        counts, read = dev.output((2,), E.I32)
        moves, read_moves = dev.output((4, 2) if compact else (1, 2), E.I32)
        kernel.execute([E.TensorView(None, E.I32, (0, 4)), none, none, none, pool], [none, none, moves if compact else none, counts, pool])
        ep.sync()
        assert read().tolist() == [0, 0]
        if compact:
            assert (read_moves() == -1).all()
        kernel.release()
    finally:
        dev.free()
