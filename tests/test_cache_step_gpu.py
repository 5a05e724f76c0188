"""The operators of a cache as a decoder layer uses them together: qkv product -> rotary positions -> append -> attention -> o product, with the pages of each step, eagerly, recorded, and
through two providers at once."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .cache_helpers import Cache, append32, attention64, pages_step, same_values
from .node_helpers import EPS, Device, as64

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HEAD, PAGE, BLOCK = 256, 6, 2, 64, 16, 32
PACKED, WIDE = (HEADS + 2 * KV) * HEAD, HEADS * HEAD
DTYPE = E.F16


class Layer:
    """One layer and its cache on one provider."""

    def __init__(self, ep, code, slots, width, pages, seed):
        rng = np.random.default_rng(seed)
        self.ep, self.dev, self.code, self.slots, self.width, self.pages = ep, Device(ep), code, slots, width, pages
        self.weights = [synth.make_weights(n, k, BLOCK, seed + i, zero_points=False, scale_lo=0.01, scale_hi=0.02, scale_dtype=DTYPE) for i, (n, k) in enumerate(((PACKED, HIDDEN), (HIDDEN, WIDE)))]
        make = lambda n, k: ep.get_kernel({"K": k, "N": n, "bits": 4, "block_size": BLOCK})  # noqa: E731
        self.qkv, self.o = make(PACKED, HIDDEN), make(HIDDEN, WIDE)
        for k in (self.qkv, self.o):
            k.set_constant_inputs([False, True, True])
        self.w = [[self.dev.view(b, E.U8), self.dev.view(s, DTYPE)] for b, s, _ in self.weights]
        self.rotary = ep.get_kernel({"head_size": HEAD, "num_heads": HEADS + KV, "scaling": 2, "factor": 8.0}, op_type="RotaryEmbedding")
        self.append = ep.get_kernel({"num_heads": HEADS, "kv_num_heads": KV, "head_size": HEAD}, op_type="CacheAppend")
        self.attend = ep.get_kernel({"num_heads": HEADS, "kv_num_heads": KV, "head_size": HEAD}, op_type="CacheAttention")
        self.step = ep.get_kernel({"page_size": PAGE}, op_type="CachePages")
        np_type = np.int8 if code == E.I8 else np.uint8
        self.host = [np.zeros((1, pages, KV, PAGE, HEAD), np_type), np.zeros((1, pages, KV, HEAD, PAGE), np_type), np.zeros((1, pages, KV), np.float32), np.zeros((1, pages, KV), np.float32)]
        self.cache = [self.dev.view(x, dt) for x, dt in zip(self.host, (code, code, E.F32, E.F32))]
        i32 = lambda x: self.dev.view(np.asarray(x, np.int32), E.I32)  # noqa: E731
        self.tables = [i32(np.full((slots, width), -1)) for _ in range(2)]
        self.lengths = [i32(np.zeros(slots)) for _ in range(2)]
        self.moves, self.counts = i32(np.full((slots, 2), -1)), i32([0, 0])
        self.parents, self.new, self.ends = i32(np.arange(slots)), i32(np.zeros(slots)), i32(np.zeros(slots + 1))

    def give(self, view, array):
        self.ep.copy_from_host(view.data, np.ascontiguousarray(array))

    def take(self, view, dtype=None):
        return self.ep.download(E.DeviceBuffer(view.data, 0), view.shape, dtype or E._NP[view.dtype])

    def buffers(self, rows):
        make = lambda shape: self.dev.view(np.zeros(shape, np.float16), DTYPE)  # noqa: E731
        return {"x": make((rows, HIDDEN)), "packed": make((rows, PACKED)), "turned": make((rows, PACKED)), "y": make((rows, WIDE)), "out": make((rows, HIDDEN)),
                "positions": self.dev.view(np.zeros(rows, np.int64), E.I64)}

    def run(self, b, turn):
        """One step over rows whose buffers are `b`; tables[turn] to tables[1 - turn]."""
        flat = [E.TensorView(v.data, v.dtype, v.shape[1:]) for v in self.cache]
        self.step.execute([self.tables[turn], self.lengths[turn], self.parents, self.new] + self.cache, [self.tables[1 - turn], self.lengths[1 - turn], self.moves, self.counts] + self.cache)
        call = flat + [self.ends, self.lengths[1 - turn], self.tables[1 - turn]]
        self.qkv.execute([b["x"], *self.w[0]], [b["packed"]])
        self.rotary.execute([b["packed"], b["positions"]], [b["turned"]])
        self.append.execute([b["turned"], E.TensorView.absent()] + call, flat)
        self.attend.execute([b["turned"]] + call, [b["y"]])
        self.o.execute([b["y"], *self.w[1]], [b["out"]])

    def read(self, b, turn):
        self.ep.sync()
        got = {name: self.take(b[name]).copy() for name in ("packed", "turned", "y", "out")}
        got.update(cache=[self.take(v).copy() for v in self.cache], table=self.take(self.tables[1 - turn]), lengths=self.take(self.lengths[1 - turn]), moves=self.take(self.moves), counts=self.take(self.counts))
        return got

    def free(self):
        self.dev.free()
        for k in (self.qkv, self.o, self.rotary, self.append, self.attend, self.step):
            k.release()


def advance(layer, rng, turn, parents, new):
    """The inputs of a step: fresh activations, positions behind what each slot has."""
    lengths = layer.take(layer.lengths[turn])
    past = np.where(np.asarray(parents) >= 0, lengths[np.asarray(parents)], 0)
    new = np.where(np.asarray(parents) >= 0, new, 0)
    b = layer.buffers(int(new.sum()))
    layer.give(layer.parents, np.asarray(parents, np.int32))
    layer.give(layer.new, new.astype(np.int32))
    layer.give(layer.ends, np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    layer.give(b["x"], rng.standard_normal((int(new.sum()), HIDDEN)).astype(np.float16))
    layer.give(b["positions"], np.concatenate([p + np.arange(n) for p, n in zip(past, new)]).astype(np.int64))
    return b, past, new


def check_step(layer, before, got, past, new, parents, table, lengths, counts_grow):
    want = pages_step(table, lengths, parents, counts_grow, PAGE, layer.pages)
    for name, w in zip(("table", "lengths", "moves", "counts"), want):
        assert np.array_equal(got[name], w), name
    # the cache after the copies, then after the append
    cache = Cache.__new__(Cache)
    cache.new, cache.past, cache.code, cache.kv_heads, cache.head, cache.page = new.tolist(), past.tolist(), layer.code, KV, HEAD, PAGE
    state = [x[0].copy() for x in before]
    for source, to in want[2]:
        if to >= 0:
            for x in state:
                x[to] = x[source]
    cache.k, cache.v, cache.ks, cache.vs = state
    cache.table, cache.ends = want[0], np.concatenate([[0], np.cumsum(new)])
    turned = got["turned"].astype(np.float32)
    append32(cache, turned[:, WIDE:WIDE + KV * HEAD].reshape(-1, KV, HEAD), turned[:, WIDE + KV * HEAD:].reshape(-1, KV, HEAD))
    assert same_values(got["cache"][0][0], cache.k, layer.code) and same_values(got["cache"][1][0], cache.v, layer.code)
    assert np.array_equal(got["cache"][2][0], cache.ks) and np.array_equal(got["cache"][3][0], cache.vs)
    y, slack = attention64(cache, turned[:, :WIDE].astype(np.float64).reshape(-1, HEADS, HEAD), HEADS)
    error = np.abs(as64(got["y"], DTYPE).reshape(y.shape) - y)
    assert (error <= EPS[DTYPE] / 2 * np.abs(y) * (1 + 2.0 ** -8) + slack + 2.0 ** -24).all()


def check_rotary(got, positions):
    d = HEAD
    f = 10000.0 ** (-np.arange(0, d, 2) / d)
    wavelength = 2 * np.pi / f
    smooth = np.clip((8192 / wavelength - 1) / 3, 0, 1)
    f = (1 - smooth) * f / 8 + smooth * f
    c, s = np.cos(positions[:, None] * f)[:, None], np.sin(positions[:, None] * f)[:, None]
    x = got["packed"].astype(np.float64).reshape(len(positions), -1, d)
    want = x.copy()
    a, b = x[:, :HEADS + KV, :d // 2], x[:, :HEADS + KV, d // 2:]
    want[:, :HEADS + KV] = np.concatenate([a * c - b * s, b * c + a * s], -1)
    size = np.abs(x) + np.abs(np.roll(x, d // 2, -1))
    assert (np.abs(got["turned"].astype(np.float64).reshape(want.shape) - want) <= EPS[DTYPE] / 2 * np.abs(want) + 2.0 ** -20 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
def test_prompts_then_beams(ep, code):
    """Prompts of four sequences, then steps in which they continue one another, end, and take one or several tokens: each node against its definition over what the one before it wrote."""
    rng = np.random.default_rng(1)
    layer = Layer(ep, code, 4, 12, 60, 2)
    try:
        turn = 0
        steps = [([0, 1, 2, 3], [70, 5, 33, 16]), ([0, 0, 2, 3], [1, 1, 1, 1]), ([1, 0, 1, 3], [1, 1, 1, 1]), ([0, -1, 2, 2], [1, 1, 3, 1]), ([3, 3, 3, -1], [1, 1, 1, 1]), ([0, 1, 2, 3], [1, 1, 1, 40])]
        for parents, new in steps:
            ep.sync()
            table, lengths = layer.take(layer.tables[turn]), layer.take(layer.lengths[turn])
            before = [layer.take(v) for v in layer.cache]
            b, past, new = advance(layer, rng, turn, parents, np.asarray(new))
            layer.run(b, turn)
            got = layer.read(b, turn)
            check_rotary(got, layer.take(b["positions"]))
            check_step(layer, before, got, past, new, np.asarray(parents), table, lengths, new)
            # what the next step goes on from: the lengths with this step's tokens
            turn = 1 - turn
            layer.give(layer.lengths[turn], (past + new).astype(np.int32))
    finally:
        layer.free()


def filled(ep, code, seed, slots=3):
    """A layer with three sequences and the buffers of a step that forks one. The step has run once: a second run finds its own token in the page that it copies, and that
    page's scale grown for it, so that the runs from the second on leave the same bits and the first may not."""
    rng = np.random.default_rng(seed)
    layer = Layer(ep, code, slots, 40, 200, seed)
    b, past, new = advance(layer, rng, 0, list(range(slots)), np.asarray([500, 30, 77][:slots]))
    layer.run(b, 0)
    ep.sync()
    layer.give(layer.lengths[1], (past + new).astype(np.int32))
    b, past, new = advance(layer, rng, 1, [0, 0, 2][:slots], np.ones(slots, int))
    layer.run(b, 1)
    return layer, b


@pytest.mark.parametrize("code", [E.I8, E.F8E4M3])
def test_recorded_step(ep, code):
    """A step as a graph, replayed with eager runs and other work between: the same bits each time."""
    layer, b = filled(ep, code, 3)
    try:
        layer.run(b, 1)
        want = layer.read(b, 1)
        ep.capture_begin()
        layer.run(b, 1)
        graph = ep.capture_end()
        for eager in (False, True, False, True):
            for name in ("packed", "turned", "y", "out"):
                layer.give(b[name], np.zeros(b[name].shape, np.float16))
            if eager:
                layer.run(b, 1)
            graph.replay()
            got = layer.read(b, 1)
            for name in want:
                pairs = zip(got[name], want[name]) if name == "cache" else [(got[name], want[name])]
                for g, w in pairs:
                    assert np.array_equal(np.ascontiguousarray(g).view(np.uint8), np.ascontiguousarray(w).view(np.uint8)), name
        graph.release()
    finally:
        layer.free()


def test_a_graph_goes_on_from_what_the_host_changes(ep):
    """Lengths, tables and activations are read where they are when a graph is replayed: other inputs in the same buffers give what an eager call gives."""
    layer, b = filled(ep, E.I8, 4)
    try:
        layer.run(b, 1)
        ep.capture_begin()
        layer.run(b, 1)
        graph = ep.capture_end()
        rng = np.random.default_rng(9)
        for lengths in ([500, 30, 77], [100, 0, 511], [1, 16, 33]):
            layer.give(layer.lengths[1], np.asarray(lengths, np.int32))
            layer.give(b["x"], rng.standard_normal(b["x"].shape).astype(np.float16))
            layer.give(b["positions"], np.asarray([lengths[0], lengths[0], lengths[2]], np.int64))
            state = [layer.take(v).copy() for v in layer.cache]
            graph.replay()
            got = layer.read(b, 1)
            for v, x in zip(layer.cache, state):
                layer.give(v, x)
            layer.run(b, 1)
            want = layer.read(b, 1)
            for name in ("y", "out", "table", "lengths", "counts"):
                assert np.array_equal(got[name], want[name]), name
        graph.release()
    finally:
        layer.free()


def test_two_providers_at_once(ep):
    """Each has a stream, nodes and a cache of its own; their steps run side by side."""
    other = E.RocmExecutionProvider(0)
    layers = [filled(ep, E.I8, 5), filled(other, E.F8E4M3, 6)]
    try:
        want = []
        for layer, b in layers:
            layer.run(b, 1)
            want.append(layer.read(b, 1))
        for _ in range(20):
            for layer, b in layers:
                layer.run(b, 1)
        for (layer, b), w in zip(layers, want):
            got = layer.read(b, 1)
            assert np.array_equal(got["out"], w["out"]) and np.array_equal(got["y"], w["y"])
    finally:
        for layer, _ in layers:
            layer.free()
        other.shutdown()


def test_workspaces(ep):
    """The caller's workspace of the size asked for serves a call; a smaller one is refused; a first call under capture needs one."""
    rng = np.random.default_rng(7)
    cache = Cache(rng, [1, 1], [3000, 40], E.I8, KV, HEAD, PAGE)
    dev = Device(ep)
    try:
        kernel = ep.get_kernel({"num_heads": HEADS, "kv_num_heads": KV, "head_size": HEAD}, op_type="CacheAttention")
        views = [dev.view(synth.to_dtype(rng.standard_normal((2, WIDE)).astype(np.float32), DTYPE), DTYPE)] + cache.views(dev)
        y, read = dev.output((2, WIDE), DTYPE)
        need, align = kernel.workspace_requirement([(v.shape, v.dtype) for v in views])
        assert need > 0 and align == 256
        ep.capture_begin()
        with pytest.raises(E.EpError, match="needs a workspace"):
            kernel.execute(views, [y])
        ep.capture_end().release()
        ws = ep.allocate(need)
        with pytest.raises(E.EpError, match="smaller than the required"):
            kernel.execute(views, [y], workspace=E.DeviceBuffer(ws.ptr, need - 1))
        kernel.execute(views, [y], workspace=ws)
        ep.sync()
        first = read().copy()
        kernel.execute(views, [y])
        ep.sync()
        assert np.array_equal(first, read())
        kernel.release()
        ep.deallocate(ws)
    finally:
        dev.free()
