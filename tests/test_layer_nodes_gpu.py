"""The operators as a decoder layer uses them together: norm -> 8-bit codes -> product, norm -> experts -> norm, beside a MatMulNBits node, eagerly and recorded."""
import numpy as np
import pytest

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

from .node_helpers import EPS, Device, Experts, as64, gated_norm64, moe64

pytestmark = pytest.mark.gpu

H, N, EXPERTS, INTER, BLOCK = 256, 384, 8, 128, 32


class Layer:
    def __init__(self, ep, rows, dtype, seed):
        rng = np.random.default_rng(seed)
        self.ep, self.rows, self.dtype, self.dev = ep, rows, dtype, Device(ep)
        make = lambda *s, mean=0.0, sd=1.0: synth.to_dtype((rng.standard_normal(s) * sd + mean).astype(np.float32), dtype)  # noqa: E731
        self.host = {"residual": make(rows, H), "attention": make(rows, H), "post": make(H, mean=1.0, sd=0.2), "pre": make(H, mean=1.0, sd=0.2), "gate": make(H, sd=0.5),
                     "logits": make(rows, EXPERTS)}
        self.b = rng.integers(-127, 128, (N, H)).astype(np.int8)
        self.sb = (rng.uniform(0.5, 1.5, N) / (73 * np.sqrt(H))).astype(np.float32)
        self.fc1, self.fc2 = Experts(rng, EXPERTS, 2 * INTER, H, BLOCK, dtype), Experts(rng, EXPERTS, H, INTER, BLOCK, dtype)
        self.nbits = synth.make_weights(N, H, BLOCK, seed, zero_points=False, scale_lo=0.01, scale_hi=0.02, scale_dtype=dtype)
        v = {name: self.dev.view(x, dtype) for name, x in self.host.items()}
        none = E.TensorView.absent()
        out = lambda shape, dt: self.dev.output(shape, dt)  # noqa: E731
        (z1, self.z1), (c, self.codes), (s, self.scale), (y8, self.y8) = out((rows, H), dtype), out((rows, H), E.I8), out((rows,), E.F32), out((rows, N), dtype)
        (n2, self.n2), (m, self.moe), (z2, self.z2), (n3, self.n3), (y4, self.y4) = out((rows, H), dtype), out((rows, H), dtype), out((rows, H), dtype), out((rows, H), dtype), out((rows, N), dtype)
        norm = ep.get_kernel({"epsilon": 1e-6}, op_type="GatedResidualNorm")
        product = ep.get_kernel({"K": H, "N": N}, op_type="MatMulInt8")
        moe = ep.get_kernel({"k": 2, "block_size": BLOCK, "swiglu_fusion": 1, "normalize_routing_weights": 1}, op_type="QMoE")
        plain = ep.get_kernel({"K": H, "N": N, "bits": 4, "block_size": BLOCK})
        plain.set_constant_inputs([False, True, True])
        self.kernels = [norm, product, moe, plain]
        f1, f2 = ([self.dev.view(f.b, E.U8), self.dev.view(f.scales, dtype)] for f in (self.fc1, self.fc2))
        w8 = [self.dev.view(self.b, E.I8), self.dev.view(self.sb, E.F32)]
        w4 = [self.dev.view(self.nbits[0], E.U8), self.dev.view(self.nbits[1], dtype)]
        self.calls = [
            lambda: norm.execute([v["residual"], v["attention"], v["post"], v["gate"], v["pre"]], [z1, c, s]),
            lambda: product.execute([c, *w8, s], [y8]),
            lambda: norm.execute([z1, none, none, none, v["pre"]], [none, n2]),
            lambda: moe.execute([n2, v["logits"], *f1, none, *f2], [m]),
            lambda: norm.execute([z1, m, v["post"], none, v["pre"]], [z2, n3]),
            lambda: plain.execute([n3, *w4], [y4]),
        ]

    def run(self):
        for call in self.calls:
            call()

    def read(self):
        self.ep.sync()
        return {name: getattr(self, name)().copy() for name in ("z1", "codes", "scale", "y8", "n2", "moe", "z2", "n3", "y4")}

    def free(self):
        self.dev.free()
        for k in self.kernels:
            k.release()


def close(got, want, dtype, slack=2.0 ** -12):
    size = np.abs(want) + np.abs(want).max(-1, keepdims=True) * slack
    assert (np.abs(as64(got, dtype) - want) <= EPS[dtype] / 2 * np.abs(want) + 2.0 ** -10 * size).all()


@pytest.mark.parametrize("dtype", [E.F16, E.BF16])
@pytest.mark.parametrize("rows", [1, 3, 24, 150])
def test_layer(ep, rows, dtype):
    """Each node against its definition over what the node before it wrote."""
    layer = Layer(ep, rows, dtype, rows)
    try:
        layer.run()
        got = layer.read()
        h = {name: as64(x, dtype) for name, x in layer.host.items()}
        options = dict(epsilon=1e-6, residual_scale=1.0, block_scale=1.0, layer=False)
        z1, n1, _ = gated_norm64(h["residual"], h["attention"], h["post"], h["gate"], h["pre"], None, None, **options)
        close(got["z1"], z1, dtype)
        scale = got["scale"].astype(np.float64)[:, None]
        assert (np.abs(got["codes"] * scale - n1) <= 0.5 * scale * (1 + 2 ** -12) + 2.0 ** -16 * np.abs(n1).max(-1, keepdims=True)).all()
        close(got["y8"], (got["codes"].astype(np.int64) @ layer.b.astype(np.int64).T) * scale * layer.sb.astype(np.float64), dtype)
        _, n2, _ = gated_norm64(as64(got["z1"], dtype), None, None, None, h["pre"], None, None, **options)
        close(got["n2"], n2, dtype)
        moe, noise = moe64(as64(got["n2"], dtype), h["logits"], layer.fc1, layer.fc2, None, k=2, normalize=True, fusion=1)
        err = np.linalg.norm(as64(got["moe"], dtype) - moe, axis=-1)
        assert (err <= (EPS[dtype] / 2 + 2.0 ** -13) * np.sqrt((moe ** 2 + noise).sum(-1))).all()
        z2, n3, _ = gated_norm64(as64(got["z1"], dtype), as64(got["moe"], dtype), h["post"], None, h["pre"], None, None, **options)
        close(got["z2"], z2, dtype)
        close(got["n3"], n3, dtype)
    finally:
        layer.free()


@pytest.mark.parametrize("rows", [1, 24, 150])
def test_recorded_layer(ep, rows):
    """The layer as a graph, replayed with eager runs between: the same bits each time."""
    layer = Layer(ep, rows, E.BF16, 50 + rows)
    try:
        layer.run()
        want = layer.read()
        ep.capture_begin()
        layer.run()
        graph = ep.capture_end()
        for eager in (False, True, False):
            if eager:
                layer.run()
            graph.replay()
            got = layer.read()
            for name in want:
                assert np.array_equal(got[name].view(np.uint8), want[name].view(np.uint8)), name
        graph.release()
    finally:
        layer.free()
