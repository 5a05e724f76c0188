"""Operands and 64-bit references of the operators beside MatMulNBits."""
from __future__ import annotations

import numpy as np

from onnx_genai_amd import ep as E
from onnx_genai_amd import synth

EPS = {E.F32: 2.0 ** -23, E.F16: 2.0 ** -10, E.BF16: 2.0 ** -7}      # a rounding is off by at most half of it, relative to the value
GUARD = 64                                                             # elements behind an output that no call may touch


class Device:
    """Uploads that live as long as one test's call."""

    def __init__(self, ep):
        self.ep, self.bufs = ep, []

    def view(self, array, dtype, shape=None, offset=0):
        """offset: elements by which the tensor lies behind a 256-byte boundary."""
        if array is None:
            return E.TensorView.absent(dtype)
        array = np.ascontiguousarray(array)
        padded = np.zeros(array.size + offset, array.dtype)
        padded[offset:] = array.ravel()
        buf = self.ep.upload(padded)
        self.bufs.append(buf)
        return E.TensorView(buf.ptr, dtype, tuple(shape or array.shape), byte_offset=offset * array.itemsize, device_index=self.ep.device_index)

    def output(self, shape, dtype, offset=0):
        np_dtype = E._NP[dtype]
        n = int(np.prod(shape))
        fill = np.full(offset + n + GUARD, 0x5A, np.uint8).astype(np_dtype) if dtype != E.F32 else np.full(offset + n + GUARD, 1e30, np.float32)
        buf = self.ep.upload(fill)
        self.bufs.append(buf)
        view = E.TensorView(buf.ptr, dtype, tuple(shape), byte_offset=offset * fill.itemsize, device_index=self.ep.device_index)

        def read():
            got = self.ep.download(buf, fill.shape, np_dtype)
            assert np.array_equal(got[:offset], fill[:offset]) and np.array_equal(got[offset + n:], fill[offset + n:]), "written outside of the output"
            return got[offset:offset + n].reshape(shape)

        return view, read

    def free(self):
        for b in self.bufs:
            self.ep.deallocate(b)


def as64(x, dtype):
    return synth.to_f32(x, dtype).astype(np.float64)


# ---- GatedResidualNorm ------------------------------------------------------------------------------------------------------


def unit64(x, epsilon, layer):
    if layer:
        x = x - x.mean(-1, keepdims=True)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)


def gated_norm64(residual, block, post_gamma, gate, pre_gamma, pre_beta, post_beta, *, epsilon, residual_scale, block_scale, layer):
    """z, n and the magnitude of z's terms (what f32 rounding errors are relative to)."""
    z = residual_scale * residual
    size = np.abs(z)
    if block is not None:
        p = block
        if post_gamma is not None:
            p = unit64(p, epsilon, layer) * post_gamma
            if post_beta is not None:
                p = p + post_beta
        if gate is not None:
            g = gate.reshape(-1, gate.shape[-1])
            p = p * np.repeat(g, p.shape[0] // g.shape[0], 0)
        z = z + block_scale * p
        size = size + np.abs(block_scale * p)
    n = unit64(z, epsilon, layer)
    if pre_gamma is not None:
        n = n * pre_gamma
    if pre_beta is not None:
        n = n + pre_beta
    return z, n, size


# ---- MatMulInt8 -------------------------------------------------------------------------------------------------------------


def codes32(a):
    """Codes and scales of rows as the operator defines them, in f32 arithmetic (numpy's f32 division is correctly rounded)."""
    a = np.asarray(a, np.float32)
    scale = (np.abs(a).max(-1) / np.float32(127)).astype(np.float32)
    safe = np.where(scale > 0, scale, np.float32(1))
    return np.where(scale[:, None] > 0, np.rint((a / safe[:, None]).astype(np.float32)), 0).astype(np.int64), scale


# ---- QMoE -------------------------------------------------------------------------------------------------------------------


class Experts:
    """One projection of all experts: random nibbles, scales for rows of unit gain, in f64 as `w`."""

    def __init__(self, rng, experts, n, k, bs, dtype, *, zero_points=False, bias=False, scale_dtype=None, bias_dtype=None):
        self.scale_dtype = scale_dtype or dtype
        self.bias_dtype = bias_dtype or dtype
        kb = -(-k // bs)
        q = rng.integers(0, 16, (experts, n, kb, bs), dtype=np.uint8)
        self.b = synth.pack_nibbles(q)
        self.scales = synth.to_dtype((rng.uniform(0.5, 1.5, (experts, n, kb)) / (5.0 * np.sqrt(k))).astype(np.float32), self.scale_dtype)
        z = rng.integers(0, 16, (experts, n, kb), dtype=np.uint8) if zero_points else np.full((experts, n, kb), 8, np.uint8)
        self.zp = synth.pack_nibbles(z) if zero_points else None
        self.w = ((q.astype(np.float64) - z[..., None]) * as64(self.scales, self.scale_dtype)[..., None]).reshape(experts, n, kb * bs)[..., :k]
        self.bias = synth.to_dtype(rng.normal(0, 0.3, (experts, n)).astype(np.float32), self.bias_dtype) if bias else None
        self.bias64 = as64(self.bias, self.bias_dtype) if bias else np.zeros((experts, n))


def route64(logits, k, normalize):
    """Weights [rows, experts]: 0 where an expert is not chosen."""
    rows, experts = logits.shape
    w = np.zeros((rows, experts))
    for t in range(rows):
        if np.isnan(logits[t]).any() or np.isposinf(logits[t]).any():
            w[t] = np.nan
            continue
        if np.isneginf(logits[t]).all():
            continue
        p = np.exp(logits[t] - logits[t].max())
        order = np.argsort(-logits[t], kind="stable")[:k]
        order = order[p[order] > 0]
        w[t, order] = p[order] / (p[order].sum() if normalize else p.sum())
    return w


def moe64(x, logits, fc1, fc2, fc3, *, k, normalize, fusion, alpha=1.0, beta=0.0, limit=np.inf):
    """y, and the mean square of what independent errors of h, each of h's own size, do to y."""
    w = route64(logits, k, normalize)
    y = np.zeros((x.shape[0], fc2.w.shape[1]))
    noise = np.zeros_like(y)
    y[np.isnan(w).any(-1)] = np.nan
    for e in range(logits.shape[1]):
        t = np.nonzero(w[:, e] > 0)[0]
        f = x[t] @ fc1.w[e].T + fc1.bias64[e]
        if fusion == 0:
            gate, up = f, x[t] @ fc3.w[e].T + fc3.bias64[e]
        elif fusion == 1:
            gate, up = f[:, 0::2], f[:, 1::2]
        else:
            gate, up = f[:, :f.shape[1] // 2], f[:, f.shape[1] // 2:]
        gate, up = np.minimum(gate, limit), np.clip(up, -limit, limit)
        h = gate / (1 + np.exp(-alpha * gate)) * (up + beta)
        y[t] += w[t, e, None] * (h @ fc2.w[e].T + fc2.bias64[e])
        noise[t] += w[t, e, None] ** 2 * (h ** 2 @ (fc2.w[e] ** 2).T)
    return y, noise
