"""Operators around a decoder layer's quantized products, as cases of one timed pass each, in their plain form and as calls of this provider.

The kinds:
  moe    `QMoE`: a mixture-of-experts layer over 4-bit expert weights, from router logits to the weighted sum of the experts
  int8   `MatMulInt8`: a product in 8-bit integers, activations quantized per token in the call, weights per channel
  norm   `GatedResidualNorm`: the norm behind a block, its gate, the scaled residual stream, and the norm before the next block
  block  norm and int8 together, as a layer uses them: the norm hands its 8-bit codes and token scales to the product

`prepare` makes what a session holds: weights and inputs on the GPU, output buffers, and, for this provider, one kernel object per node.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

_provider = None


def _ep():
    """The provider's module and one provider per process and GPU, as a session has it."""
    global _provider
    from onnx_genai_amd import ep as E
    if _provider is None:
        _provider = E.RocmExecutionProvider(0)
    return E, _provider


def _moe(name, rows, dtype, experts, k, hidden, inter, block, *, fusion=1, zero_points=False, bias=False, clamped=False, normalize=True, padded=0):
    """fusion 1: gate and up rows of fc1 alternate, 2: all gate rows, then all up rows. clamped: sigmoid slope 1.702, up + 1, values clamped at 7.
    padded: rows at the end that belong to no sequence; their logits are all -inf."""
    return {"name": name, "kind": "moe", "rows": rows, "dtype": dtype, "experts": experts, "k": k, "hidden": hidden, "inter": inter, "block": block, "fusion": fusion,
            "zero_points": zero_points, "bias": bias, "clamped": clamped, "normalize": normalize, "padded": padded}


def _int8(name, rows, dtype, k, n, *, bias=False):
    return {"name": name, "kind": "int8", "rows": rows, "dtype": dtype, "k": k, "n": n, "bias": bias}


def _norm(name, rows, dtype, hidden, *, layer=False, post=True, gates=1, residual_scale=1.0):
    """layer: layer norm instead of RMS norm. post: a norm behind the block too. gates: rows of the gate, each for rows / gates tokens; 0 for none."""
    return {"name": name, "kind": "norm", "rows": rows, "dtype": dtype, "hidden": hidden, "layer": layer, "post": post, "gates": gates, "residual_scale": residual_scale}


def _block(name, rows, dtype, hidden, n):
    return {"name": name, "kind": "block", "rows": rows, "dtype": dtype, "hidden": hidden, "n": n, "layer": False, "post": True, "gates": 1, "residual_scale": 1.0}


def listed():
    return [
        # one user's next token through a layer of many narrow experts: the smallest call, where latency counts
        _moe("moe_token", 1, "bf16", 64, 8, 2048, 1024, 32),
        # three users' tokens through a few wide experts (the MLP of an 8B model, eight times), with zero points
        _moe("moe_wide_3", 3, "f16", 8, 2, 4096, 14336, 32, fusion=2, zero_points=True),
        # a batch of 48 sequences: nearly every expert is read, each for a few tokens
        _moe("moe_batch_48", 48, "bf16", 64, 8, 2048, 1024, 64),
        # a ragged prompt in a padded batch, sizes that are no multiple of 128, biases and clamped activation
        _moe("moe_prompt_777", 777, "f16", 16, 4, 2880, 2880, 32, bias=True, clamped=True, padded=9),
        # a long prompt through many narrow experts
        _moe("moe_prompt_4096", 4096, "bf16", 64, 8, 2048, 1024, 128),
        # one token through the qkv projection of an 8B model
        _int8("int8_token", 1, "bf16", 4096, 6144),
        # a ragged prompt through the down projection of a 7B model, with a bias: a long sum, few output tiles
        _int8("int8_prompt_500", 500, "bf16", 18944, 3584, bias=True),
        # a long prompt through the gate projection of an 8B model: the largest product
        _int8("int8_prompt_8192", 8192, "bf16", 4096, 14336),
        # a batch of 24 sequences between attention and MLP of a 7B model: norm, codes, gate projection
        _block("block_24", 24, "f16", 3584, 18944),
        # one token's norms between two blocks of a 7B model
        _norm("norm_token", 1, "bf16", 3584),
        # three images' or clips' tokens, each with a gate row of its own, layer norm, a width that no vector load divides
        _norm("norm_odd_333", 333, "f16", 2881, layer=True, post=False, gates=3, residual_scale=0.7071),
        # a long prompt's norms at an 8B model's width
        _norm("norm_prompt_8192", 8192, "bf16", 4096),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    """A case of the ranges around the listed ones: rows and widths over their whole range, odd ones among them, each option on and off."""
    kind = rng.choice(["moe", "moe", "int8", "norm", "block"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "moe":
        while True:
            hidden, inter = _log_int(rng, 256, 4096), _log_int(rng, 256, 14336)
            if rng.random() < 0.75:
                hidden, inter = -(-hidden // 32) * 32, -(-inter // 32) * 32
            experts = rng.choice([4, 8, 16, 32, 64, 128])
            k, rows = rng.randint(1, min(8, experts)), _log_int(rng, 1, 4096)
            if experts * hidden * inter <= 8 * 4096 * 14336 and rows * k * hidden * inter <= 4096 * 8 * 2048 * 1024:
                break
        c = _moe("", rows, dtype, experts, k, hidden, inter, rng.choice([32, 64, 128]), fusion=rng.choice([1, 2]), zero_points=rng.random() < 0.4,
                 bias=rng.random() < 0.4, clamped=rng.random() < 0.3, normalize=rng.random() < 0.7, padded=rng.randint(0, rows // 8))
    elif kind == "norm":
        while True:
            rows, hidden = _log_int(rng, 1, 8192), _log_int(rng, 64, 16384)
            if rng.random() < 0.6:
                hidden = -(-hidden // 8) * 8
            if rows * hidden <= 8192 * 4096:
                break
        dtype = rng.choice(["f16", "bf16", "f32"])
        gates = rng.choice([0, 1, 1, rng.choice([g for g in range(1, min(rows, 64) + 1) if rows % g == 0])])
        c = _norm("", rows, dtype, hidden, layer=rng.random() < 0.3, post=rng.random() < 0.5, gates=gates, residual_scale=rng.choice([1.0, 0.5, 1.25]))
    else:
        while True:
            rows, k, n = _log_int(rng, 1, 8192), _log_int(rng, 128, 18944), _log_int(rng, 64, 28672)
            if rng.random() < 0.75:
                k, n = -(-k // 64) * 64, -(-n // 16) * 16
            if rows * k * n <= 8192 * 4096 * 14336 and k * n <= 8192 * 28672 and rows * n <= 8192 * 14336 and rows * k <= 8192 * 14336:
                break
        c = _int8("", rows, rng.choice([dtype, dtype, "f32"]), k, n, bias=rng.random() < 0.4) if kind == "int8" else _block("", rows, dtype, k, n)
    del c["name"]
    return c


def _nibbles(g, experts, n, k, case, bias):
    """One projection of all experts in the ONNX layout: packed weights, scales, zero points and bias, from the generator alone."""
    block = case["block"]
    kb = -(-k // block)
    count = experts * n * kb * block // 2
    b = torch.randint(-2**63, 2**63 - 1, (-(-count // 8),), dtype=torch.int64, device="cuda", generator=g).view(torch.uint8)[:count].view(experts, n, kb, block // 2)
    # rows of unit gain: q - zp is about 6.5 with random zero points, 4.6 with the default
    spread = 6.5 if case["zero_points"] else 4.6
    scales = ((torch.rand((experts, n, kb), device="cuda", generator=g) + 0.5) / (spread * math.sqrt(k))).to(TORCH[case["dtype"]])
    zp = torch.randint(0, 256, (experts, n, -(-kb // 2)), dtype=torch.uint8, device="cuda", generator=g) if case["zero_points"] else None
    return b, scales, zp, (torch.randn((experts, n), device="cuda", generator=g) * 0.3).to(TORCH[case["dtype"]]) if bias else None


def _prepare_moe(case, g, randn, s):
    m, e, h, i = case["rows"], case["experts"], case["hidden"], case["inter"]
    dt = TORCH[case["dtype"]]
    s["x"] = randn(m, h).to(dt)
    s["logits"] = (randn(m, e) * 1.5).to(dt)
    if case["padded"]:
        s["logits"][m - case["padded"]:] = -math.inf
    s["fc1"] = _nibbles(g, e, 2 * i, h, case, case["bias"])
    s["fc2"] = _nibbles(g, e, h, i, case, case["bias"])
    s["y"] = torch.empty((m, h), dtype=dt, device="cuda")


def _prepare_int8(case, g, randn, s):
    m, n = case["rows"], case["n"]
    k = case["hidden"] if case["kind"] == "block" else case["k"]
    if case["kind"] == "int8":
        # activations with a few strong channels, as a decoder's are
        strong = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 8.0, 1.0)
        s["a"] = (randn(m, k) * strong).to(TORCH[case["dtype"]])
    s["b"] = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
    s["b_scale"] = (torch.rand(n, device="cuda", generator=g) + 0.5) / (73.3 * math.sqrt(k))
    s["bias"] = randn(n).to(TORCH[case["dtype"]]) if case.get("bias") else None
    s["out"] = torch.empty((m, n), dtype=TORCH[case["dtype"]], device="cuda")


def _prepare_norm(case, g, randn, s):
    m, h, dt = case["rows"], case["hidden"], TORCH[case["dtype"]]
    around_one = lambda *shape: (torch.rand(shape, device="cuda", generator=g) * 0.5 + 0.75).to(dt)  # noqa: E731
    s["residual"], s["block"] = (randn(m, h) * 3).to(dt), randn(m, h).to(dt)
    s["post_gamma"] = around_one(h) if case["post"] else None
    s["gate"] = (randn(case["gates"], h) * 0.5).to(dt) if case["gates"] else None
    s["pre_gamma"] = around_one(h)
    s["pre_beta"] = (randn(h) * 0.1).to(dt) if case["layer"] else None
    s["z"] = torch.empty((m, h), dtype=dt, device="cuda")
    if case["kind"] == "block":
        s["codes"], s["code_scale"] = torch.empty((m, h), dtype=torch.int8, device="cuda"), torch.empty(m, dtype=torch.float32, device="cuda")
    else:
        s["n"] = torch.empty((m, h), dtype=dt, device="cuda")


EPSILON = 1e-6


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["kind"] == "moe":
        _prepare_moe(case, g, randn, s)
    if case["kind"] in ("norm", "block"):
        _prepare_norm(case, g, randn, s)
    if case["kind"] in ("int8", "block"):
        _prepare_int8(case, g, randn, s)
    if own:
        s["nodes"] = _nodes(case, s)
    torch.cuda.synchronize()
    return s


def run(s):
    case = s["case"]
    if own:
        for node in s["nodes"]:
            node(s)
    elif case["kind"] == "moe":
        s["y"] = _plain_moe(s, case)
    elif case["kind"] == "int8":
        s["out"] = _plain_product(*_plain_codes(s["a"].float()), s).to(s["a"].dtype)
    elif case["kind"] == "norm":
        z, n = _plain_norm(s, case)
        s["z"], s["n"] = z.to(s["block"].dtype), n.to(s["block"].dtype)
    else:
        z, n = _plain_norm(s, case)
        s["z"], s["out"] = z.to(s["block"].dtype), _plain_product(*_plain_codes(n), s).to(s["block"].dtype)
    if case["kind"] == "moe":
        return s["y"]
    return {"z": s["z"], "n": s["n"]} if case["kind"] == "norm" else {"z": s["z"], "y": s["out"]} if case["kind"] == "block" else s["out"]


# ---- the provider's calls ------------------------------------------------------------------------------------------


def _nodes(case, s):
    """The pass as calls: each node is a kernel object with its constant tensors' views, as a session keeps it."""
    E, ep = _ep()
    code = {torch.float32: E.F32, torch.float16: E.F16, torch.bfloat16: E.BF16, torch.uint8: E.U8, torch.int8: E.I8}
    view = lambda t: E.TensorView(t.data_ptr(), code[t.dtype], tuple(t.shape)) if t is not None else E.TensorView.absent()  # noqa: E731

    def moe():
        attrs = {"k": case["k"], "block_size": case["block"], "swiglu_fusion": case["fusion"], "normalize_routing_weights": int(case["normalize"])}
        if case["clamped"]:
            attrs.update(activation_alpha=1.702, activation_beta=1.0, swiglu_limit=7.0)
        (b1, s1, z1, c1), (b2, s2, z2, c2) = s["fc1"], s["fc2"]
        none = E.TensorView.absent()
        # input, router_probs, fc1 (weights, scales, bias), fc2 (the same), fc3 (absent: gate and up are both in fc1), zero points of fc1 and fc2
        rest = [view(b1), view(s1), view(c1), view(b2), view(s2), view(c2), none, none, none, view(z1), view(z2)]
        kernel = ep.get_kernel(attrs, op_type="QMoE")
        kernel.set_constant_inputs([False, False] + [True] * len(rest))
        return lambda s: kernel.execute([view(s["x"]), view(s["logits"])] + rest, [view(s["y"])])

    def product():
        k, n = s["b"].shape[1], s["b"].shape[0]
        weights, bias = [view(s["b"]), view(s["b_scale"])], view(s["bias"])
        kernel = ep.get_kernel({"K": k, "N": n}, op_type="MatMulInt8")
        kernel.set_constant_inputs([False, True, True, False, True])
        if case["kind"] == "block":        # the codes and scales that the norm wrote
            return lambda s: kernel.execute([view(s["codes"])] + weights + [view(s["code_scale"]), bias], [view(s["out"])])
        return lambda s: kernel.execute([view(s["a"])] + weights + [E.TensorView.absent(), bias], [view(s["out"])])

    def norm():
        rest = [view(s["post_gamma"]), view(s["gate"]), view(s["pre_gamma"]), view(s["pre_beta"])]
        kernel = ep.get_kernel({"epsilon": EPSILON, "layer_norm": int(case["layer"]), "residual_scale": case["residual_scale"]}, op_type="GatedResidualNorm")
        outputs = (lambda s: [view(s["z"]), view(s["codes"]), view(s["code_scale"])]) if case["kind"] == "block" else (lambda s: [view(s["z"]), view(s["n"])])
        return lambda s: kernel.execute([view(s["residual"]), view(s["block"])] + rest, outputs(s))

    return {"moe": lambda: [moe()], "int8": lambda: [product()], "norm": lambda: [norm()], "block": lambda: [norm(), product()]}[case["kind"]]()


# ---- the plain forms, in 32 bits ---------------------------------------------------------------------------------------


def _dequantize(w, ids):
    """(q - zero point) * scale of the experts `ids`: [experts, n, kb * block] in 32 bits."""
    b, scales, zp, _ = w
    b, scales = b[ids], scales[ids].float()
    q = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()                   # [.., n, kb, block], the even element in the low nibble
    if zp is None:
        q = q - 8.0
    else:
        z = zp[ids]
        z = torch.stack([z & 15, z >> 4], -1).flatten(-2)[..., :scales.shape[-1]].float()
        q = q - z[..., None]
    return (q * scales[..., None]).flatten(-2)


def _plain_activation(gate, up, case):
    alpha, beta = (1.702, 1.0) if case["clamped"] else (1.0, 0.0)
    if case["clamped"]:
        gate, up = torch.clamp(gate, max=7.0), torch.clamp(up, -7.0, 7.0)
    return gate / (1.0 + torch.exp(-alpha * gate)) * (up + beta)


def _plain_moe(s, case):
    h, i, k = case["hidden"], case["inter"], case["k"]
    x, logits = s["x"].float(), s["logits"].float()
    # the k largest logits, the lowest index first among equal ones; a row of -inf has no expert
    top, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    peak = logits.max(-1, keepdim=True).values
    live = peak > -math.inf
    e = torch.where(live, torch.exp(top - torch.where(live, peak, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True) if case["normalize"] else torch.exp(logits - torch.where(live, peak, 0.0)).sum(-1, keepdim=True)
    weights = torch.where(live, e / torch.where(live, total, 1.0), 0.0)
    rows = (lambda w: (w[..., 0::2, :], w[..., 1::2, :])) if case["fusion"] == 1 else (lambda w: (w[..., :i, :], w[..., i:, :]))
    halves = lambda c, e: rows(c[e].float()[..., None]) if c is not None else (0.0, 0.0)  # noqa: E731
    if ids.numel() <= 32:
        # few tokens: each (token, expert) pair with its own copy of the expert's weights
        pair = ids.flatten()
        xt = x.repeat_interleave(k, 0)[..., None]
        (wg, wu), (cg, cu) = rows(_dequantize(s["fc1"], pair)[..., :h]), halves(s["fc1"][3], pair)
        act = _plain_activation(wg @ xt + cg, wu @ xt + cu, case)
        y = (_dequantize(s["fc2"], pair)[..., :i] @ act)[..., 0]
        if s["fc2"][3] is not None:
            y = y + s["fc2"][3][pair].float()
        return (y.view(-1, k, h) * weights[..., None]).sum(1).to(s["x"].dtype)
    # many tokens: one expert after the other over the tokens that chose it
    y = torch.zeros_like(x)
    for expert in range(case["experts"]):
        token, slot = torch.nonzero((ids == expert) & (weights > 0), as_tuple=True)
        if not token.numel():
            continue
        (wg, wu), (cg, cu) = rows(_dequantize(s["fc1"], expert)[..., :h]), halves(s["fc1"][3], expert)
        xt = x[token].T
        act = _plain_activation(wg @ xt + cg, wu @ xt + cu, case)
        out = act.T @ _dequantize(s["fc2"], expert)[..., :i].T
        if s["fc2"][3] is not None:
            out = out + s["fc2"][3][expert].float()
        y.index_add_(0, token, out * weights[token, slot, None])                # a token is there once for each expert
    return y.to(s["x"].dtype)


def _plain_codes(a):
    """Codes in -127 .. 127 (held as 32-bit floats) and the scale of each token; a row of zeros has scale 0."""
    scale = a.abs().amax(-1, keepdim=True) / 127.0
    return torch.where(scale > 0, torch.round(a / torch.where(scale > 0, scale, 1.0)), 0.0), scale


def _plain_product(codes, scale, s):
    y = (codes @ s["b"].float().T) * scale * s["b_scale"]
    return y if s["bias"] is None else y + s["bias"].float()


def _plain_unit(x, case):
    if case["layer"]:
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON)


def _plain_norm(s, case):
    y, m = s["block"].float(), case["rows"]
    if s["post_gamma"] is not None:
        y = _plain_unit(y, case) * s["post_gamma"].float()
    if s["gate"] is not None:
        y = (y.view(case["gates"], m // case["gates"], -1) * s["gate"].float()[:, None]).view(m, -1)
    z = case["residual_scale"] * s["residual"].float() + y
    n = _plain_unit(z, case) * s["pre_gamma"].float()
    return z, n if s["pre_beta"] is None else n + s["pre_beta"].float()


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits: experts one by one over the pairs that chose them, integer sums in 64 bits, two-pass moments."""
    s = {"case": case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    if case["kind"] == "moe":
        _prepare_moe(case, g, randn, s)
        return _exact_moe(case, s)
    if case["kind"] in ("norm", "block"):
        _prepare_norm(case, g, randn, s)
        z, n = _exact_norm(case, s)
        if case["kind"] == "norm":
            return {"z": z, "n": n}
    _prepare_int8(case, g, randn, s)
    if case["kind"] == "int8":
        return _exact_product(s["a"].double(), s)
    return {"z": z, "y": _exact_product(n, s)}


def _exact_weights(w, expert, k):
    b, scales, zp, _ = w
    byte = b[expert].to(torch.int64).flatten(1)
    column = torch.arange(k, device="cuda")
    q = (byte[:, column // 2] >> (4 * (column % 2))) & 15
    block = column // (2 * b.shape[-1])
    z = 8 if zp is None else (zp[expert].to(torch.int64)[:, block // 2] >> (4 * (block % 2))) & 15
    return (q - z).double() * scales[expert].double()[:, block]


def _exact_moe(case, s):
    h, i, k = case["hidden"], case["inter"], case["k"]
    x, logits = s["x"].double(), s["logits"].double()
    # rank of an expert in its row: how many are larger, or equal with a lower index
    index = torch.arange(case["experts"], device="cuda")
    rank = torch.stack([((logits > logits[:, e:e + 1]) | ((logits == logits[:, e:e + 1]) & (index < e))).sum(-1) for e in range(case["experts"])], -1)
    p = torch.nan_to_num(torch.softmax(logits, -1), nan=0.0)
    chosen = (rank < k) & (p > 0)
    if case["normalize"]:
        total = (p * chosen).sum(-1, keepdim=True)
        p = torch.where(total > 0, p / torch.where(total > 0, total, 1.0), 0.0)
    y = torch.zeros((case["rows"], h), dtype=torch.float64, device="cuda")
    row = torch.arange(i, device="cuda")
    gate_row, up_row = (2 * row, 2 * row + 1) if case["fusion"] == 1 else (row, row + i)
    for e in range(case["experts"]):
        t = chosen[:, e].nonzero()[:, 0]
        if not t.numel():
            continue
        f = x[t] @ _exact_weights(s["fc1"], e, h).T
        if s["fc1"][3] is not None:
            f = f + s["fc1"][3][e].double()
        gate, up = f[:, gate_row], f[:, up_row]
        if case["clamped"]:
            gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0)
            act = gate * torch.sigmoid(1.702 * gate) * (up + 1.0)
        else:
            act = gate * torch.sigmoid(gate) * up
        out = act @ _exact_weights(s["fc2"], e, i).T
        if s["fc2"][3] is not None:
            out = out + s["fc2"][3][e].double()
        y[t] += out * p[t, e][:, None]
    return y


def _exact_product(a, s):
    scale = a.abs().amax(-1, keepdim=True) / 127
    codes = torch.where(scale > 0, (a / torch.where(scale > 0, scale, 1.0)).round(), 0.0)
    y = (codes @ s["b"].double().T) * (scale * s["b_scale"].double())
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_norm(case, s):
    def unit(v):
        if case["layer"]:
            return (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + EPSILON)
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPSILON)

    f = s["block"].double()
    if s["post_gamma"] is not None:
        f = unit(f) * s["post_gamma"].double()
    if s["gate"] is not None:
        f = f * s["gate"].double().repeat_interleave(case["rows"] // case["gates"], 0)
    z = s["residual"].double() * case["residual_scale"] + f
    n = unit(z) * s["pre_gamma"].double()
    return z, n if s["pre_beta"] is None else n + s["pre_beta"].double()


def work(case):
    m, item = case["rows"], 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "moe":
        e, k, h, i, block = case["experts"], case["k"], case["hidden"], case["inter"], case["block"]
        tokens = m - case["padded"]
        active = e * (1.0 - (1.0 - k / e) ** tokens)                            # experts that some token chooses, on average

        def projection(n, depth):
            kb = -(-depth // block)
            return n * (kb * block // 2 + kb * item + (-(-kb // 2) if case["zero_points"] else 0) + (item if case["bias"] else 0))

        nbytes = active * (projection(2 * i, h) + projection(h, i)) + m * (2 * h + e) * item
        return {"bytes": int(nbytes), "flops": 6 * tokens * k * h * i}
    nbytes = flops = 0
    if case["kind"] in ("norm", "block"):
        h = case["hidden"]
        # block output and residual in, the new stream out, and the normalized rows, where they are an output
        nbytes += m * h * item * (4 if case["kind"] == "norm" else 3) + h * item * (1 + case["post"] + case["gates"] + case["layer"])
        flops += m * h * (16 if case["post"] else 10)
    if case["kind"] in ("int8", "block"):
        k = case["hidden"] if case["kind"] == "block" else case["k"]
        n = case["n"]
        nbytes += n * k + 4 * n + m * n * item + (m * k * item if case["kind"] == "int8" else 0)
        flops += 2 * m * n * k
    return {"bytes": nbytes, "flops": flops}
