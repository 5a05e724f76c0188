"""Operators around a paged 8-bit cache of keys and values, as cases of one timed pass each, in their plain form and as calls of this provider.

The kinds:
  rotary  `RotaryEmbedding`: queries and keys of packed rows turned by their positions; values in the same rows pass through
  append  `CacheAppend`: new tokens' keys and values into their pages, as 8-bit codes with a scale for each page and head
  attend  `CacheAttention`: queries against the pages of their sequences
  pages   `CachePages`: block tables of the next step (forked, freed and grown sequences, or a compacted pool) and the pages that move for it

A page holds `page` tokens of every head of one layer: codes of the keys [pages, heads, page, head], of the values [pages, heads, head, page], scales
[pages, heads]. `prepare` makes what a session holds: activations, caches and tables on the GPU, output buffers, and, for this provider, one kernel object per node.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}

_provider = None


def _ep():
    """The provider's module and one provider per process and GPU, as a session has it."""
    global _provider
    from onnx_genai_amd import ep as E
    if _provider is None:
        _provider = E.RocmExecutionProvider(0)
    return E, _provider


def _rotary(name, rows, dtype, heads, kv_heads, head, *, part=0, interleaved=False, theta=10000.0, scaling="none", factor=1.0, original=8192, start=0):
    """part: leading elements of a head that turn (0: all of them). start: position of the first row; the rows belong to one sequence."""
    return {"name": name, "kind": "rotary", "rows": rows, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head, "part": part, "interleaved": interleaved,
            "theta": theta, "scaling": scaling, "factor": factor, "original": original, "start": start}


def _append(name, sequences, rows, past, dtype, code, kv_heads, head, page):
    """rows: new tokens of all sequences, spread unevenly where there are more rows than sequences; past: most tokens that a sequence already has."""
    return {"name": name, "kind": "append", "sequences": sequences, "rows": rows, "past": past, "dtype": dtype, "code": code, "kv_heads": kv_heads, "head": head, "page": page}


def _attend(name, sequences, rows, past, dtype, code, heads, kv_heads, head, page, *, window=0, softcap=0.0, even=False):
    """As `append`; even: every sequence has `past` tokens. window: how many tokens a query sees, itself among them (0: all before it)."""
    return {"name": name, "kind": "attend", "sequences": sequences, "rows": rows, "past": past, "dtype": dtype, "code": code, "heads": heads, "kv_heads": kv_heads, "head": head,
            "page": page, "window": window, "softcap": softcap, "even": even}


def _pages(name, sequences, beams, past, layers, kv_heads, head, page, *, compact=False, pool=0):
    """sequences: slots of the table, `beams` of them to a prompt; past: most tokens of a sequence; pool: pages of a layer (0: what the sequences need and a quarter more)."""
    return {"name": name, "kind": "pages", "sequences": sequences, "beams": beams, "past": past, "layers": layers, "kv_heads": kv_heads, "head": head, "page": page,
            "compact": compact, "pool": pool}


def listed():
    return [
        # one user's next token in a 7B model: the smallest call, where latency counts
        _rotary("rotary_token", 1, "bf16", 28, 4, 128, theta=1e6, start=2900),
        # a ragged chunk far into a long text: pairs side by side, less than half of an odd head, frequencies stretched sixteen times
        _rotary("rotary_far_777", 777, "f16", 32, 32, 80, part=32, interleaved=True, scaling="yarn", factor=16.0, original=4096, start=1000003),
        # a long prompt of an 8B model with the scaling its long contexts use
        _rotary("rotary_prompt_8192", 8192, "bf16", 32, 8, 128, theta=5e5, scaling="llama3", factor=8.0),
        # the next token of each of 48 sequences of a 7B model: pages begun earlier, some of which need a larger scale
        _append("append_batch_48", 48, 48, 4000, "bf16", "int8", 4, 128, 64),
        # a long prompt of an 8B model: whole pages
        _append("append_prompt_8192", 1, 8192, 0, "bf16", "e4m3", 8, 128, 64),
        # one user's next token in a 7B model after a short text: latency
        _attend("attend_token", 1, 1, 1000, "bf16", "int8", 28, 4, 128, 64),
        # the next token of 64 sequences of all lengths in an 8B model, small pages
        _attend("attend_batch_64", 64, 64, 8192, "bf16", "e4m3", 32, 8, 128, 32),
        # one user's next token after a whole book: one row of work over a long axis
        _attend("attend_long_131072", 1, 1, 131071, "bf16", "int8", 32, 8, 128, 64, even=True),
        # chunks of three prompts of a 0.5B model behind what is cached of them, in a sliding window, with small pages
        _attend("attend_chunks_3", 3, 1111, 3000, "f16", "int8", 14, 2, 64, 16, window=1024),
        # a long prompt of an 8B model against itself: the largest products
        _attend("attend_prompt_8192", 1, 8192, 0, "bf16", "int8", 32, 8, 128, 64, even=True),
        # a step of beam search over eight prompts of a 7B model: beams continue one another, begun pages are copied
        _pages("fork_beams_32", 32, 4, 1500, 28, 4, 128, 64),
        # a pool of a 0.5B model that is half empty, packed into its front
        _pages("compact_1500", 48, 1, 1300, 24, 2, 64, 64, compact=True, pool=1500),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    """A case of the ranges around the listed ones: tokens and sequences over their whole range, each head layout, type and option."""
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "pages"])
    dtype, code = rng.choice(["f16", "bf16"]), rng.choice(["int8", "e4m3"])
    head, page = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8, 16])
    if kind == "rotary":
        while True:
            rows = _log_int(rng, 1, 16384)
            if rows * (heads + 2 * kv_heads) * head <= 8192 * 48 * 128:
                break
            heads, kv_heads = max(1, heads // 2), max(1, kv_heads // 2)
        scaling = rng.choice(["none", "linear", "llama3", "yarn"])
        c = _rotary("", rows, rng.choice([dtype, "f32"]), heads, kv_heads, head, part=rng.choice([0, 0, head // 2, 16, 26]), interleaved=rng.random() < 0.4,
                    theta=rng.choice([1e4, 5e5, 1e6]), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]), original=rng.choice([4096, 8192]),
                    start=_log_int(rng, 1, 2000000) - 1)
    elif kind == "append":
        while True:
            sequences, rows, past = _log_int(rng, 1, 128), _log_int(rng, 1, 16384), _log_int(rng, 1, 8192) - 1
            if rows * kv_heads * head <= 8192 * 8 * 128 and (sequences * past + rows) * kv_heads * head <= (1 << 28):
                break
        c = _append("", sequences, rows, past, dtype, code, kv_heads, head, page)
    elif kind == "attend":
        while True:
            sequences = _log_int(rng, 1, 128)
            # single tokens and a few of them (drafted ones) are as common as chunks of a prompt
            rows = sequences * rng.randint(1, 4) if rng.random() < 0.5 else _log_int(rng, 1, 8192)
            past = _log_int(rng, 1, 131072) - 1
            most = past + (rows if sequences == 1 else min(rows, 2 * rows // sequences + 1))
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8, 16])
            # (the plain form pads to the longest sequence: its scores and its 32-bit copy of the cache stay within the prompt's)
            padded = sequences * most
            if rows * most * heads * head <= 8192 * 4096 * 32 * 128 and padded * kv_heads * head <= (1 << 29) and sequences * min(rows, 2 * rows // sequences + 1) * most * heads <= (1 << 31):
                break
        c = _attend("", sequences, rows, past, dtype, code, heads, kv_heads, head, page, window=rng.choice([0, 0, 0, 1, 100, 1024, 4096]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                    even=rng.random() < 0.3)
    else:
        compact = rng.random() < 0.5
        while True:
            beams = 1 if compact else rng.choice([1, 2, 4, 8])
            sequences, past, layers = beams * _log_int(rng, 1, 128 // beams), _log_int(rng, 1, 4096), rng.choice([1, 2, 12, 24, 32])
            need = sequences * (-(-past // page) + 2)
            if need * page * kv_heads * head * layers <= (1 << 29):
                break
        c = _pages("", sequences, beams, past, layers, kv_heads, head, page, compact=compact, pool=need + _log_int(rng, 1, 2 * need) if compact else 0)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------------


def _spread(total, parts, g):
    """`total` dealt out to `parts` sequences: one each where the numbers agree, at random up to twice the mean otherwise. Some may get none."""
    if total == parts:
        return [1] * parts
    weight = (torch.rand(parts, generator=g) + 0.05).double()
    edge = torch.round(torch.cumsum(weight, 0) / weight.sum() * total).long().tolist()
    cut = [b - a for a, b in zip([0] + edge[:-1], edge)]
    most = 2 * total // parts + 1
    over = 0
    for i, n in enumerate(cut):                 # what is over the most goes to the next ones
        cut[i], over = min(most, n + over), max(0, n + over - most)
    for i in range(parts):
        more = min(over, most - cut[i])
        cut[i], over = cut[i] + more, over - more
    return cut


def _lengths(case, g):
    n, past = case["sequences"], case["past"]
    new = _spread(case["rows"], n, g)
    before = [past] * n if case.get("even") else torch.randint(0, past + 1, (n,), generator=g).tolist()
    return new, before


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(need, pool, g):
    """Pages at random places of the pool for sequences that need so many each; -1 behind them."""
    width, order = max(max(need), 1), torch.randperm(pool, generator=g).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return _int32(rows)


def _codes(shape, code, g):
    """Codes as normally distributed keys and values have them: the largest of a page at the type's end."""
    out = torch.empty(shape, dtype=TORCH[code], device="cuda")
    for part in out.split(max(1, (1 << 27) // max(1, out[0].numel()))):
        x = torch.randn(part.shape, device="cuda", generator=g)
        part.copy_((x * 32).round_().clamp_(-127, 127) if code == "int8" else (x * 112).clamp_(-448, 448))
    return out


def _cache(case, pool, g, s):
    h, d, b, code = case["kv_heads"], case["head"], case["page"], case["code"]
    s["k"], s["v"] = _codes((pool, h, b, d), code, g), _codes((pool, h, d, b), code, g)
    spread = 32.0 if code == "int8" else 112.0
    s["ks"], s["vs"] = ((torch.rand((pool, h), device="cuda", generator=g) + 0.5) / spread for _ in range(2))


def _inputs(case, seed):
    """What a pass reads, from the seed alone."""
    g, host = torch.Generator(device="cuda"), torch.Generator()
    g.manual_seed(seed)
    host.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["kind"] == "rotary":
        s["x"] = randn(case["rows"], (case["heads"] + 2 * case["kv_heads"]) * case["head"]).to(TORCH[case["dtype"]])
        s["positions"] = torch.arange(case["start"], case["start"] + case["rows"], device="cuda")
        s["y"] = torch.empty_like(s["x"])
        return s
    if case["kind"] == "pages":
        return _page_inputs(case, g, host, s)
    new, before = _lengths(case, host)
    need = [-(-(a + b) // case["page"]) for a, b in zip(new, before)]
    pool = case["sequences"] * (case["past"] // case["page"] + 2) + case["rows"] // case["page"] + 1
    _cache(case, pool, g, s)
    s["table"], s["past"] = _tables(need, pool, host), _int32(before)
    s["ends"] = _int32([0] + torch.tensor(new).cumsum(0).tolist())
    dt, rows, d = TORCH[case["dtype"]], case["rows"], case["head"]
    if case["kind"] == "append":
        # a few strong channels, as keys have them
        strong = torch.where(torch.rand(case["kv_heads"] * d, device="cuda", generator=g) < 0.02, 4.0, 1.0)
        s["new_k"], s["new_v"] = (randn(rows, case["kv_heads"] * d) * strong).to(dt), randn(rows, case["kv_heads"] * d).to(dt)
    else:
        # heads from even to sharp attention
        sharp = torch.rand(case["heads"], device="cuda", generator=g) * 3 + 0.3
        s["q"] = (randn(rows, case["heads"], d) * sharp[:, None]).to(dt).view(rows, -1)
        s["y"] = torch.empty_like(s["q"])
        s["longest"], s["most"] = max(new), max(a + b for a, b in zip(new, before))
    return s


def _page_inputs(case, g, host, s):
    n, beams, page, past, layers = case["sequences"], case["beams"], case["page"], case["past"], case["layers"]
    # the beams of a prompt share the pages that the prompt filled, and have a few of their own
    lengths, rows, at = [], [], 0
    total = case["pool"] or n * (past // page + 2) * 5 // 4
    order = torch.randperm(total, generator=host).tolist()
    width = past // page + 2
    for first in range(0, n, beams):
        length = int(torch.randint(max(1, past // 2), past + 1, (1,), generator=host))
        shared = length // page // 2 if beams > 1 else 0
        prompt = order[at:at + shared]
        at += shared
        for _ in range(beams):
            mine = -(-length // page) - shared
            rows.append((prompt + order[at:at + mine] + [-1] * width)[:width])
            at += mine
            lengths.append(length)
    s["table"], s["lengths"] = _int32(rows), _int32(lengths)
    if not case["compact"]:
        # the best beam continues twice as often as it stays, now and then a sequence has ended
        pick = torch.randint(0, beams, (n,), generator=host)
        pick = torch.minimum(pick, torch.randint(0, beams, (n,), generator=host))
        parents = (torch.arange(n) // beams * beams + pick).tolist()
        ended = (torch.rand(n, generator=host) < 0.05).tolist()
        s["parents"], s["new"] = _int32([-1 if e else p for p, e in zip(parents, ended)]), _int32([1] * n)
    h, d = case["kv_heads"], case["head"]
    s["pools"] = [torch.randint(-127, 128, (layers, total, h, page, d), dtype=torch.int8, device="cuda", generator=g),
                  torch.randint(-127, 128, (layers, total, h, d, page), dtype=torch.int8, device="cuda", generator=g),
                  torch.rand((layers, total, h), device="cuda", generator=g), torch.rand((layers, total, h), device="cuda", generator=g)]
    s["next"], s["next_lengths"] = torch.full_like(s["table"], -1), torch.zeros_like(s["lengths"])
    s["moves"] = torch.full((total // 2 if case["compact"] else n, 2), -1, dtype=torch.int32, device="cuda")
    s["counts"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary":
        s["frequencies"], s["factor"] = _frequencies(case)
        s["frequencies"] = torch.tensor(s["frequencies"], dtype=torch.float64, device="cuda")
    if own:
        s["node"] = _node(case, s)
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        s["node"]()
    else:
        {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "pages": _plain_pages}[s["case"]["kind"]](s, s["case"])
    return _outputs(s)


def _outputs(s):
    kind = s["case"]["kind"]
    if kind in ("rotary", "attend"):
        return s["y"]
    if kind == "append":
        return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    return {"table": s["next"], "lengths": s["next_lengths"], "moves": s["moves"], "counts": s["counts"], "pools": s["pools"]}


# ---- the provider's calls ------------------------------------------------------------------------------------------


def _node(case, s):
    """The pass as a call: a kernel object and the views of what it reads and writes, as a session keeps them."""
    E, ep = _ep()
    code = {torch.float32: E.F32, torch.float16: E.F16, torch.bfloat16: E.BF16, torch.int8: E.I8, torch.float8_e4m3fn: E.F8E4M3, torch.int32: E.I32, torch.int64: E.I64}
    view = lambda t: E.TensorView(t.data_ptr(), code[t.dtype], tuple(t.shape)) if t is not None else E.TensorView.absent()  # noqa: E731
    kind = case["kind"]
    if kind == "rotary":
        attrs = {"head_size": case["head"], "num_heads": case["heads"] + case["kv_heads"], "rotary_embedding_dim": case["part"], "interleaved": int(case["interleaved"]),
                 "rope_theta": case["theta"], "scaling": ["none", "linear", "llama3", "yarn"].index(case["scaling"]), "factor": case["factor"],
                 "original_max_position": case["original"]}
        op, inputs, outputs = "RotaryEmbedding", [s["x"], s["positions"]], [s["y"]]
    elif kind == "append":
        attrs = {"kv_num_heads": case["kv_heads"], "head_size": case["head"]}
        cache = [s["k"], s["v"], s["ks"], s["vs"]]
        op, inputs, outputs = "CacheAppend", [s["new_k"], s["new_v"]] + cache + [s["ends"], s["past"], s["table"]], cache
    elif kind == "attend":
        attrs = {"num_heads": case["heads"], "kv_num_heads": case["kv_heads"], "head_size": case["head"], "softcap": case["softcap"], "local_window_size": case["window"] or -1}
        op, inputs, outputs = "CacheAttention", [s["q"], s["k"], s["v"], s["ks"], s["vs"], s["ends"], s["past"], s["table"]], [s["y"]]
    else:
        attrs = {"page_size": case["page"], "compact": int(case["compact"])}
        op, inputs = "CachePages", [s["table"], s["lengths"], s.get("parents"), s.get("new")] + s["pools"]
        outputs = [s["next"], s["next_lengths"], s["moves"], s["counts"]] + s["pools"]
    kernel = ep.get_kernel(attrs, op_type=op)
    inputs, outputs = [view(t) for t in inputs], [view(t) for t in outputs]
    return lambda: kernel.execute(inputs, outputs)


# ---- the plain forms, in 32 bits ---------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each pair, and what cosine and sine are multiplied by."""
    part, theta, factor, original = case["part"] or case["head"], case["theta"], case["factor"], case["original"]
    f = [theta ** (-2.0 * i / part) for i in range(part // 2)]
    if case["scaling"] == "linear":
        return [x / factor for x in f], 1.0
    if case["scaling"] == "llama3":
        # turns within the first context: few are slowed down, many stay, between them a blend
        def blend(x):
            smooth = (original * x / (2 * math.pi) - 1.0) / (4.0 - 1.0)
            smooth = min(1.0, max(0.0, smooth))
            return (1 - smooth) * x / factor + smooth * x
        return [blend(x) for x in f], 1.0
    if case["scaling"] == "yarn":
        pair = lambda turns: part * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), part - 1)
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(part // 2)]
        return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _plain_rotary(s, case):
    rows, heads, d, part = case["rows"], case["heads"] + case["kv_heads"], case["head"], case["part"] or case["head"]
    x = s["x"].float().view(rows, -1, d)
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["factor"]).float()[:, None], (torch.sin(angle) * s["factor"]).float()[:, None]
    turned = x[:, :heads, :part]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :part // 2], turned[..., part // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([torch.cat([turned, x[:, :heads, part:]], -1), x[:, heads:]], 1)
    s["y"] = y.view(rows, -1).to(s["x"].dtype)


def _quantized(x, scale, code):
    """x / scale as codes (held as 32-bit floats), 0 where the scale is."""
    q = torch.where(scale > 0, x / torch.where(scale > 0, scale, 1.0), 0.0)
    return torch.round(q) if code == "int8" else q


def _plain_append(s, case):
    h, d, page, code, rows = case["kv_heads"], case["head"], case["page"], case["code"], case["rows"]
    row = torch.arange(rows, device="cuda")
    ends, past = s["ends"].long(), s["past"].long()
    sequence = torch.searchsorted(ends, row, right=True) - 1
    position = past[sequence] + row - ends[sequence]
    pages, slot = s["table"].long()[sequence, position // page], position % page
    # pages begun earlier that new tokens go to
    begun = (past % page > 0) & (ends[1:] > ends[:-1])
    first = s["table"].long().gather(1, (past // page).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0]
    first, fill = first[begun], (past % page)[begun]
    kept = torch.arange(page, device="cuda") < fill[:, None]
    for new, cache, scales, along in ((s["new_k"], s["k"], s["ks"], 2), (s["new_v"], s["v"], s["vs"], 3)):
        x = new.float().view(rows, h, d)
        amax = torch.zeros_like(scales).index_reduce_(0, pages, x.abs().amax(-1), "amax")
        fresh = amax / torch.full_like(amax, TOP[code])                          # (a division; by a plain number it would be a product with its inverse)
        old = scales[first]
        fresh[first] = torch.maximum(old, fresh[first])
        ratio = torch.where(fresh[first] > 0, old / torch.where(fresh[first] > 0, fresh[first], 1.0), 0.0)
        bits = cache.view(torch.int8)
        before = bits[first]
        recoded = before.view(cache.dtype).float() * ratio[..., None, None]
        recoded = (torch.round(recoded) if code == "int8" else recoded).to(cache.dtype).view(torch.int8)
        bits[first] = torch.where(kept[:, None, :, None] if along == 2 else kept[:, None, None, :], recoded, before)
        scales[pages] = fresh[pages]
        q = _quantized(x, fresh[pages][..., None], code).to(cache.dtype).view(torch.int8)
        if along == 2:
            bits[pages, :, slot] = q
        else:
            bits[pages, :, :, slot] = q


def _gathered(cache, scales, table):
    """The pages of each sequence in 32 bits: [sequences, pages, heads, ..]."""
    return cache.view(torch.int8)[table].view(cache.dtype).float() * scales[table][..., None, None]


def _plain_attend(s, case):
    h, d, page, group, n = case["kv_heads"], case["head"], case["page"], case["heads"] // case["kv_heads"], case["sequences"]
    width, dt = -(-s["most"] // page), s["q"].dtype
    table = s["table"].long()[:, :width].clamp(min=0)
    ends, past = s["ends"].long(), s["past"].long()
    new = ends[1:] - ends[:-1]
    # queries of each sequence, behind one another: [sequences, kv heads, longest * group, head]
    at = torch.arange(s["longest"], device="cuda")
    row = (ends[:-1, None] + at).clamp(max=case["rows"] - 1)
    q = s["q"].float().view(-1, h, group, d)[row].permute(0, 2, 1, 3, 4).reshape(n, h, -1, d)
    k = _gathered(s["k"], s["ks"], table).transpose(1, 2).reshape(n, h, width * page, d)
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
    del k
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    slot = torch.arange(width * page, device="cuda")
    seen = past[:, None] + at                                                   # the query's own slot
    live = slot <= seen[..., None]
    if case["window"]:
        live &= slot > seen[..., None] - case["window"]
    score = score.view(n, h, s["longest"], group, -1).masked_fill_(~live[:, None, :, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1)
    v = _gathered(s["v"], s["vs"], table).permute(0, 2, 1, 4, 3).reshape(n, h, width * page, d)
    v = torch.where((slot < (past + new)[:, None])[:, None, :, None], v, 0.0)   # what lies behind a sequence's end
    y = torch.matmul(score.view(n, h, -1, width * page), v).view(n, h, s["longest"], group, d) / total[..., None]
    y = y.permute(0, 2, 1, 3, 4).reshape(n * s["longest"], -1)
    s["y"] = y[(at < new[:, None]).flatten()].to(dt)


def _plain_pages(s, case):
    page, table, total = case["page"], s["table"].long(), s["pools"][0].shape[1]
    n, width = table.shape
    column = torch.arange(width, device="cuda")
    if case["compact"]:
        used = column < -(-s["lengths"].long() // page)[:, None]
        held = torch.zeros(total, dtype=torch.bool, device="cuda")
        held[table[used]] = True
        count = held.sum()
        front = torch.arange(total, device="cuda") < count
        sources, holes = torch.nonzero(held & ~front)[:, 0], torch.nonzero(~held & front)[:, 0]
        to = torch.arange(total, device="cuda")
        to[sources] = holes
        s["next"] = torch.where(used, to[table.clamp(min=0)], -1).int()
        s["next_lengths"] = s["lengths"].clone()
        s["moves"] = torch.full_like(s["moves"], -1)
        s["moves"][:sources.numel()] = torch.stack([sources, holes], -1).int()
        s["counts"] = torch.stack([count, torch.zeros_like(count)]).int()
    else:
        parents = s["parents"].long()
        alive = parents >= 0
        row = table[parents.clamp(min=0)]
        length = torch.where(alive, s["lengths"].long()[parents.clamp(min=0)], 0)
        full, rest = length // page, length % page > 0
        last = row.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
        whole = column < full[:, None]
        held = torch.zeros(total, dtype=torch.bool, device="cuda")
        held[row[whole]] = True
        # the first of the sequences that would write into a begun page keeps it, unless it is a whole page of another one
        same = (last[:, None] == last[None]) & rest[:, None] & rest[None]
        keeps = rest & ~torch.tril(same, -1).any(1) & ~held[last]
        held[last[keeps]] = True
        copies = rest & ~keeps
        pages = -(-(length + torch.where(alive, s["new"].long(), 0)) // page)
        fresh = (column >= full[:, None]) & (column < pages[:, None]) & ~(keeps[:, None] & (column == full[:, None]))
        place = torch.cumsum(fresh.flatten(), 0).view(n, width) - 1
        free = torch.nonzero(~held)[:, 0]
        got = free[place.clamp(min=0)]
        s["next"] = torch.where(fresh, got, torch.where(whole | (keeps[:, None] & (column == full[:, None])), row, -1)).int()
        s["next_lengths"] = length.int()
        to = s["next"].long().gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
        s["moves"] = torch.where(copies[:, None], torch.stack([last, to], -1), -1).int()
        count = held.sum() + fresh.sum()
        s["counts"] = torch.stack([count, torch.zeros_like(count)]).int()
        sources, holes = last[copies], to[copies]
    for pool in s["pools"]:
        pool[:, holes] = pool[:, sources]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits; None for codes, scales' codes and tables, which are whole numbers."""
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend, "pages": lambda case, s: None}[case["kind"]](case, s)


def _exact_rotary(case, s):
    d, part, heads = case["head"], case["part"] or case["head"], case["heads"] + case["kv_heads"]
    x = s["x"].double().view(case["rows"], -1, d)
    y = x.clone()
    frequencies, factor = _frequencies(case)
    for i, f in enumerate(frequencies):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + part // 2)
        turn = torch.polar(torch.full((case["rows"], 1), factor, dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * f)
        z = torch.complex(x[:, :heads, a], x[:, :heads, b]) * turn
        y[:, :heads, a], y[:, :heads, b] = z.real, z.imag
    return y.flatten(1)


def _exact_append(case, s):
    page, h, d = case["page"], case["kv_heads"], case["head"]
    ends, past, table = s["ends"].tolist(), s["past"].tolist(), s["table"].tolist()
    scales = []
    for new, old in ((s["new_k"], s["ks"]), (s["new_v"], s["vs"])):
        peak, scale = new.double().view(-1, h, d).abs().amax(-1), old.double().clone()
        for i in range(case["sequences"]):
            at, end, pos = ends[i], ends[i + 1], past[i]
            while at < end:
                count = min(end - at, page - pos % page)
                p, top = table[i][pos // page], peak[at:at + count].amax(0) / TOP[case["code"]]
                scale[p] = torch.maximum(scale[p], top) if pos % page else top
                at, pos = at + count, pos + count
        scales.append(scale)
    return {"k": None, "v": None, "ks": scales[0], "vs": scales[1]}


def _exact_attend(case, s):
    h, d, page, group = case["kv_heads"], case["head"], case["page"], case["heads"] // case["kv_heads"]
    y = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda").view(-1, h, group, d)
    ends, past = s["ends"].tolist(), s["past"].tolist()
    for i in range(case["sequences"]):
        n = ends[i + 1] - ends[i]
        length = past[i] + n
        if n == 0:
            continue
        pages = s["table"][i, :-(-length // page)].long()
        q = s["q"][ends[i]:ends[i + 1]].double().view(n, h, group, d)
        own_slot = torch.arange(past[i], length, device="cuda")[:, None]
        slot = torch.arange(length, device="cuda")[None]
        hidden = (slot > own_slot) | ((slot <= own_slot - case["window"]) if case["window"] else False)
        for head in range(h):
            k, v = (c.view(torch.int8)[pages, head].view(c.dtype).double() * m[pages, head].double()[:, None, None] for c, m in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            k, v = k.reshape(-1, d)[:length], v.transpose(1, 2).reshape(-1, d)[:length]
            for member in range(group):
                score = q[:, head, member] @ k.T / math.sqrt(d)
                if case["softcap"]:
                    score = torch.tanh(score / case["softcap"]) * case["softcap"]
                y[ends[i]:ends[i + 1], head, member] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return y.flatten(1)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    item = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "rotary":
        values = case["rows"] * (case["heads"] + 2 * case["kv_heads"]) * case["head"]
        return {"bytes": 2 * values * item + 8 * case["rows"], "flops": 3 * case["rows"] * (case["heads"] + case["kv_heads"]) * (case["part"] or case["head"])}
    if case["kind"] == "append":
        values = 2 * case["rows"] * case["kv_heads"] * case["head"]
        return {"bytes": values * (item + 1), "flops": 3 * values}
    if case["kind"] == "attend":
        n, rows = case["sequences"], case["rows"]
        mean = case["past"] if case["even"] else case["past"] / 2                # tokens cached before, on average
        fresh = rows / n
        sees = mean + (fresh + 1) / 2
        if case["window"]:
            sees = min(sees, case["window"])
        reads = n * min(mean + fresh, (case["window"] or math.inf) + fresh)
        cache = reads * case["kv_heads"] * (2 * case["head"] + 8 / case["page"])
        return {"bytes": int(cache + 2 * rows * case["heads"] * case["head"] * item), "flops": int(4 * rows * sees * case["heads"] * case["head"])}
    one = case["layers"] * case["kv_heads"] * (2 * case["page"] * case["head"] + 8)
    need = case["sequences"] * (-(-3 * case["past"] // 4) // case["page"] + 0.5)  # pages in use, on average
    if case["compact"]:
        moved = need * max(0.0, 1 - need / case["pool"])                         # those in use behind the front that they fill
    else:
        # sequences that share a begun page with an earlier one of the same parent: the mean number, as the parents are drawn
        b = case["beams"]
        parents = sum(1 - (1 - (2 * (b - j) - 1) / b ** 2) ** b for j in range(b))
        moved = case["sequences"] / b * (b - parents) * 0.95 * (1 - 1 / case["page"])
    return {"bytes": int(2 * moved * one + 8 * need), "flops": 0}
