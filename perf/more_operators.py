"""Positions, 8-bit floats and experts in a decoder layer: the cases that are measured, their plain forms, and their values in 64 bits.

Five operators:

* ``rotate``   norms of queries and keys head by head and the rotation of their positions (one axis or several), the keys and
  values written into a paged int8 cache and read back, or the keys kept as they are
* ``rows``     rows in 8-bit floats with a scale for each 128 columns: of values, of a residual's addition and a norm, of a gated
  activation; and the values these stand for
* ``matmul``   a product of 8-bit float rows with a scale for each 128 columns and weights with one for each 128 x 128
* ``experts``  the same product for rows sorted by expert, each with its expert's weights, read from the tokens' rows
* ``route``    the order of tokens sorted by expert, and the experts' rows weighted and added back to their tokens

``run`` computes them with elementary torch operations where ``own`` is false, and calls ``spinnv2_amd.decoder`` where it is true.
"""

import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
BLOCK = 128


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one new token for each of four sequences: latency
        dict(name="rotate decode 4", op="rotate", tokens=4, heads=32, kv_heads=8, dim=128, pairs=64, axes=1, split=True, norm=True,
             page=16, first=70001, type="bf16"),
        # a long prompt with an image's three axes, into the cache
        dict(name="rotate prompt 8190", op="rotate", tokens=8190, heads=32, kv_heads=8, dim=128, pairs=64, axes=3, split=True, norm=True,
             page=64, first=0, type="bf16"),
        # float32 heads of 80, of which the first 32 turn, pairs side by side, no norm, no cache
        dict(name="rotate fp32 777", op="rotate", tokens=777, heads=12, kv_heads=12, dim=80, pairs=16, axes=1, split=False, norm=False,
             page=0, first=1500, type="fp32"),
        # the norm ahead of a projection while four sequences are decoded: latency
        dict(name="rows norm 4x2048", op="rows", kind="norm", rows=4, cols=2048, type="bf16"),
        # the gate between the two products of a prompt's tokens
        dict(name="rows gate 8190x8192", op="rows", kind="gate", rows=8190, cols=8192, type="bf16"),
        # one token through a square projection: the weights' bytes
        dict(name="matmul 1x4096x4096", op="matmul", m=1, n=4096, k=4096, type="bf16", bias=False),
        # a few ragged tokens, a last block that is not full, with a bias, float32 out
        dict(name="matmul 77x1000x2000", op="matmul", m=77, n=1000, k=2000, type="fp32", bias=True),
        # a prompt's tokens through a wide projection: the matrix cores
        dict(name="matmul 8192x8192x8192", op="matmul", m=8192, n=8192, k=8192, type="bf16", bias=False),
        # 64 sequences' new tokens, eight experts each: every expert's weights for a few rows
        dict(name="experts 64 of 64", op="experts", tokens=64, chosen=8, experts=64, n=2048, k=2048, type="bf16"),
        # a prompt's tokens, four experts each: the matrix cores, ragged groups
        dict(name="experts 4001 of 32", op="experts", tokens=4001, chosen=4, experts=32, n=4096, k=2048, type="bf16"),
        # 64 sequences' new tokens sorted and added back: latency
        dict(name="route 64 of 64", op="route", tokens=64, chosen=8, experts=64, cols=2048, type="bf16"),
        # a prompt's tokens sorted and added back
        dict(name="route 8190 of 128", op="route", tokens=8190, chosen=8, experts=128, cols=2048, type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotate", "rows", "matmul", "experts", "route"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rotate":
        kv, dim = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 80, 96, 128, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        most = 8190 * (32 + 2 * 8) * 128 * 2 // ((heads + 2 * kv) * dim * BYTES[kind])
        pairs = rng.choice([dim // 2, dim // 2, dim // 4, rng.randrange(1, dim // 2 + 1)])
        return dict(op=op, tokens=_spread(rng, 1, min(8190, most)), heads=heads, kv_heads=kv, dim=dim, pairs=pairs,
                    axes=rng.choice([1, 1, 2, 3]), split=rng.random() < 0.7, norm=rng.random() < 0.7,
                    page=rng.choice([0, 16, 32, 64, 256]), first=_spread(rng, 1, 1000000), type=kind)
    if op == "rows":
        source, cols = rng.choice(["norm", "values", "gate"]), _spread(rng, 64, 16384)
        rows = _spread(rng, 1, max(1, min(16384, 8190 * 8192 // cols // BYTES[kind] * 2)))
        return dict(op=op, kind=source, rows=rows, cols=cols, type=kind)
    if op == "matmul":
        n, k = _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        return dict(op=op, m=_spread(rng, 1, min(8192, max(1, (1 << 37) // (n * k)))), n=n, k=k, type=kind, bias=rng.random() < 0.3)
    experts = _spread(rng, 2, 256)
    chosen = rng.randrange(1, min(8, experts) + 1)
    if op == "experts":
        n, k = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
        experts = max(2, min(experts, (1 << 28) // (n * k)))
        chosen = min(chosen, experts)
        return dict(op=op, tokens=_spread(rng, 1, min(8192, max(1, (1 << 37) // (n * k * chosen)))), chosen=chosen, experts=experts, n=n, k=k,
                    type=kind)
    cols = _spread(rng, 64, 8192)
    most = 8190 * 9 * 2048 * 2 // ((chosen + 1) * cols * BYTES[kind])
    return dict(op=op, tokens=_spread(rng, 1, max(1, min(16384, most))), chosen=chosen, experts=experts, cols=cols, type=kind)


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "rotate":
        t, q, kv = case["tokens"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        if case["page"]:  # codes and scales out and in, values out
            moved = t * (2 * q * size + 4 * kv * size + 4 * kv + 16 * case["kv_heads"])
        else:
            moved = t * 2 * (q + kv) * size
        return {"bytes": moved + 4 * t * case["axes"] + 4 * case["pairs"], "flops": 6 * t * (q + kv)}
    if case["op"] == "rows":
        n = case["rows"] * case["cols"]
        # norm: input, residual in and out; gate: two inputs; then codes out and in, the values out
        inward = {"norm": 3, "values": 1, "gate": 2}[case["kind"]] * size
        return {"bytes": n * (inward + 2 + size) + 8 * case["rows"] * _blocks(case["cols"]), "flops": 8 * n}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size + 4 * (m + _blocks(n)) * _blocks(k) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "experts":
        t, rows, n, k = case["tokens"], case["tokens"] * case["chosen"], case["n"], case["k"]
        used = min(case["experts"], rows)
        return {"bytes": t * k + used * n * k + rows * n * size + 4 * (t + used * _blocks(n)) * _blocks(k) + 4 * rows, "flops": 2 * rows * n * k}
    rows = case["tokens"] * case["chosen"]
    return {"bytes": (rows + case["tokens"]) * case["cols"] * size + 16 * rows, "flops": 2 * rows * case["cols"]}


# ----------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _codes8(g, *shape):
    """8-bit floats as a quantiser by blocks makes them of normal values: the largest of 128 near 448."""
    return (_normal(g, *shape) * 160).clamp_(-448, 448).to(F8)


def _chosen(g, tokens, chosen, experts):
    """Each token's experts, none twice; some experts are liked more than others."""
    liking = _normal(g, experts) * 0.7 + torch.rand(tokens, experts, generator=g, device=g.device).clamp_(min=1e-9).log_().neg_().log_().neg_()
    return liking.topk(chosen, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    d = _device()
    g = torch.Generator(device=d)
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "rotate":
        n, heads, kv, dim, pairs = (case[x] for x in ("tokens", "heads", "kv_heads", "dim", "pairs"))
        # one product's output, whose columns are the queries, keys and values
        s["qkv"] = _normal(g, n, (heads + 2 * kv) * dim).to(t)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, dim)) for x in s["qkv"].split([heads * dim, kv * dim, kv * dim], 1))
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * _normal(g, dim)).to(t) if case["norm"] else None for _ in range(2))
        s["frequencies"] = (1000000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=d) / pairs)).float()
        # runs of pairs for the axes one after the other
        s["axis"] = (torch.arange(pairs, device=d) * case["axes"] // pairs).to(torch.int32) if case["axes"] > 1 else None
        at = torch.arange(n, device=d)
        s["positions"] = torch.stack([case["first"] + at, at // 40 % 50, at % 40][:case["axes"]], 1).to(torch.int32)
        s["q_out"] = torch.empty(n, heads, dim, dtype=t, device=d)
        s["k_out"] = torch.empty(n, kv, dim, dtype=t, device=d)
        if case["page"]:
            page = case["page"]
            s["v_out"] = torch.empty_like(s["k_out"])
            pages = -(-n // page)
            s["table"] = torch.randperm(pages, generator=g, device=d).to(torch.int32)[None].contiguous()
            s["slots"] = s["table"][0, at // page].long() * page + at % page
            for x in ("k", "v"):
                s[x + "_codes"] = torch.zeros(pages, kv, page, dim, dtype=torch.int8, device=d)
                s[x + "_scale"] = torch.zeros(pages, kv, page, device=d)
            s["offsets"] = torch.tensor([0, n], dtype=torch.int32, device=d)
    elif case["op"] == "rows":
        rows, cols = case["rows"], case["cols"]
        wide = 2 * cols if case["kind"] == "gate" else cols
        # a few channels far larger than the others, as residual streams have them
        loud = 1.0 if case["kind"] == "gate" else torch.where(torch.rand(cols, generator=g, device=d) < 0.005, 30.0, 1.0)
        s["x"] = (_normal(g, rows, wide) * loud).to(t)
        s["residual"] = (_normal(g, rows, cols) * loud).to(t) if case["kind"] == "norm" else None
        s["weight"] = (1 + 0.2 * _normal(g, cols)).to(t) if case["kind"] == "norm" else None
        s["sum"] = torch.empty(rows, cols, dtype=t, device=d) if case["kind"] == "norm" else None
        s["q"] = torch.empty(rows, cols, dtype=F8, device=d)
        s["scale"] = torch.empty(rows, _blocks(cols), dtype=torch.float32, device=d)
        s["values"] = torch.empty(rows, cols, dtype=t, device=d)
    elif case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["b"] = _codes8(g, m, k), _codes8(g, n, k)
        s["a_scale"] = 0.005 + 0.005 * torch.rand(m, _blocks(k), generator=g, device=d)
        s["b_scale"] = 0.0001 + 0.0001 * torch.rand(_blocks(n), _blocks(k), generator=g, device=d)
        s["bias"] = _normal(g, n) if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=t, device=d)
    else:
        tokens, chosen, experts = case["tokens"], case["chosen"], case["experts"]
        s["ids"] = _chosen(g, tokens, chosen, experts)
        if case["op"] == "experts":
            n, k = case["n"], case["k"]
            s["a"] = _codes8(g, tokens, k)
            s["a_scale"] = 0.005 + 0.005 * torch.rand(tokens, _blocks(k), generator=g, device=d)
            s["b"] = _codes8(g, experts, n, k)
            s["b_scale"] = 0.0001 + 0.0001 * torch.rand(experts, _blocks(n), _blocks(k), generator=g, device=d)
            s["order"] = torch.argsort(s["ids"].flatten(), stable=True).to(torch.int32)
            s["offsets"] = torch.searchsorted(s["ids"].flatten().sort().values.long(), torch.arange(experts + 1, device=d)).to(torch.int32)
            s["bounds"] = s["offsets"].tolist()  # for the plain form's loop over experts
            s["out"] = torch.empty(tokens * chosen, n, dtype=t, device=d)
        else:
            cols = case["cols"]
            s["weights"] = torch.softmax(_normal(g, tokens, chosen), 1)
            s["y"] = _normal(g, tokens * chosen, cols).to(t)
            s["offsets"] = torch.empty(experts + 1, dtype=torch.int32, device=d)
            s["order"] = torch.empty(tokens * chosen, dtype=torch.int32, device=d)
            s["place"] = torch.empty(tokens, chosen, dtype=torch.int32, device=d)
            s["out"] = torch.empty(tokens, cols, dtype=t, device=d)
    return s


# ------------------------------------------------------------------- runs

def run(s):
    if own:
        return _run_own(s)
    return {"rotate": _rotate, "rows": _rows, "matmul": _matmul, "experts": _experts, "route": _route}[s["op"]](s)


def _run_own(s):
    from spinnv2_amd import decoder

    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "rotate":
        norm = dict(norm=s["norm"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        if not s["page"]:
            decoder.rotate(s["q"], s["k"], s["positions"], s["frequencies"], s["q_out"], s["k_out"], axes=s["axis"],
                           interleaved=not s["split"], stream=stream, **norm)
            return {"q": s["q_out"], "k": s["k_out"]}
        if "cache" not in s:  # a program makes it once
            s["cache"] = decoder.KvCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        decoder.rotate(s["q"], s["k"], s["positions"], s["frequencies"], s["q_out"], None, axes=s["axis"], interleaved=not s["split"],
                       cache=s["cache"], v=s["v"], slots=s["slots"], stream=stream, **norm)
        s["cache"].read(s["table"], None, s["offsets"], s["k_out"], s["v_out"], stream=stream)
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if s["op"] == "rows":
        if s["kind"] == "norm":
            decoder.rmsnorm_f8(s["x"], s["weight"], s["q"], s["scale"], residual=s["residual"], residual_out=s["sum"], eps=EPS, stream=stream)
        elif s["kind"] == "gate":
            decoder.gate_f8(s["x"], s["q"], s["scale"], stream=stream)
        else:
            decoder.quantize_f8(s["x"], s["q"], s["scale"], stream=stream)
        decoder.dequantize_f8(s["q"], s["scale"], s["values"], stream=stream)
        return {"values": s["values"], "sum": s["sum"], "scale": s["scale"]}
    if s["op"] == "matmul":
        decoder.matmul_f8(s["a"], s["a_scale"], s["b"], s["b_scale"], s["out"], bias=s["bias"], stream=stream)
        return s["out"]
    if s["op"] == "experts":
        decoder.matmul_f8_experts(s["a"], s["a_scale"], s["b"], s["b_scale"], s["offsets"], s["out"], order=s["order"], per_token=s["chosen"],
                                  stream=stream)
        return s["out"]
    decoder.sort_tokens(s["ids"], s["offsets"], s["order"], s["place"], stream=stream)
    decoder.combine(s["y"], s["place"], s["weights"], s["out"], stream=stream)
    return {"offsets": s["offsets"], "order": s["order"], "place": s["place"], "out": s["out"]}


def _turned(s, x, weight):
    """Heads with their norm and their positions' rotation, in 64 bits: the angles of far positions need them, and so do keys next to
    the border of two codes."""
    wide = x.double()
    if s["norm"]:
        wide = wide * (wide.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.double()
    pairs = s["pairs"]
    positions = s["positions"].double() if s["axis"] is None else s["positions"][:, s["axis"].long()].double()
    angle = (positions * s["frequencies"].double())[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if s["split"] else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    a, b = wide[..., first], wide[..., second]
    out = wide.clone()
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out.to(x.dtype)


def _rotate(s):
    q, k = _turned(s, s["q"], s["q_weight"]), _turned(s, s["k"], s["k_weight"])
    if not s["page"]:
        return {"q": q, "k": k}
    page, out = s["page"], {"q": q}
    place, row = s["slots"] // page, s["slots"] % page
    for name, x in (("k", k), ("v", s["v"])):
        wide = x.double()
        top = wide.abs().amax(-1, keepdim=True)
        s[name + "_codes"][place, :, row] = torch.where(top > 0, (wide * 127 / top).round(), 0.0).to(torch.int8)
        s[name + "_scale"][place, :, row] = (top / 127).squeeze(-1).float()
        out[name] = (s[name + "_codes"][place, :, row].float() * s[name + "_scale"][place, :, row, None]).to(x.dtype)
    return out


def _in_blocks(x):
    """[.., cols] as [.., blocks, 128], zeros behind the last column."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))


def _rows(s):
    cols, t = s["cols"], s["x"].dtype
    h, norm = None, 1.0
    if s["kind"] == "gate":
        gate, up = s["x"][:, :cols].double(), s["x"][:, cols:].double()
        wide = gate / (1 + torch.exp(-gate)) * up
    elif s["kind"] == "norm":
        h = (s["x"].float() + s["residual"].float()).to(t)
        norm = (h.double().square().mean(-1, keepdim=True) + EPS).rsqrt()
        wide = h.double() * s["weight"].double()  # the norm is one factor for the whole row: the codes are those of h * weight
    else:
        wide = s["x"].double()
    blocks = _in_blocks(wide)
    top = blocks.abs().amax(-1, keepdim=True)
    # to 4 bits of 2^-9 at least, in 64 bits since a value next to the border of two codes has to fall on its own side
    y = torch.where(top > 0, blocks * 448 / top, 0.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    step = torch.where(y.abs() >= step * 16, step * 2, torch.where((y.abs() < step * 8) & (step > 2.0 ** -9), step / 2, step))
    codes = (y / step).round() * step
    scale = (top.squeeze(-1) * norm / 448).float()
    values = (codes.float() * scale[..., None]).flatten(-2)[:, :cols].to(t)
    return {"values": values, "sum": h, "scale": scale}


def _scaled_rows(a, scale):
    """8-bit floats [.., rows, k] times their scales [.., rows, blocks], in 32 bits."""
    return a.float() * scale.repeat_interleave(BLOCK, -1)[..., :a.shape[-1]]


def _product(a, a_scale, b, b_scale):
    wide = _scaled_rows(b, b_scale.repeat_interleave(BLOCK, 0)[:b.shape[0]])
    return torch.matmul(_scaled_rows(a, a_scale), wide.t())


def _matmul(s):
    y = _product(s["a"], s["a_scale"], s["b"], s["b_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"].dtype)


def _experts(s):
    row = s["order"].long() // s["chosen"]
    out = torch.empty_like(s["out"])
    for e in range(s["experts"]):
        low, high = s["bounds"][e], s["bounds"][e + 1]
        if high > low:
            out[low:high] = _product(s["a"].view(torch.uint8)[row[low:high]].view(F8), s["a_scale"][row[low:high]], s["b"][e],
                                     s["b_scale"][e]).to(out.dtype)
    return out


def _route(s):
    ids = s["ids"].flatten().long()
    experts = torch.arange(s["experts"], device=ids.device)
    count = (ids[:, None] == experts).int()
    offsets = torch.cat([count.new_zeros(1), count.sum(0).cumsum(0)]).to(torch.int32)
    at = torch.arange(ids.shape[0], device=ids.device)
    place = offsets[ids].long() + count.cumsum(0)[at, ids] - 1
    order = torch.empty_like(place)
    order[place] = at
    rows = s["y"][place.view(s["ids"].shape)].float()
    out = (rows * s["weights"][..., None]).sum(1).to(s["y"].dtype)
    return {"offsets": offsets, "order": order.to(torch.int32), "place": place.to(torch.int32).view(s["ids"].shape), "out": out}


# ----------------------------------------------------- the values in 64 bits

def _e4m3():
    """The 8-bit floats from zero on, in 64 bits: 2^-9 .. 7 2^-9, then eight to each power of two up to 448."""
    return torch.tensor([i * 2.0 ** -9 for i in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1],
                        dtype=torch.float64, device=_device())


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            if case["norm"]:
                x = x / torch.sqrt((x * x).sum(2, keepdim=True) / case["dim"] + EPS) * s[name + "_weight"].double()
            p = s["positions"].double()
            p = p[:, :1].expand(-1, case["pairs"]) if s["axis"] is None else p.gather(1, s["axis"].long().expand(p.shape[0], -1))
            turn = torch.polar(torch.ones_like(p), p * s["frequencies"].double())[:, None, :]
            n = 2 * case["pairs"]
            head = x[..., :n].unflatten(2, (2, -1)).transpose(2, 3) if case["split"] else x[..., :n].unflatten(2, (-1, 2))
            head = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
            head = (head.transpose(2, 3) if case["split"] else head).flatten(2)
            out[name] = torch.cat([head, x[..., n:]], 2)
        if not case["page"]:
            return out
        for name, x in (("k", out["k"].to(s["k"].dtype)), ("v", s["v"])):  # a key is held in its own type before its codes
            x = x.double()
            top = x.abs().max(dim=2, keepdim=True).values
            out[name] = torch.round(x * 127 / top) * (top / 127)
        return out
    if case["op"] == "rows":
        rows, cols = case["rows"], case["cols"]
        total, factor = None, torch.ones(rows, 1, dtype=torch.float64, device=s["x"].device)
        x = s["x"].double()
        if case["kind"] == "gate":
            x = x[:, :cols] * torch.sigmoid(x[:, :cols]) * x[:, cols:]
        elif case["kind"] == "norm":
            total = (x + s["residual"].double()).to(s["x"].dtype).double()  # the sum is held in its own type
            factor = 1 / torch.sqrt((total * total).sum(1, keepdim=True) / cols + EPS)
            x = total * s["weight"].double()
        table = _e4m3()
        border = (table[1:] + table[:-1]) / 2
        values, scales = torch.empty_like(x), []
        for i in range(0, cols, BLOCK):
            part = x[:, i:i + BLOCK]
            top = part.abs().max(dim=1, keepdim=True).values
            y = part.abs() * 448 / top
            at = torch.searchsorted(border, y.contiguous())  # a border itself goes down, and up from an odd code
            up = (at < border.shape[0]) & (border[at.clamp(max=border.shape[0] - 1)] == y) & (at % 2 == 1)
            code = table[at + up.long()]
            scales.append(top * factor / 448)
            values[:, i:i + BLOCK] = torch.copysign(code, part) * scales[-1]
        return {"values": values, "sum": total, "scale": torch.cat(scales, 1)}
    if case["op"] == "matmul":
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=s["a"].device)
        for block, i in enumerate(range(0, case["k"], BLOCK)):
            part = torch.mm(s["a"][:, i:i + BLOCK].double(), s["b"][:, i:i + BLOCK].double().t().contiguous())
            scale = s["b_scale"][:, block].double()[torch.arange(case["n"], device=y.device) // BLOCK]
            y += part * torch.outer(s["a_scale"][:, block].double(), scale)
        return y if s["bias"] is None else y + s["bias"].double()
    flat = s["ids"].flatten().long()
    if case["op"] == "experts":
        y = torch.empty(flat.shape[0], case["n"], dtype=torch.float64, device=flat.device)
        a = s["a"].double() * s["a_scale"].double().repeat_interleave(BLOCK, 1)[:, :case["k"]]
        at = 0
        for e in range(case["experts"]):
            tokens = (flat == e).nonzero()[:, 0] // case["chosen"]
            w = s["b"][e].double() * s["b_scale"][e].double().repeat_interleave(BLOCK, 0)[:case["n"]].repeat_interleave(BLOCK, 1)[:, :case["k"]]
            y[at:at + len(tokens)] = torch.mm(a[tokens], w.t().contiguous())
            at += len(tokens)
        return y
    order = torch.cat([(flat == e).nonzero()[:, 0] for e in range(case["experts"])])
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=order.device)
    place = place.view(s["ids"].shape)
    out = torch.zeros(case["tokens"], case["cols"], dtype=torch.float64, device=flat.device)
    for j in range(case["chosen"]):
        out += s["weights"][:, j:j + 1].double() * s["y"][place[:, j]].double()
    counts = torch.bincount(flat, minlength=case["experts"])
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return {"offsets": offsets.to(torch.int32), "order": order.to(torch.int32), "place": place.to(torch.int32), "out": out}
