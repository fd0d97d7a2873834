"""The operators of a decoder layer in 8 bits: the cases that are measured, their plain forms, and their values in 64 bits.

Four operators of a decoder that holds activations, weights and cache as int8 with scales:

* ``norm``    the residual's addition, a root-mean-square norm and int8 rows with one scale each, and the values these stand for
* ``matmul``  a product of int8 rows and int8 weights with a scale for each token and each output channel
* ``cache``   keys and values quantised as they are written into a paged cache, and read back from it
* ``attend``  attention of new tokens to a paged int8 cache: single tokens, whole prompts, an encoder's states

``run`` computes them with elementary torch operations where ``own`` is false, and calls ``spinnv2_amd.decoder`` where it is true.
"""

import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the norm ahead of a projection while four sequences are decoded: latency
        dict(name="norm decode 4x2048", op="norm", rows=4, cols=2048, type="bf16", residual=True),
        # the same norm over the tokens of a long prompt, not a multiple of any tile
        dict(name="norm prompt 8190x4096", op="norm", rows=8190, cols=4096, type="bf16", residual=True),
        # float32 activations, as this runtime's packages hold them, without a residual, rows of an odd length
        dict(name="norm fp32 777x1001", op="norm", rows=777, cols=1001, type="fp32", residual=False),
        # one token through a square projection: the weights' bytes
        dict(name="matmul 1x4096x4096", op="matmul", m=1, n=4096, k=4096, type="bf16", bias=False),
        # the classifier of the ResNet benchmark at its batch of 64, with its bias, float32 out
        dict(name="matmul 64x1000x2048", op="matmul", m=64, n=1000, k=2048, type="fp32", bias=True),
        # a prompt's tokens through a wide projection: the matrix cores
        dict(name="matmul 8192x8192x8192", op="matmul", m=8192, n=8192, k=8192, type="bf16", bias=False),
        # one new token for each of 64 sequences, some of them idle: the new tokens written, and read back
        dict(name="cache append 64", op="cache", seqs=64, first=700, tokens=1, heads=8, dim=128, page=16, type="bf16", idle=5),
        # the prompts of three sequences written and read back
        dict(name="cache prompts 3x8191", op="cache", seqs=3, first=0, tokens=8191, heads=8, dim=128, page=64, type="fp16", idle=0),
        # one sequence of a few hundred tokens decoding: latency
        dict(name="attend 1 of 333", op="attend", seqs=1, queries=1, low=333, high=333, heads=32, kv_heads=8, dim=128, page=16,
             type="bf16", causal=True, window=0),
        # 64 sequences of ragged lengths up to 16384 decoding: the cache's bytes
        dict(name="attend 64 of 16384", op="attend", seqs=64, queries=1, low=3001, high=16384, heads=32, kv_heads=8, dim=128, page=64,
             type="bf16", causal=True, window=0),
        # the last 4001 tokens of two prompts, one of them behind an earlier part: the matrix cores
        dict(name="attend prompts 2x4001", op="attend", seqs=2, queries=4001, low=4001, high=6007, heads=32, kv_heads=8, dim=128,
             page=64, type="bf16", causal=True, window=0),
        # eight decoders' tokens attending to an encoder's states of another length
        dict(name="attend encoder 8x77 of 1500", op="attend", seqs=8, queries=77, low=1500, high=1500, heads=12, kv_heads=12, dim=64,
             page=32, type="fp16", causal=False, window=0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "matmul", "cache", "attend"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        cols = _spread(rng, 64, 16384)
        return dict(op=op, rows=_spread(rng, 1, max(1, min(16384, (8190 * 4096) // cols // BYTES[kind] * 2))), cols=cols, type=kind,
                    residual=rng.random() < 0.7)
    if op == "matmul":
        n, k = _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        return dict(op=op, m=_spread(rng, 1, min(8192, max(1, (1 << 37) // (n * k)))), n=n, k=k, type=kind, bias=rng.random() < 0.3)
    heads_kv = rng.choice([1, 2, 4, 8, 12])
    dim, page = rng.choice([64, 80, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
    room = (3 * 8191 * 8 * 128) // (heads_kv * dim)  # tokens of the largest listed cache write
    if op == "cache":
        seqs = _spread(rng, 1, 64)
        tokens = _spread(rng, 1, min(8191, max(1, room // seqs)))
        return dict(op=op, seqs=seqs, first=rng.randrange(0, 1000), tokens=tokens, heads=heads_kv, dim=dim, page=page, type=kind,
                    idle=rng.randrange(0, seqs))
    heads = heads_kv * rng.choice([1, 2, 4, 5, 8])
    causal = rng.random() < 0.75
    if rng.random() < 0.6:  # single tokens, or the few of a drafted continuation
        seqs, queries = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7])
        high = _spread(rng, 16, min(16384, max(16, 64 * 16384 * 8 * 128 // (seqs * heads_kv * dim) // 4)))
    else:
        queries = _spread(rng, 8, 2048)
        seqs = _spread(rng, 1, max(1, min(16, 4096 // queries)))
        high = max(_spread(rng, 16, 4096), queries if causal else 16)
    low = rng.randrange(max(1, high // 3), high + 1)
    return dict(op=op, seqs=seqs, queries=queries, low=max(low, min(queries, high)) if causal else low, high=high, heads=heads,
                kv_heads=heads_kv, dim=dim, page=page, type=kind, causal=causal, window=rng.choice([0, 0, 0, 100, 1000]) if causal else 0)


def _lengths(case):
    """The lengths of a case's sequences, from `low` to `high` in a mixed order, the last the longest."""
    b, low, high = case["seqs"], case["low"], case["high"]
    return [high if i == b - 1 else low + (high - low) * (i * 37 % b) // b for i in range(b)]


def _pairs(case):
    """How many (query, key) pairs a case's masks leave for each head, and how many keys some query attends to."""
    pairs = keys = 0
    for n in _lengths(case):
        for i in range(case["queries"]):
            last = n - case["queries"] + i if case["causal"] else n - 1
            start = max(0, last + 1 - case["window"]) if case["window"] else 0
            pairs += max(0, last + 1 - start)
        keys += n - (max(0, n - case["queries"] + 1 - case["window"]) if case["window"] else 0)
    return pairs, keys


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        # input, residual in and out, codes out and in, the values out
        return {"bytes": n * ((3 if case["residual"] else 1) * size + 2 + size) + case["cols"] * size + 8 * case["rows"], "flops": 8 * n}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size + 4 * (m + n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if case["op"] == "cache":
        n = case["seqs"] * case["tokens"] * case["heads"] * 2
        # values in, codes and scales out and in, values out
        return {"bytes": n * (2 * case["dim"] * size + 2 * case["dim"] + 8), "flops": 4 * n * case["dim"]}
    pairs, keys = _pairs(case)
    return {"bytes": 2 * keys * case["kv_heads"] * (case["dim"] + 4) + 2 * case["seqs"] * case["queries"] * case["heads"] * case["dim"] * size,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ----------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _codes(g, *shape):
    """int8 codes as an absolute-maximum quantiser makes them of normal values."""
    return (_normal(g, *shape) * 45).round_().clamp_(-127, 127).to(torch.int8)


def _pages(g, lengths, page):
    """(table, pages): every sequence's pages, in random order from 1 on; page 0 belongs to no sequence."""
    need = [max(1, -(-n // page)) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device=g.device).to(torch.int32) + 1
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=g.device)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 1


def _offsets(counts, device):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=device)


def prepare(case, seed):
    d = _device()
    g = torch.Generator(device=d)
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # a few channels far larger than the others, as residual streams have them
        loud = torch.where(torch.rand(cols, generator=g, device=d) < 0.005, 30.0, 1.0)
        s["x"] = (_normal(g, rows, cols) * loud).to(t)
        s["residual"] = (_normal(g, rows, cols) * loud).to(t) if case["residual"] else None
        s["weight"] = (1 + 0.2 * _normal(g, cols)).to(t)
        s["sum"] = torch.empty(rows, cols, dtype=t, device=d) if case["residual"] else None
        s["q"] = torch.empty(rows, cols, dtype=torch.int8, device=d)
        s["scale"] = torch.empty(rows, dtype=torch.float32, device=d)
        s["values"] = torch.empty(rows, cols, dtype=t, device=d)
    elif case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["b"] = _codes(g, m, k), _codes(g, n, k)
        s["a_scale"] = 0.02 + 0.01 * torch.rand(m, generator=g, device=d)
        s["b_scale"] = 0.0005 + 0.0005 * torch.rand(n, generator=g, device=d)
        s["bias"] = _normal(g, n) if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=t, device=d)
    elif case["op"] == "cache":
        b, first, tokens, heads, dim, page = (case[x] for x in ("seqs", "first", "tokens", "heads", "dim", "page"))
        s["table"], pages = _pages(g, [first + tokens] * b, page)
        total = b * tokens
        s["k"], s["v"] = (_normal(g, total, heads, dim).to(t) for _ in range(2))
        at = torch.arange(total, device=d)
        at, place = at // tokens, first + at % tokens
        slots = s["table"][at, place // page].long() * page + place % page
        s["slots"] = torch.where(at < case["idle"], -1, slots)  # an idle sequence writes nothing
        for x in ("k", "v"):
            s[x + "_codes"] = _codes(g, pages, heads, page, dim)
            s[x + "_scale"] = 0.01 + 0.01 * torch.rand(pages, heads, page, generator=g, device=d)
            s["out_" + x] = torch.empty(total, heads, dim, dtype=t, device=d)
        s["firsts"] = torch.full((b,), first, dtype=torch.int32, device=d)
        s["offsets"] = _offsets([tokens] * b, d)
    else:
        b, queries, heads, kv, dim, page = (case[x] for x in ("seqs", "queries", "heads", "kv_heads", "dim", "page"))
        lengths = _lengths(case)
        s["table"], pages = _pages(g, lengths, page)
        for x in ("k", "v"):
            s[x + "_codes"] = _codes(g, pages, kv, page, dim)
            s[x + "_scale"] = 0.015 + 0.015 * torch.rand(pages, kv, page, generator=g, device=d)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=d)
        s["offsets"] = _offsets([queries] * b, d)
        s["q"] = (1.5 * _normal(g, b * queries, heads, dim)).to(t)
        s["out"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------------- runs

def run(s):
    if own:
        return _run_own(s)
    return {"norm": _norm, "matmul": _matmul, "cache": _cache, "attend": _attend}[s["op"]](s)


def _run_own(s):
    from spinnv2_amd import decoder

    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "norm":
        decoder.rmsnorm_i8(s["x"], s["weight"], s["q"], s["scale"], residual=s["residual"], residual_out=s["sum"], eps=EPS, stream=stream)
        decoder.dequantize_i8(s["q"], s["scale"], s["values"], stream=stream)
        return {"values": s["values"], "sum": s["sum"], "scale": s["scale"]}
    if s["op"] == "matmul":
        decoder.matmul_i8(s["a"], s["a_scale"], s["b"], s["b_scale"], s["out"], bias=s["bias"], stream=stream)
        return s["out"]
    if "handles" not in s:  # a program makes them once
        s["handles"] = _handles(decoder, s)
    cache, workspace = s["handles"]
    if s["op"] == "cache":
        cache.write(s["k"], s["v"], s["slots"], stream=stream)
        cache.read(s["table"], s["firsts"], s["offsets"], s["out_k"], s["out_v"], stream=stream)
        return {"k": s["out_k"], "v": s["out_v"]}
    decoder.attention(s["q"], cache, s["table"], s["lengths"], s["offsets"], s["out"], max_queries=s["queries"], max_length=s["high"],
                      causal=s["causal"], window=s["window"], workspace=workspace, stream=stream)
    return s["out"]


def _handles(decoder, s):
    """What a program keeps for its calls: the cache, and the workspace of its attention."""
    cache = decoder.KvCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    if s["op"] == "cache":
        return cache, None
    size = decoder.attention_workspace(s["seqs"], s["seqs"] * s["queries"], s["heads"], cache, max_queries=s["queries"], max_length=s["high"])
    return cache, torch.empty(size, dtype=torch.uint8, device=s["q"].device)


def _quantise(x):
    """(codes, scales): the last axis of x by its absolute maximum, in 64 bits, since a value next to the border of two codes has to
    fall on its own side; ties to the even code."""
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.where(top > 0, (x * 127 / top).round(), 0.0)
    return codes, top / 127


def _norm(s):
    t = s["x"].dtype
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(t)
    wide = h.double()
    norm = (wide.square().mean(-1, keepdim=True) + EPS).rsqrt()
    # the norm is one factor for the whole row: the codes are those of h * weight
    codes, top = _quantise(wide * s["weight"].double())
    scale = (top * norm).float()
    return {"values": (codes.float() * scale).to(t), "sum": None if s["residual"] is None else h, "scale": scale.squeeze(-1)}


def _matmul(s):
    y = torch.matmul(s["a"].float(), s["b"].float().t()) * s["a_scale"][:, None] * s["b_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"].dtype)


def _cache(s):
    page, t = s["page"], s["k"].dtype
    # tokens without a slot go to page 0, which no sequence reads
    to = s["slots"].clamp(min=0)
    total = s["out_k"].shape[0]
    at = torch.arange(total, device=to.device)
    seq = torch.searchsorted(s["offsets"][1:], at, right=True)
    place = s["firsts"][seq] + at - s["offsets"][seq]
    pages, rows = s["table"][seq, place // page].long(), place % page
    out = {}
    for x in ("k", "v"):
        codes, scale = _quantise(s[x].double())
        s[x + "_codes"][to // page, :, to % page] = codes.to(torch.int8)
        s[x + "_scale"][to // page, :, to % page] = scale.squeeze(-1).float()
        out[x] = (s[x + "_codes"][pages, :, rows].float() * s[x + "_scale"][pages, :, rows, None]).to(t)
    return out


def _attend(s):
    b, queries, heads, kv, dim, page, high = (s[x] for x in ("seqs", "queries", "heads", "kv_heads", "dim", "page", "high"))
    d = s["q"].device
    place = torch.arange(high, device=d)
    pages, rows = s["table"][:, place // page].long(), place % page
    there = (place < s["lengths"][:, None])[:, :, None, None]
    k, v = (torch.where(there, s[x + "_codes"][pages, :, rows].float() * s[x + "_scale"][pages, :, rows, None], 0.0) for x in ("k", "v"))
    group = heads // kv
    q = s["q"].float().view(b, queries, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, group * queries, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, kv, group, queries, high) / math.sqrt(dim)
    length = s["lengths"][:, None, None]
    last = length - queries + torch.arange(queries, device=d)[None, :, None] if s["causal"] else length - 1
    keep = place <= last
    if s["window"]:
        keep = keep & (place > last - s["window"])
    keep = keep[:, None, None]
    scores = torch.where(keep, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(b, kv, group * queries, high), v.permute(0, 2, 1, 3).contiguous()).view(b, kv, group, queries, dim)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b * queries, heads, dim).to(s["q"].dtype)


# ----------------------------------------------------- the values in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()  # the sum is held in its own type
        y = h * s["weight"].double()
        top = y.abs().max(dim=1, keepdim=True).values
        scale = top / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS) / 127
        values = torch.round(y * 127 / top) * scale
        return {"values": values, "sum": None if s["residual"] is None else h, "scale": scale[:, 0]}
    if case["op"] == "matmul":
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=s["a"].device)
        wide = s["b"].double().t().contiguous()
        for i in range(0, case["m"], 1024):
            y[i:i + 1024] = torch.mm(s["a"][i:i + 1024].double(), wide) * torch.outer(s["a_scale"][i:i + 1024].double(), s["b_scale"].double())
        return y if s["bias"] is None else y + s["bias"].double()
    page = case["page"]
    if case["op"] == "cache":
        out = {}
        for x in ("k", "v"):
            new = s[x].double()
            top = new.abs().max(dim=2, keepdim=True).values
            y = torch.round(new * 127 / top) * (top / 127)
            for i in range(case["idle"]):  # what the cache held before
                place = torch.arange(case["first"], case["first"] + case["tokens"], device=y.device)
                p, r = s["table"][i][place // page].long(), place % page
                y[i * case["tokens"]:(i + 1) * case["tokens"]] = (s[x + "_codes"].transpose(1, 2)[p, r].double()
                                                                  * s[x + "_scale"].transpose(1, 2)[p, r].double()[..., None])
            out[x] = y
        return out
    queries, heads, kv, dim = (case[x] for x in ("queries", "heads", "kv_heads", "dim"))
    out = torch.zeros(case["seqs"] * queries, heads, dim, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(_lengths(case)):
        pages = s["table"][i, :-(-n // page)].long()
        # [pages, heads, page, dim] as [heads, tokens, dim]
        k, v = ((s[x + "_codes"][pages].double() * s[x + "_scale"][pages].double()[..., None]).transpose(0, 1).reshape(kv, -1, dim)[:, :n]
                for x in ("k", "v"))
        place = torch.arange(n, device=out.device)
        last = (n - queries + torch.arange(queries, device=out.device))[:, None] if case["causal"] else torch.full((queries, 1), n, device=out.device)
        mask = place[None] > last
        if case["window"]:
            mask |= place[None] <= last - case["window"]
        for h in range(heads):
            x = torch.mm(s["q"][i * queries:(i + 1) * queries, h].double(), k[h * kv // heads].t().contiguous()) * dim ** -0.5
            x = torch.softmax(x.masked_fill(mask, -math.inf), 1).nan_to_num(0.0)
            out[i * queries:(i + 1) * queries, h] = torch.mm(x, v[h * kv // heads].contiguous())
    return out
