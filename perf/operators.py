"""Workloads of the block-scaled 8-bit operators and the expert router: their plain forms beside the framework's calls.

Five kinds of work:

* ``quantize``: rows to e4m3 with an fp32 scale for each group of 128 values.
* ``gemm``: the product of such rows with an e4m3 matrix that has a scale for each 128x128 block.
* ``linear``: that matrix applied to 16-bit rows, which are quantized on the way.
* ``moe``: a whole routed-expert layer of such matrices for a few tokens (activations stay 16-bit).
* ``route``: the top-k of a router's logits, with the weights of the chosen experts.

Weights are normal values rounded to e4m3 under scales spread over a factor of four; activations are normal with
a few channels twenty times as large, as hidden states have them; logits are normal."""

from __future__ import annotations

import math

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST = E4M3_MAX * 2.0 ** -126       # a group's largest magnitude counts as this at least: its scale stays a normal number


def _quantize(name, rows, k, dtype="bf16", pow2=False):
    return {"name": name, "kind": "quantize", "rows": rows, "k": k, "dtype": dtype, "pow2": pow2}


def _gemm(name, rows, k, n, out="bf16"):
    return {"name": name, "kind": "gemm", "rows": rows, "k": k, "n": n, "out": out}


def _linear(name, rows, k, n, dtype="bf16"):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype}


def _moe(name, rows, *, hidden=4096, inter=2048, experts=256, topk=8, dtype="bf16", limit=10.0, share=1):
    return {"name": name, "kind": "moe", "rows": rows, "hidden": hidden, "inter": inter, "experts": experts,
            "topk": topk, "dtype": dtype, "limit": limit, "share": share}


def _route(name, rows, experts, topk, scoring, *, dtype="fp32", bias=False, scale=1.0):
    return {"name": name, "kind": "route", "rows": rows, "experts": experts, "topk": topk, "scoring": scoring,
            "dtype": dtype, "bias": bias, "scale": scale}


def listed():
    return [
        # a ragged decode batch's hidden state, quantized once for the matrices that read it
        _quantize("quantize 13 rows", 13, 4096),
        # a long prefill chunk with power-of-two scales
        _quantize("quantize 8000 rows pow2", 8000, 4096, "fp16", pow2=True),
        # two sequences decoding through one low-rank projection
        _gemm("gemm 2 rows", 2, 1536, 4096, out="fp32"),
        # a prefill chunk of 512 tokens on the square projection
        _gemm("gemm 512 rows", 512, 4096, 4096, out="fp16"),
        # a long ragged prefill chunk on the widest projection
        _gemm("gemm 4000 rows", 4000, 4096, 12288),
        # one sequence decoding on the square projection
        _linear("linear 1 row", 1, 4096, 4096),
        # a large decode batch, ragged
        _linear("linear 77 rows", 77, 4096, 4096, "fp16"),
        # one sequence decoding through the 256-expert layer
        _moe("moe 1 row", 1),
        # a full decode batch on it
        _moe("moe 16 rows", 16, dtype="fp16"),
        # a speculative batch on one of two expert-parallel ranks: half of the ids belong to the other
        _moe("moe 41 rows, half the experts", 41, share=2),
        # a decode batch through the 256-expert router
        _route("route 16 rows", 16, 256, 8, "softmax"),
        # a long prefill chunk with a selection bias
        _route("route 8000 rows biased", 8000, 256, 8, "sigmoid", bias=True, scale=2.5),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, step * round(v / step))))


def draw(rng):
    kind = rng.choice(("quantize", "gemm", "gemm", "linear", "moe", "moe", "route"))
    if kind == "quantize":
        c = _quantize("", _spread(rng, 1, 8000), _spread(rng, 16, 4096), rng.choice(("fp16", "bf16")),
                      rng.random() < 0.5)
    elif kind == "gemm":
        c = _gemm("", _spread(rng, 1, 4000), _spread(rng, 256, 4096, 16), _spread(rng, 64, 12288),
                  rng.choice(("fp16", "bf16", "fp32")))
    elif kind == "linear":
        c = _linear("", _spread(rng, 1, 1000), _spread(rng, 256, 4096, 16), _spread(rng, 64, 12288),
                    rng.choice(("fp16", "bf16")))
    elif kind == "moe":
        share = rng.choice((1, 1, 2))
        c = _moe("", _spread(rng, 1, 16 if share == 1 else 41), hidden=_spread(rng, 512, 4096, 128),
                 inter=_spread(rng, 128, 2048, 128), experts=_spread(rng, 8, 256, 2), topk=rng.randint(1, 8),
                 dtype=rng.choice(("fp16", "bf16")), limit=rng.choice((10.0, 0.0)), share=share)
    else:
        c = _route("", _spread(rng, 1, 8000), _spread(rng, 8, 512), rng.randint(1, 8),
                   rng.choice(("softmax", "sigmoid", "sqrtsoftplus")), dtype=rng.choice(("fp32", "bf16")),
                   bias=rng.random() < 0.5, scale=rng.choice((1.0, 2.5)))
    c.pop("name", None)
    return c


# ---------------------------------------------------------------- inputs


def _generator(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return torch.Generator(device=dev).manual_seed(int(seed))


def _activations(gen, rows, k, dtype):
    x = torch.randn((rows, k), generator=gen, device=gen.device)
    wide = torch.rand((k,), generator=gen, device=gen.device) < 0.005
    return (x * torch.where(wide, 20.0, 1.0)).to(DTYPE[dtype])


def _matrix(gen, k, *n):
    """An e4m3 matrix [*n, k] and its block scales; a product of k normal values has a variance near one."""
    dev = gen.device
    w = torch.empty((*n, k), dtype=E4M3, device=dev)
    for part in (w.flatten(0, -3) if w.dim() > 2 else w.unsqueeze(0)).split(16):
        part.copy_((torch.randn(part.shape, generator=gen, device=dev) * 100.0).clamp(-E4M3_MAX, E4M3_MAX))
    shape = (*n[:-1], -(-n[-1] // 128), -(-k // 128))
    scale = (torch.rand(shape, generator=gen, device=dev) * 1.5 + 0.5) / (100.0 * math.sqrt(k))
    return w, scale


def prepare(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "quantize":
        return {"case": case, "x": _activations(gen, case["rows"], case["k"], case["dtype"])}
    if kind == "gemm":
        x = _activations(gen, case["rows"], case["k"], "bf16")
        a, a_scale = _plain_quantize(x, False)
        w, w_scale = _matrix(gen, case["k"], case["n"])
        return {"case": case, "a": a, "a_scale": a_scale, "w": w, "w_scale": w_scale}
    if kind == "linear":
        w, w_scale = _matrix(gen, case["k"], case["n"])
        return {"case": case, "x": _activations(gen, case["rows"], case["k"], case["dtype"]), "w": w,
                "w_scale": w_scale}
    experts = case["experts"]
    logits = torch.randn((case["rows"], experts), generator=gen, device=gen.device)
    if kind == "route":
        bias = torch.randn((experts,), generator=gen, device=gen.device) * 0.1 if case["bias"] else None
        return {"case": case, "logits": logits.to(DTYPE[case["dtype"]]), "bias": bias}
    h, i, local = case["hidden"], case["inter"], experts // case["share"]
    w13, s13 = _matrix(gen, h, local, 2 * i)
    w2, s2 = _matrix(gen, i, local, h)
    x = torch.randn((case["rows"], h), generator=gen, device=gen.device).to(DTYPE[case["dtype"]])
    top = logits.topk(case["topk"], dim=1)
    emap = None
    if case["share"] > 1:        # this rank has every share-th expert
        g = torch.arange(experts, device=gen.device)
        emap = torch.where((g % case["share"] == 0) & (g // case["share"] < local), g // case["share"], -1)
    return {"case": case, "x": x, "w13": w13, "s13": s13, "w2": w2, "s2": s2, "ids": top.indices.to(torch.int32),
            "weights": torch.softmax(top.values, dim=1), "emap": emap}


# ---------------------------------------------------------------- the plain forms


def _plain_quantize(x, pow2):
    rows, k = x.shape
    groups = -(-k // 128)
    v = torch.nn.functional.pad(x.float(), (0, groups * 128 - k)).view(rows, groups, 128)
    most = v.abs().amax(dim=2).clamp(min=LEAST)
    if pow2:
        mantissa, exponent = torch.frexp(most / E4M3_MAX)
        scale = ((exponent - (mantissa == 0.5).int() + 127) << 23).view(torch.float32)
        q = v / scale.unsqueeze(2)
    else:
        scale = most / E4M3_MAX
        q = v * E4M3_MAX / most.unsqueeze(2)
    return q.view(rows, groups * 128)[:, :k].to(E4M3), scale


def _grow(scale, rows, k):
    """Block scales [..., rows/128, k/128] as one value for each element [..., rows, k]."""
    return scale.repeat_interleave(128, dim=-2)[..., :rows, :].repeat_interleave(128, dim=-1)[..., :k]


def _plain_gemm(a, a_scale, w, w_scale, dtype):
    n, k = w.shape
    a = a.float() * a_scale.repeat_interleave(128, dim=1)[:, :k]
    return (a @ (w.float() * _grow(w_scale, n, k)).t()).to(dtype)


def _plain_moe(s):
    c, x = s["case"], s["x"]
    ids = s["ids"].long() if s["emap"] is None else s["emap"][s["ids"].long()]
    active = torch.unique(ids)
    active = active[active >= 0]
    take = lambda w: w.view(torch.uint8)[active].view(E4M3).float()  # noqa: E731
    w13 = take(s["w13"]) * _grow(s["s13"][active], 2 * c["inter"], c["hidden"])
    g, u = (x.float() @ w13.transpose(1, 2)).split(c["inter"], dim=2)
    if c["limit"]:
        g, u = g.clamp(max=c["limit"]), u.clamp(-c["limit"], c["limit"])
    del w13
    w2 = take(s["w2"]) * _grow(s["s2"][active], c["hidden"], c["inter"])
    d = (g / (1.0 + torch.exp(-g)) * u) @ w2.transpose(1, 2)
    share = ((ids.unsqueeze(2) == active) * s["weights"].unsqueeze(2)).sum(dim=1)        # [rows, active]
    return (d * share.t().unsqueeze(2)).sum(dim=0).to(x.dtype)


def _plain_route(logits, topk, scoring, bias, scale):
    v = logits.double()
    fit = ~torch.isnan(v) & (v != -math.inf)
    if scoring == "softmax":
        e = torch.where(fit, torch.exp(v - v.masked_fill(~fit, -math.inf).amax(dim=1, keepdim=True)), 0.0)
        score = e / e.sum(dim=1, keepdim=True)
    elif scoring == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-v))
    else:
        score = torch.sqrt(v.clamp(min=0.0) + torch.log1p(torch.exp(-v.abs())))
    rank = (v if bias is None else score + bias.double()).masked_fill(~fit, -math.inf)
    ids = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :topk]
    there = fit.gather(1, ids)
    chosen = torch.where(there, score.gather(1, ids), 0.0)
    total = chosen.sum(dim=1, keepdim=True)
    weights = torch.where(total > 0, chosen / total, 0.0) * scale
    return torch.where(there, ids, -1).to(torch.int32), weights.float()


# ---------------------------------------------------------------- run


def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        from dsv4_carve_amd import ops

        if kind == "quantize":
            return ops.fp8_quantize(state["x"], pow2=c["pow2"])
        if kind == "gemm":
            return ops.fp8_gemm(state["a"], state["a_scale"], state["w"], state["w_scale"], out_dtype=DTYPE[c["out"]])
        if kind == "linear":
            return ops.fp8_linear(state["x"], state["w"], state["w_scale"])
        if kind == "moe":
            return ops.fp8_moe(state["x"], state["w13"], state["s13"], state["w2"], state["s2"], state["ids"],
                               state["weights"], swiglu_limit=c["limit"] or None, expert_map=state["emap"])
        return ops.moe_route(state["logits"], c["topk"], scoring=c["scoring"], bias=state["bias"], scale=c["scale"])
    if kind == "quantize":
        return _plain_quantize(state["x"], c["pow2"])
    if kind == "gemm":
        return _plain_gemm(state["a"], state["a_scale"], state["w"], state["w_scale"], DTYPE[c["out"]])
    if kind == "linear":
        return _plain_gemm(*_plain_quantize(state["x"], False), state["w"], state["w_scale"], state["x"].dtype)
    if kind == "moe":
        return _plain_moe(state)
    return _plain_route(state["logits"], c["topk"], c["scoring"], state["bias"], c["scale"])


# ---------------------------------------------------------------- work


def work(case):
    kind, rows = case["kind"], case["rows"]
    blocks = lambda n, k: -(-n // 128) * -(-k // 128)  # noqa: E731
    if kind == "quantize":
        values = rows * case["k"]
        return {"bytes": 3.0 * values + 4.0 * rows * -(-case["k"] // 128), "flops": 3.0 * values}
    if kind in ("gemm", "linear"):
        k, n = case["k"], case["n"]
        matrix = n * k + 4.0 * blocks(n, k)
        if kind == "linear":
            return {"bytes": matrix + 2.0 * rows * (k + n), "flops": 2.0 * rows * k * n}
        return {"bytes": matrix + rows * (k + 4.0 * -(-k // 128)) + (4.0 if case["out"] == "fp32" else 2.0) * rows * n,
                "flops": 2.0 * rows * k * n}
    e, topk = case["experts"], case["topk"]
    if kind == "route":
        return {"bytes": rows * (e * (4.0 if case["dtype"] == "fp32" else 2.0) + 8.0 * topk), "flops": 2.0 * rows * e}
    h, i = case["hidden"], case["inter"]
    local = e // case["share"]
    active = local * (1.0 - (1.0 - topk / e) ** rows)
    expert = 3.0 * h * i + 4.0 * (blocks(2 * i, h) + blocks(h, i))
    return {"bytes": active * expert + 4.0 * rows * h + 8.0 * rows * topk,
            "flops": 6.0 * rows * topk * local / e * h * i}


# ---------------------------------------------------------------- the 64-bit results


def _e4m3_64(v):
    """Each 64-bit value's nearest e4m3 value, ties to the even significand; |v| <= 448."""
    exponent = torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent.long()       # v < 2 ** exponent
    step = ((exponent - 4 + 1023) << 52).view(torch.float64)
    return torch.round(v / step) * step


def _quantize64(x, pow2):
    values, scales = [], []
    for part in x.double().split(128, dim=1):
        most = part.abs().max(dim=1, keepdim=True).values.clamp(min=LEAST)
        if pow2:
            scale = torch.full_like(most, 2.0 ** -126)
            for _ in range(256):
                scale = torch.where(scale * E4M3_MAX < most, scale * 2.0, scale)
            values.append(_e4m3_64(part / scale))
        else:
            scale = most / E4M3_MAX
            values.append(_e4m3_64(part * E4M3_MAX / most))
        scales.append(scale)
    return torch.cat(values, dim=1), torch.cat(scales, dim=1)


def _gemm64(a, a_scale, w, w_scale):
    out = torch.zeros((a.shape[0], w.shape[0]), dtype=torch.float64, device=a.device)
    for b in range(a_scale.shape[1]):
        at = slice(128 * b, 128 * (b + 1))
        per_row = w_scale[:, b].double().repeat_interleave(128)[:w.shape[0]]
        out += (a[:, at].double() * a_scale[:, b:b + 1].double()) @ w[:, at].double().t() * per_row
    return out


def _moe64(s):
    c, x = s["case"], s["x"].double()
    out = torch.zeros_like(x)
    ones = torch.ones((x.shape[0], 1), dtype=torch.float64, device=x.device)

    def times(v, w, scale):
        return _gemm64(v, ones.expand(-1, scale.shape[1])[:v.shape[0]], w, scale)

    ids, emap = s["ids"].tolist(), None if s["emap"] is None else s["emap"].tolist()
    where = {}
    for r, row in enumerate(ids):
        for j, e in enumerate(row):
            e = e if emap is None else emap[e]
            if e >= 0:
                where.setdefault(e, []).append((r, j))
    for e, slots in where.items():
        rows = torch.tensor([r for r, _ in slots], device=x.device)
        cols = torch.tensor([j for _, j in slots], device=x.device)
        h = times(x[rows], s["w13"][e], s["s13"][e])
        g, u = h[:, :c["inter"]], h[:, c["inter"]:]
        if c["limit"]:
            g, u = torch.minimum(g, torch.full_like(g, c["limit"])), u.clamp(-c["limit"], c["limit"])
        d = times(g * torch.sigmoid(g) * u, s["w2"][e], s["s2"][e])
        out.index_add_(0, rows, d * s["weights"][rows, cols].double().unsqueeze(1))
    return out


def _route64(logits, topk, scoring, bias, scale):
    v = logits.double()
    score = {"softmax": lambda: torch.softmax(v, dim=1), "sigmoid": lambda: torch.sigmoid(v),
             "sqrtsoftplus": lambda: torch.logaddexp(v, torch.zeros_like(v)).sqrt()}[scoring]()
    key = v if bias is None else score + bias.double()
    ids = torch.empty((v.shape[0], topk), dtype=torch.int32, device=v.device)
    left = key.clone()
    for j in range(topk):
        best = left.max(dim=1, keepdim=True).values
        at = (left == best).to(torch.int8).argmax(dim=1)
        ids[:, j] = at
        left.scatter_(1, at.unsqueeze(1), -math.inf)
    chosen = score.gather(1, ids.long())
    return ids, chosen / chosen.sum(dim=1, keepdim=True) * scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _quantize64(s["x"], case["pow2"])
    if kind == "gemm":
        return _gemm64(s["a"], s["a_scale"], s["w"], s["w_scale"])
    if kind == "linear":
        return _gemm64(*_quantize64(s["x"], False), s["w"], s["w_scale"])
    if kind == "moe":
        return _moe64(s)
    return _route64(s["logits"], case["topk"], case["scoring"], s["bias"], case["scale"])
