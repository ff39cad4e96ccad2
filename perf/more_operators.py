"""Workloads of the operators around an 8-bit decoder layer's products: their plain forms beside the framework's calls.

Three kinds of work:

* ``norm``: the residual's addition and the root-mean-square norm, with an e4m3 result that has an fp32 scale for each
  group of 128 values, as the block-scaled products read it.
* ``append``: new keys and values into a paged cache of e4m3 values with one power-of-two scale for each page and head.
  A page that has tokens already keeps the larger of its scale and the new tokens'; where that is larger than before,
  its old values are rounded to it.
* ``attention``: causal attention of the last tokens of each sequence over that cache, with grouped heads.

A cache is four tensors: k e4m3 [pages, kv_heads, page, dim] and v e4m3 [pages, kv_heads, dim, page] with k_scale and
v_scale fp32 [pages, kv_heads].  A sequence's pages are a row of its table; its length counts the new tokens."""

from __future__ import annotations

import math

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST = E4M3_MAX * 2.0 ** -126       # a group's largest magnitude counts as this at least: its scale stays a normal number
EPS = 1e-6
GOLDEN = 0.6180339887498949


def _norm(name, rows, k, dtype="bf16", *, residual=None, weight="bf16", pow2=False, normed=False):
    return {"name": name, "kind": "norm", "rows": rows, "k": k, "dtype": dtype, "residual": residual or "", "weight": weight,
            "pow2": pow2, "normed": normed}


def _append(name, seqs, queries, length, *, kv_heads=8, dim=128, page=64, dtype="bf16", ragged=True):
    return {"name": name, "kind": "append", "seqs": seqs, "queries": queries, "length": length, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def _attention(name, seqs, queries, length, *, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", window=0,
               sinks=False, lse=False, ragged=True):
    return {"name": name, "kind": "attention", "seqs": seqs, "queries": queries, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "lse": lse,
            "ragged": ragged}


def listed():
    return [
        # one sequence decoding: its hidden state in front of the next product
        _norm("norm 1 row", 1, 4096, residual="bf16"),
        # a ragged batch's low-rank projection, for a product and for 16-bit readers
        _norm("norm 333 rows of 1536", 333, 1536, "fp16", weight="fp32", pow2=True, normed=True),
        # a long prefill chunk
        _norm("norm 8000 rows", 8000, 4096, residual="bf16"),
        # a decode batch's new tokens
        _append("append 13 tokens", 13, 1, 5000, page=16),
        # a prefill chunk of several sequences, some with a begun page
        _append("append 4 chunks", 4, 2000, 6000, dtype="fp16"),
        # one sequence decoding, a short context
        _attention("attention 1 token", 1, 1, 1000, page=16),
        # a full decode batch of ragged contexts
        _attention("attention 64 tokens", 64, 1, 8192),
        # one sequence decoding on a long context, its part of a split context (the sums' logarithms are wanted)
        _attention("attention 1 token of 131072", 1, 1, 131072, heads=64, page=128, dtype="fp16", lse=True),
        # drafted tokens of a batch in a layer with a window and sinks, small heads
        _attention("attention 16 x 5 drafted", 16, 5, 6000, heads=64, dim=64, page=32, dtype="fp16", window=1024, sinks=True),
        # wide heads that share one cache head
        _attention("attention 24 tokens wide", 24, 1, 3500, heads=16, kv_heads=1, dim=256, page=32),
        # a prefill chunk behind a long context
        _attention("attention chunk of 512", 1, 512, 16384),
        # whole ragged prompts
        _attention("attention 4 prompts", 4, 3000, 3000, kv_heads=4, dtype="fp16", page=16),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, step * round(v / step))))


def draw(rng):
    kind = rng.choice(("norm", "append", "attention", "attention"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "norm":
        c = _norm("", _spread(rng, 1, 8000), _spread(rng, 64, 4096, rng.choice((1, 16, 128))),
                  rng.choice(("fp16", "bf16", "fp32")) if rng.random() < 0.3 else dtype,
                  weight=rng.choice((dtype, "fp32")), pow2=rng.random() < 0.5, normed=rng.random() < 0.3)
        c["residual"] = rng.choice(("", c["dtype"], "fp32" if c["dtype"] != "fp16" else c["dtype"]))
        c["rows"] = min(c["rows"], 8000 if c["dtype"] != "fp32" else 3000)
    else:
        heads = rng.choice((1, 2, 4, 8))
        dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
        page = rng.choice((16, 32, 64, 128))
        if kind == "append":
            seqs = _spread(rng, 1, 64)
            queries = 1 if rng.random() < 0.4 else _spread(rng, 1, max(2, 8000 // seqs))
            c = _append("", seqs, queries, queries + _spread(rng, 1, 4000), kv_heads=heads,
                        dim=min(dim, 128) if queries > 100 else dim, page=page, dtype=dtype, ragged=rng.random() < 0.8)
        else:
            group = rng.choice((1, 2, 3, 4, 5, 8, 16))
            if rng.random() < 0.6:
                seqs = _spread(rng, 1, 64)
                queries = rng.choice((1, 1, 1, 2, 4, 7))
                most = 131072 * 8 * 128 // (seqs * heads * dim)
                length = queries + _spread(rng, 1, min(131072, max(64, most)))
            else:
                seqs = _spread(rng, 1, 6)
                queries = _spread(rng, 16, max(17, 2000 // seqs))
                most = 50_000_000 * 32 * 128 // (seqs * queries * heads * group * dim)      # as many products as the longest prompts
                length = queries + _spread(rng, 1, min(16384, max(16, most // 8)))
            c = _attention("", seqs, queries, length, heads=heads * group, kv_heads=heads, dim=dim, page=page, dtype=dtype,
                           window=rng.choice((0, 0, 128, 1000)), sinks=rng.random() < 0.3, lse=rng.random() < 0.3,
                           ragged=rng.random() < 0.8)
    c.pop("name", None)
    return c


# ---------------------------------------------------------------- inputs


def _shapes(case):
    """Each sequence's (new tokens, length): the largest first, then down to a tenth if ragged."""
    out = []
    for i in range(case["seqs"]):
        part = 1.0 - 0.9 * ((i * GOLDEN) % 1.0) if case["ragged"] else 1.0
        n = max(1, round(case["queries"] * part))
        out.append((n, max(n, round(case["length"] * part))))
    return out


def _generator(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return torch.Generator(device=dev).manual_seed(int(seed))


def _channels(gen, x, share, size):
    """x with a few of its last dimension's channels larger, as hidden states and keys have them."""
    wide = torch.rand(x.shape[1:], generator=gen, device=gen.device) < share
    return x * torch.where(wide, size, 1.0)


def _cache(gen, pages, heads, page, dim):
    """A cache full of tokens, each page's values under the smallest power of two that holds them."""
    out = []
    for shape in ((pages, heads, page, dim), (pages, heads, dim, page)):
        codes = torch.empty(shape, dtype=E4M3, device=gen.device)
        scale = torch.empty(shape[:2], device=gen.device)
        for at in range(0, pages, 512):
            part = torch.randn((min(512, pages - at), *shape[1:]), generator=gen, device=gen.device)
            part = part * torch.exp2(torch.randint(-2, 2, (*part.shape[:2], 1, 1), generator=gen, device=gen.device).float())
            s = _pow2(part.abs().amax(dim=(2, 3)))
            codes[at:at + 512] = (part / s[..., None, None]).to(E4M3)
            scale[at:at + 512] = s
        out += [codes, scale]
    return tuple(out)


def prepare(case, seed):
    gen = _generator(seed)
    dev = gen.device
    if case["kind"] == "norm":
        rows, k = case["rows"], case["k"]
        x = _channels(gen, torch.randn((rows, k), generator=gen, device=dev), 0.005, 20.0).to(DTYPE[case["dtype"]])
        residual = None
        if case["residual"]:
            r = _channels(gen, torch.randn((rows, k), generator=gen, device=dev) * 4.0, 0.002, 50.0)
            residual = r.to(DTYPE[case["residual"]])
        weight = (torch.rand((k,), generator=gen, device=dev) * 1.5 + 0.25).to(DTYPE[case["weight"]])
        return {"case": case, "x": x, "residual": residual, "weight": weight}
    shapes = _shapes(case)
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-length // page) for _, length in shapes]
    pages = sum(need)
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros((len(shapes), max(need)), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    counts = [n for n, _ in shapes]
    tokens = sum(counts)
    starts = None
    if max(counts) > 1:
        starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=dev)
    state = {"case": case, "shapes": shapes, "table": table, "starts": starts, "cache": _cache(gen, pages, heads, page, dim),
             "lengths": torch.tensor([length for _, length in shapes], dtype=torch.int32, device=dev)}
    if case["kind"] == "append":
        k = _channels(gen, torch.randn((tokens, heads, dim), generator=gen, device=dev), 0.02, 8.0)
        v = torch.randn((tokens, heads, dim), generator=gen, device=dev)
        state |= {"k": k.to(DTYPE[case["dtype"]]), "v": v.to(DTYPE[case["dtype"]])}
    else:
        q = torch.randn((tokens, case["heads"], dim), generator=gen, device=dev) * 2.0
        state |= {"q": q.to(DTYPE[case["dtype"]]), "sinks": None}
        if case["sinks"]:
            state["sinks"] = torch.randn((case["heads"],), generator=gen, device=dev) + 3.0
    return state


# ---------------------------------------------------------------- the plain forms


def _pow2(most):
    """The smallest power of two that is not below most / 448."""
    mantissa, exponent = torch.frexp(most.float().clamp(min=LEAST) / E4M3_MAX)
    return ((exponent - (mantissa == 0.5).int() + 127) << 23).view(torch.float32)


def _round_e4m3(v):
    """64-bit values, |v| <= 448, as the nearest e4m3 values, ties to the even significand."""
    exponent = torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent.long()       # v < 2 ** exponent
    step = ((exponent - 4 + 1023) << 52).view(torch.float64)
    return (torch.round(v / step) * step).to(torch.float32).to(E4M3)


def _plain_norm(s):
    c, x = s["case"], s["x"]
    rows, k = x.shape
    h = x.double() if s["residual"] is None else x.double() + s["residual"].double()
    r = torch.rsqrt((h * h).sum(dim=1, keepdim=True) / k + EPS)
    g = h * s["weight"].double()
    groups = -(-k // 128)
    v = torch.nn.functional.pad(g, (0, groups * 128 - k)).view(rows, groups, 128)
    most = v.abs().amax(dim=2)
    top = (most * r).clamp(min=LEAST)
    if c["pow2"]:
        mantissa, exponent = torch.frexp(top / E4M3_MAX)
        scale = ((exponent - (mantissa == 0.5).int() + 127) << 23).view(torch.float32)
        q = v * r.unsqueeze(2) / scale.unsqueeze(2)
    else:                              # the row's factor is in a value and in the group's largest: without it, ties stay ties
        scale = (top / E4M3_MAX).float()
        q = torch.where((top > LEAST).unsqueeze(2), v * E4M3_MAX / most.unsqueeze(2), v * r.unsqueeze(2) * E4M3_MAX / LEAST)
    out = [_round_e4m3(q).view(rows, groups * 128)[:, :k].contiguous(), scale]
    if s["residual"] is not None:
        out.append(h.to(s["residual"].dtype))
    if c["normed"]:
        out.append((g * r).to(x.dtype))
    return out


def _plain_append(s):
    c, dev = s["case"], s["k"].device
    page, pages = c["page"], s["cache"][0].shape[0]
    seq = torch.tensor([i for i, (n, _) in enumerate(s["shapes"]) for _ in range(n)], device=dev)
    pos = torch.tensor([length - n + j for n, length in s["shapes"] for j in range(n)], device=dev)
    at, slot = s["table"].long()[seq, pos // page], pos % page
    begun = [(i, length - n) for i, (n, length) in enumerate(s["shapes"]) if (length - n) % page]
    for which, new in ((0, s["k"].float()), (2, s["v"].float())):
        codes, scale = s["cache"][which], s["cache"][which + 1]
        most = torch.zeros((pages, c["kv_heads"]), device=dev)
        most.index_reduce_(0, at, new.abs().amax(dim=2), "amax")
        touched = torch.zeros((pages, 1), dtype=torch.bool, device=dev)
        touched[at] = True
        fresh = torch.where(touched, _pow2(most), scale)
        if begun:
            rows = torch.tensor([i for i, _ in begun], device=dev)
            base = torch.tensor([b for _, b in begun], device=dev)
            p = s["table"].long()[rows, base // page]
            fresh[p] = torch.maximum(fresh[p], scale[p])
            old = codes.view(torch.uint8)[p].view(E4M3)
            there = torch.arange(page, device=dev) < (base % page).view(-1, 1)
            there = there[:, None, :, None] if which == 0 else there[:, None, None, :]
            moved = (old.float() * (scale[p] / fresh[p])[..., None, None]).to(E4M3)
            codes.view(torch.uint8)[p] = torch.where(there, moved.view(torch.uint8), old.view(torch.uint8))
        scale.copy_(fresh)
        made = (new / fresh[at].unsqueeze(2)).to(E4M3).view(torch.uint8)
        if which == 0:
            codes.view(torch.uint8)[at, :, slot] = made
        else:
            codes.view(torch.uint8)[at, :, :, slot] = made
    return s["cache"]


def _plain_attention(s):
    c, q = s["case"], s["q"]
    heads, dim, kv, page = c["heads"], c["dim"], c["kv_heads"], c["page"]
    group = heads // kv
    k_codes, k_scale, v_codes, v_scale = s["cache"]
    out = torch.empty_like(q)
    lse = torch.empty((q.shape[0], heads), device=q.device)
    sinks = None if s["sinks"] is None else s["sinks"].view(kv, 1, group, 1)
    at = 0
    for i, (n, length) in enumerate(s["shapes"]):
        first = max(0, length - n + 1 - c["window"]) // page if c["window"] else 0
        p = s["table"][i, first:-(-length // page)].long()
        keys = torch.arange(first * page, length, device=q.device)
        k = k_codes.view(torch.uint8)[p].view(E4M3).float() * k_scale[p][..., None, None]
        v = v_codes.view(torch.uint8)[p].view(E4M3).float() * v_scale[p][..., None, None]
        k = k.permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :len(keys)]
        v = v.permute(1, 0, 3, 2).reshape(kv, -1, dim)[:, :len(keys)]
        rows = q[at:at + n].float().view(n, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, n * group, dim)
        score = (rows @ k.transpose(1, 2)).mul_(1.0 / math.sqrt(dim)).view(kv, n, group, -1)
        query = torch.arange(length - n, length, device=q.device).view(n, 1)
        hidden = keys > query
        if c["window"]:
            hidden |= keys <= query - c["window"]
        score.masked_fill_(hidden.view(1, n, 1, -1), -math.inf)
        most = score.amax(dim=3, keepdim=True)
        if sinks is not None:
            most = torch.maximum(most, sinks)
        weight = score.sub_(most).exp_()
        total = weight.sum(dim=3, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sinks - most)
        o = (weight.view(kv, n * group, -1) @ v).view(kv, n, group, dim) / total
        out[at:at + n] = o.permute(1, 0, 2, 3).reshape(n, heads, dim).to(q.dtype)
        lse[at:at + n] = (most + torch.log(total)).squeeze(3).permute(1, 0, 2).reshape(n, heads)
        at += n
    return (out, lse) if c["lse"] else out


# ---------------------------------------------------------------- run


def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        from dsv4_carve_amd import ops

        if kind == "norm":
            made = ops.fp8_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS, pow2=c["pow2"],
                                normed_dtype=state["x"].dtype if c["normed"] else None)
            return [t for t in made if t is not None]
        cache = ops.Fp8Cache(*state["cache"])
        if kind == "append":
            return tuple(ops.fp8_cache_append(state["k"], state["v"], cache, state["table"], state["lengths"],
                                              state["starts"]))
        return ops.fp8_attention(state["q"], cache, state["table"], state["lengths"], state["starts"],
                                 window=c["window"] or None, sinks=state["sinks"], return_lse=c["lse"])
    if kind == "norm":
        return _plain_norm(state)
    if kind == "append":
        return tuple(_plain_append(state))
    return _plain_attention(state)


# ---------------------------------------------------------------- work


def work(case):
    size = {"": 0.0, "fp16": 2.0, "bf16": 2.0, "fp32": 4.0}
    if case["kind"] == "norm":
        rows, k, x = case["rows"], case["k"], size[case["dtype"]]
        each = x + 2.0 * size[case["residual"]] + 1.0 + (x if case["normed"] else 0.0)
        return {"bytes": rows * k * each + 4.0 * rows * -(-k // 128) + size[case["weight"]] * k, "flops": 8.0 * rows * k}
    shapes = _shapes(case)
    tokens, kv, dim, page = sum(n for n, _ in shapes), case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        begun = sum(1 for n, length in shapes if (length - n) % page)
        touched = sum(-(-length // page) - (length - n) // page for n, length in shapes)
        return {"bytes": 2.0 * kv * (tokens * dim * 3.0 + 4.0 * touched + 4.0 * begun), "flops": 4.0 * tokens * kv * dim}
    keys = pairs = 0
    for n, length in shapes:
        low = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        keys += length - low
        if case["window"]:
            pairs += sum(min(case["window"], length - n + j + 1) for j in range(n))
        else:
            pairs += n * (length - n) + n * (n + 1) // 2
    return {"bytes": 2.0 * keys * kv * (dim + 4.0 / page) + 4.0 * tokens * case["heads"] * dim,
            "flops": 4.0 * pairs * case["heads"] * dim}


# ---------------------------------------------------------------- the 64-bit results


def _grid(dev):
    """The 127 e4m3 values from 0 to 448, in 64 bits."""
    small = [m * 2.0 ** -9 for m in range(8)]
    return torch.tensor(small + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119], dtype=torch.float64,
                        device=dev)


def _nearest(v):
    """Each value's nearest on the e4m3 grid; one in the middle of two goes to the even one."""
    grid = _grid(v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    a = v.abs().contiguous()
    low = torch.bucketize(a, middle)
    high = torch.bucketize(a, middle, right=True)
    return torch.copysign(grid[torch.where(low % 2 == 0, low, high)], v)


def _least_power(most):
    """The smallest 2**e >= most / 448, by trial."""
    scale = torch.exp2(torch.floor(torch.log2(most / E4M3_MAX)) - 2)
    for _ in range(4):
        scale = torch.where(scale * E4M3_MAX < most, scale * 2.0, scale)
    return scale


def _norm64(s):
    c = s["case"]
    h = s["x"].to(torch.float64)
    if s["residual"] is not None:
        h = h + s["residual"].to(torch.float64)
    size = torch.sqrt(torch.mean(torch.square(h), dim=1, keepdim=True) + EPS)
    y = h * s["weight"].to(torch.float64)
    values, scales = [], []
    for part in y.split(128, dim=1):
        most = torch.max(torch.abs(part), dim=1, keepdim=True).values
        if c["pow2"]:
            scale = _least_power(torch.clamp(most / size, min=LEAST))
            values.append(_nearest(part / size / scale))
        else:
            least = LEAST * size                                   # the smallest that a group's largest counts as, before the division
            scale = torch.maximum(most, least) / size / E4M3_MAX
            values.append(_nearest(part * E4M3_MAX / torch.maximum(most, least)))
        scales.append(scale)
    y = y / size
    out = [torch.cat(values, dim=1), torch.cat(scales, dim=1)]
    if s["residual"] is not None:
        out.append(h)
    if c["normed"]:
        out.append(y)
    return out


def _append64(s):
    c, page = s["case"], s["case"]["page"]
    out = [t.double() for t in s["cache"]]
    table, at = s["table"].tolist(), 0
    for i, (n, length) in enumerate(s["shapes"]):
        here, base = 0, length - n
        while here < n:
            slot = (base + here) % page
            some = min(n - here, page - slot)
            p = table[i][(base + here) // page]
            for which, new in ((0, s["k"]), (2, s["v"])):
                x = new[at + here:at + here + some].double()                                   # [some, heads, dim]
                scale = _least_power(x.abs().amax(dim=(0, 2)).clamp(min=LEAST))
                block = out[which][p] if which == 0 else out[which][p].transpose(1, 2)         # [heads, page, dim]
                if slot:
                    scale = torch.maximum(scale, out[which + 1][p])
                    block[:, :slot] = _nearest(block[:, :slot] * (out[which + 1][p] / scale).view(-1, 1, 1))
                block[:, slot:slot + some] = _nearest(x.transpose(0, 1) / scale.view(-1, 1, 1))
                out[which + 1][p] = scale
            here += some
        at += n
    return tuple(out)


def _attention64(s):
    c, q = s["case"], s["q"]
    kv, dim, page = c["kv_heads"], c["dim"], c["page"]
    group = c["heads"] // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    at = 0
    for i, (n, length) in enumerate(s["shapes"]):
        p = s["table"][i, :-(-length // page)].long()
        where = torch.arange(length - n, length, device=q.device).view(-1, 1) - torch.arange(length, device=q.device)
        seen = (where >= 0) & (where < (c["window"] or length + 1))                            # [n, length]
        for h in range(kv):
            k = (s["cache"][0][:, h].view(torch.uint8)[p].view(E4M3).double() * s["cache"][1][p, h].double().view(-1, 1, 1))
            v = (s["cache"][2][:, h].view(torch.uint8)[p].view(E4M3).double() * s["cache"][3][p, h].double().view(-1, 1, 1))
            k = k.reshape(-1, dim)[:length]
            v = v.transpose(1, 2).reshape(-1, dim)[:length]
            for j in range(h * group, (h + 1) * group):
                logits = torch.where(seen, q[at:at + n, j].double() @ k.t() / math.sqrt(dim), -math.inf)
                most = logits.max(dim=1).values
                if s["sinks"] is not None:
                    most = torch.clamp(most, min=float(s["sinks"][j]))
                e = torch.exp(logits - most.view(-1, 1))
                total = e.sum(dim=1)
                if s["sinks"] is not None:
                    total = total + torch.exp(float(s["sinks"][j]) - most)
                out[at:at + n, j] = e @ v / total.view(-1, 1)
                lse[at:at + n, j] = most + torch.log(total)
        at += n
    return (out, lse) if c["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _norm64(s)
    if case["kind"] == "append":
        return _append64(s)
    return _attention64(s)
