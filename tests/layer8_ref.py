"""64-bit references of the norm, the 8-bit cache and the attention over it, on whatever device the inputs are."""

from __future__ import annotations

import torch

from tests.fp8_ref import E4M3, LEAST, U, half_step, power, round_e4m3


def pow2_scale(most):
    """The smallest power of two s with most <= 448 s."""
    m, e = torch.frexp(most / 448.0)
    return power(e - (m == 0.5).int())


# ---------------------------------------------------------------- norm


def norm(x, weight, residual, eps, pow2):
    """(quotients rounded to e4m3, scales, h, y), 64-bit, of finite rows [m, k]."""
    h = x.double() if residual is None else x.double() + residual.double()
    r = 1.0 / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + eps)
    g = h * weight.double()
    q, scales = [], []
    for part in g.split(128, dim=1):
        most = part.abs().amax(1, keepdim=True)
        top = (most * r).clamp(min=LEAST)
        if pow2:
            scale = pow2_scale(top)
            q.append(part * r / scale)
        else:
            scale = top / 448.0
            q.append(torch.where(top > LEAST, part * 448.0 / most, part * r * 448.0 / LEAST))
        scales.append(scale)
    return round_e4m3(torch.cat(q, 1)), torch.cat(scales, 1), h, g * r


# ---------------------------------------------------------------- cache


def sequences(table, lengths, starts, tokens, page):
    """(first token, new tokens, length, keys that have room) of each sequence, out-of-range values cut as documented."""
    room = table.shape[1] * page
    out = []
    largest = 0                                            # starts that decrease count as the largest before them
    for s, length in enumerate(lengths.tolist()):
        if starts is None:
            first, n = s, 1
        else:
            first = largest = max(largest, min(max(int(starts[s]), 0), tokens))
            n = max(min(int(starts[s + 1]), tokens) - first, 0)
        out.append((first, n, max(length, 0), min(max(length, 0), room)))
    return out


def append(k, v, cache, table, lengths, starts):
    """The four tensors after the write, in 64 bits; NaN codes are NaN."""
    out = [t.double().clone() for t in cache]
    pages, heads, page, dim = cache[0].shape
    for s, (first, n, length, end) in enumerate(sequences(table, lengths, starts, k.shape[0], page)):
        at = max(length - n, 0)
        while at < end:
            place, lo = divmod(at, page)
            hi = min(end - place * page, page)
            p = int(table[s, place])
            if 0 <= p < pages:
                token = first + at - (length - n)
                for i, new in ((0, k), (2, v)):
                    x = new[token:token + hi - lo].double().transpose(0, 1)                    # [heads, some, dim]
                    x = torch.where(x.isinf(), torch.nan, x)
                    scale = pow2_scale(x.nan_to_num(0.0).abs().amax((1, 2)).clamp(min=LEAST))
                    block = out[0][p] if i == 0 else out[2][p].transpose(1, 2)                 # [heads, page, dim]
                    if lo:
                        scale = torch.maximum(scale, out[i + 1][p])
                        block[:, :lo] = round_e4m3(block[:, :lo] * (out[i + 1][p] / scale)[:, None, None])
                    block[:, lo:hi] = round_e4m3(x / scale[:, None, None])
                    out[i + 1][p] = scale
            at = (place + 1) * page
    return out


# ---------------------------------------------------------------- attention


def attention(q, cache, table, lengths, starts=None, *, scale=None, window=None, sinks=None):
    """(out, its bound, lse, its bound, rows of sequences), 64-bit.

    The bound: a logit is a sum of dim exact products in fp32 and two more roundings; a weight's relative error is that
    of its logit, the exponential's, and its 16-bit form's, 2^-11 for a bf16 result and 2^-21 for an fp16 one (two
    parts); weights far below the largest of weight times scale w are cut at 2^-25 of 2^6 of it; sums are fp32."""
    tokens, heads, dim = q.shape
    pages, kv, page, _ = cache[0].shape
    group = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((tokens, heads, dim), dtype=torch.float64, device=q.device)
    tol, lse = torch.zeros_like(out), torch.full((tokens, heads), -torch.inf, dtype=torch.float64, device=q.device)
    lse_tol, mine = torch.zeros_like(lse), torch.zeros(tokens, dtype=torch.bool, device=q.device)
    weight_eps = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -21
    for s, (first, n, length, end) in enumerate(sequences(table, lengths, starts, tokens, page)):
        mine[first:first + n] = True
        if not n:
            continue
        ids = table[s, :-(-end // page)].long()
        there = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:end]
        ids = ids.clamp(0, pages - 1)
        i = torch.arange(length - n, length, device=q.device).view(-1, 1)
        j = torch.arange(end, device=q.device)
        seen = (j <= i) & there
        if window:
            seen &= j > i - window
        for h in range(heads):
            c = h // group
            kd = (cache[0].view(torch.uint8)[ids, c].view(E4M3).double() * cache[1][ids, c].double()[:, None, None])
            vs = cache[3][ids, c].double().repeat_interleave(page)[:end]
            vd = cache[2].view(torch.uint8)[ids, c].view(E4M3).double().transpose(1, 2).reshape(-1, dim)[:end]
            vd = vd * vs[:, None]
            kd = kd.reshape(-1, dim)[:end]
            x = q[first:first + n, h].double()
            logit = torch.where(seen, (x @ kd.t()) * scale, -torch.inf)
            size = torch.where(seen, (x.abs() @ kd.abs().t()) * abs(scale), 0.0)
            most = logit.amax(1, keepdim=True) if end else torch.full((n, 1), -torch.inf, device=q.device).double()
            if sinks is not None:
                most = torch.maximum(most, sinks[h].double())
            safe = torch.where(most == -torch.inf, 0.0, most)
            w = torch.exp(logit - safe)
            total = w.sum(1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks[h].double() - safe)
            some = torch.where(total > 0, total, 1.0)
            if vd.isnan().any():
                terms = torch.where(seen[:, :, None], w[:, :, None] * vd, 0.0)
                o, absolute = terms.sum(1), terms.abs().sum(1)
            else:
                o, absolute = w @ vd, w @ vd.abs()
            off = ((dim + 2) * U * size.amax(1, keepdim=True) if end else 0.0) + 4 * U * safe.abs() + 6 * U
            if sinks is not None:
                off = off + 4 * U * sinks[h].double().abs()
            eps = 2 * off + weight_eps + (end + 40) * U
            cut = 448 * 2.0 ** -31 * end * ((w * vs).amax(1, keepdim=True) if end else 0.0)
            at = slice(first, first + n)
            out[at, h] = o / some
            tol[at, h] = (absolute * eps + cut) / some + out[at, h].abs() * half_step(q.dtype) + 2.0 ** -24 * (
                q.dtype == torch.float16)
            lse[at, h] = (safe + torch.log(total))[:, 0]
            lse_tol[at, h] = (off + (end + 40) * U + 4 * U * lse[at, h:h + 1].nan_to_num(0.0, neginf=0.0).abs())[:, 0]
    return out, tol, lse, lse_tol, mine


def make_cache(gen, pages, kv, page, dim, octaves=2):
    """A cache whose every place holds a value, scales spread over powers of two."""
    dev = gen.device
    out = []
    for shape in ((pages, kv, page, dim), (pages, kv, dim, page)):
        x = torch.randn(shape, generator=gen, device=dev)
        s = torch.exp2(torch.randint(-octaves, octaves + 1, shape[:2], generator=gen, device=dev).float()) * 2.0 ** -7
        out += [(x * 128).clamp(-448, 448).to(E4M3), s]
    return out


def make_table(gen, lengths, page, spare=1):
    """Pages for each sequence in a random order, and how many there are; a row's other places name no page."""
    need = [-(-max(n, 0) // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=gen, device=gen.device).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), 1) + 1), -7, dtype=torch.int32, device=gen.device)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare
