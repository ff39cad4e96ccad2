"""64-bit references of the block-scaled 8-bit operators and the router, on whatever device the inputs are."""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn
LEAST = 448.0 * 2.0 ** -126
U = 2.0 ** -23                       # one step of an fp32 sum, however the matrix unit rounds it


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def power(e):
    """2 ** e in 64 bits, exactly (exp2 and ldexp are rounded on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def round_e4m3(v):
    """Nearest e4m3 value of each |v| <= 448 (64-bit), ties to the even significand."""
    step = power(torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(v / step) * step


def quantize(x, pow2=False):
    """(unrounded quotients, scales) in 64 bits; NaN does not count for a group's largest magnitude."""
    k = x.shape[-1]
    quot, scales = [], []
    for part in x.double().reshape(-1, k).split(128, dim=1):
        most = part.abs().nan_to_num(0.0, posinf=float("inf")).amax(dim=1, keepdim=True).clamp(min=LEAST)
        if pow2:
            m, e = torch.frexp(most / 448.0)
            scale = torch.where(most.isinf(), most, power((e - (m == 0.5).int()).clamp(max=1000)))
            quot.append(part / scale)
        else:
            scale = most / 448.0
            quot.append(part * 448.0 / most)
        scales.append(scale)
    return torch.cat(quot, 1).reshape(x.shape), torch.cat(scales, 1).reshape(*x.shape[:-1], -1)


def grow(scale, n, k):
    return scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def weight(w, w_scale):
    return w.double() * grow(w_scale, *w.shape[-2:])


def rows(a, a_scale):
    return a.double() * a_scale.double().repeat_interleave(128, -1)[..., :a.shape[-1]]


def steps(k):
    """Roundings on the way of one product into its sum: a block's 128, the blocks', the joining of waves, the scales'."""
    return 128 + k // 128 + 1 + 16 + 4


def cut(a, w):
    """What the 8-bit matrix instruction may leave out of a @ w^T: it cuts each product to a multiple of 2^-13 of the
    largest power of two of its eight, so up to seven times that for each group of eight values of k (a cut result of
    eight may also round once more to a step as large)."""
    total = torch.zeros((a.shape[0], w.shape[0]), dtype=torch.float64, device=a.device)
    for at in range(0, a.shape[1], 8):
        most = torch.zeros_like(total)
        for i in range(at, min(at + 8, a.shape[1])):
            most = torch.maximum(most, a[:, i:i + 1].abs() * w[:, i].abs())
        total += most
    return total * 8 * 2.0 ** -13


def gemm(a, a_scale, w, w_scale, dtype):
    """(result, how far an fp32-accumulated product rounded once to `dtype` may be from it).  For 16 bits the bound has
    room for the 8-bit matrix instruction, which no kernel uses: tests of a 16-bit result against the rounded fp32 one
    go without it."""
    x, m = rows(a, a_scale), weight(w, w_scale)
    ref = x @ m.t()
    tol = (x.abs() @ m.abs().t()) * steps(a.shape[1]) * U + ref.abs() * half_step(dtype) + 2.0 ** -24 * (
        dtype is torch.float16)
    return ref, tol + cut(x, m) if dtype is not torch.float32 else tol


def moe(x, w13, s13, w2, s2, ids, wts, limit, emap, dtype):
    """(result, bound) of the layer with an activation of 16 significant bits, row by row."""
    xd, inter = x.double(), w2.shape[2]
    out, tol = torch.zeros_like(xd), torch.zeros_like(xd)
    lim = float("inf") if limit is None else limit
    for r in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[r, j])
            if emap is not None:
                e = int(emap[e]) if 0 <= e < emap.numel() else -1
            if not 0 <= e < w13.shape[0]:
                continue
            m13, m2 = weight(w13[e], s13[e]), weight(w2[e], s2[e])
            h, h_tol = m13 @ xd[r], (m13.abs() @ xd[r].abs()) * steps(x.shape[1]) * U
            g, u = h[:inter].clamp(max=lim), h[inter:].clamp(-lim, lim)
            act = g * torch.sigmoid(g) * u
            # |d silu| <= 1.1; the exponential, quotient and product are within 8 steps
            a_tol = 1.1 * u.abs() * h_tol[:inter] + (g * torch.sigmoid(g)).abs() * h_tol[inter:] + act.abs() * 8 * U
            a_tol = a_tol + act.abs() * 2.0 ** -17
            wt = abs(float(wts[r, j]))
            out[r] += float(wts[r, j]) * (m2 @ act)
            n = (steps(inter) + 128) * max(1, ids.numel()) ** 0.5 + ids.numel()
            tol[r] += wt * (m2.abs() @ (a_tol + act.abs() * n * U))
    return out, tol + out.abs() * half_step(dtype) + 2.0 ** -24 * (dtype is torch.float16)


def route(logits, topk, scoring, bias, renormalize, scale):
    v = logits.double()
    fit = ~torch.isnan(v) & (v != -torch.inf)
    if scoring == "softmax":
        e = torch.where(fit, torch.exp(v - torch.where(fit, v, -torch.inf).amax(1, keepdim=True)), 0.0)
        score = e / e.sum(1, keepdim=True)
    elif scoring == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-v))
    else:
        score = torch.sqrt(v.clamp(min=0) + torch.log1p(torch.exp(-v.abs())))
    key = v if bias is None else score + bias.double()
    key = torch.where(fit & ~torch.isnan(key), key, -torch.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True)
    ids = torch.where(order.values[:, :topk] != -torch.inf, order.indices[:, :topk], -1)
    s = torch.where(ids >= 0, score.gather(1, ids.clamp(min=0)), 0.0)
    if renormalize:
        total = s.sum(1, keepdim=True)
        s = torch.where(total != 0, s / total, 0.0)
    return ids, s * scale


def matrix(gen, *shape):
    """Random e4m3 [.., n, k] over the type's whole finite range, with block scales."""
    dev = gen.device
    w = (torch.randn(shape, generator=gen, device=dev) * torch.exp2(
        torch.randint(-8, 8, shape, generator=gen, device=dev).float())).clamp(-448, 448).to(E4M3)
    s = torch.rand((*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128)), generator=gen, device=dev)
    return w, (s * 1.5 + 0.5) * 2.0 ** -6
