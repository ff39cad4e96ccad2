"""The block-scaled 8-bit operators and the router on the GPU, against 64-bit references."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import ops
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def gen_of(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def normal(gen, *shape, dtype=torch.bfloat16, spread=True):
    x = torch.randn(shape, generator=gen, device=gen.device)
    if spread:
        x = x * torch.exp2(torch.randint(-6, 7, shape, generator=gen, device=gen.device).float())
    return x.to(dtype)


def within(got, ref, tol, what=""):
    d = (got.double() - ref).abs()
    assert torch.isfinite(got.double()).all(), what
    worst = (d - tol).max()
    assert worst <= 0, f"{what}: {float(d.max()):.3g} off, {float(worst):.3g} over the bound"


# ---------------------------------------------------------------- quantization


def check_quantized(x, q, scale, pow2):
    quot, want = R.quantize(x, pow2)
    assert q.dtype == R.E4M3 and q.shape == x.shape and scale.shape == want.shape
    assert torch.equal(scale, want.float())
    rounded = R.round_e4m3(quot)
    if x.dtype == torch.float32 and not pow2:
        # 448 x and the quotient are rounded once each, 2^-24 of their value; the rounded quotient can lie on the other
        # side of a border only if the exact one is nearer to it than that, and then both neighbours are equally far but
        # for twice the error.  How many values are that near depends on the input alone, so no share is asked for.
        assert ((q.double() - quot).abs() <= (rounded - quot).abs() + 2.0 ** -21 * quot.abs()).all()
    else:
        assert torch.equal(q.double(), rounded)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (3, 127), (5, 128), (7, 129), (2, 144), (33, 1536), (257, 512), (1, 16384)])
def test_quantize(dev, dtype, pow2, rows, k):
    x = normal(gen_of(dev, rows + k), rows, k, dtype=dtype)
    check_quantized(x, *ops.fp8_quantize(x, pow2=pow2), pow2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [256, 250])
def test_quantize_values_on_rounding_borders(dev, dtype, k):
    """Every quotient of few-bit values: ties are common, and all groups' largest values are different."""
    most = torch.arange(1, 129, device=dev).float().reshape(-1, 1) / 64
    x = most * (torch.randint(0, 897, (128, k), generator=gen_of(dev, 5), device=dev) / 896.0)
    x = x.to(dtype)
    x[:, 0::128] = most.to(dtype)
    for pow2 in (False, True):
        check_quantized(x, *ops.fp8_quantize(x, pow2=pow2), pow2)


@pytest.mark.parametrize("k", [256, 200])
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_extremes(dev, k, pow2):
    """Zero and subnormal groups, the types' largest values."""
    for dtype in TYPES:
        f = torch.finfo(dtype)
        for v in (0.0, f.tiny, f.smallest_normal * 2.0 ** -5, f.max, -f.max):
            x = torch.zeros((2, k), dtype=dtype, device=dev)
            x[0, 3:9] = v
            x[1, :] = v
            q, scale = ops.fp8_quantize(x, pow2=pow2)
            assert torch.isfinite(q.float()).all() and (scale > 0).all() and torch.isfinite(scale).all()
            check_quantized(x, q, scale, pow2)


@pytest.mark.parametrize("k", [384, 380])
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_nan_and_infinity(dev, k, pow2):
    x = normal(gen_of(dev, 1), 2, k)
    x[0, 5], x[0, 300] = float("nan"), float("-inf")
    q, scale = ops.fp8_quantize(x, pow2=pow2)
    clean = x.clone()
    clean[0, 5] = 0
    want_q, want_s = ops.fp8_quantize(clean[:, :256].contiguous(), pow2=pow2)
    keep = torch.ones(256, dtype=torch.bool, device=dev)
    keep[5] = False
    assert torch.isnan(q[0, 5].float()) and torch.equal(q[:, :256].float()[:, keep], want_q.float()[:, keep])
    assert torch.equal(scale[:, :2], want_s) and torch.isinf(scale[0, 2]) and torch.isfinite(scale[1, 2])
    assert torch.isnan(q[0, 300].float()) and (q[0, 256:300].float() == 0).all() and (q[0, 301:].float() == 0).all()


def test_quantize_empty_leading_dims_and_unaligned(dev):
    q, s = ops.fp8_quantize(torch.empty((0, 256), dtype=torch.bfloat16, device=dev))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    x = normal(gen_of(dev, 2), 2, 3, 256)
    q, s = ops.fp8_quantize(x)
    q2, s2 = ops.fp8_quantize(x.view(6, 256))
    assert s.shape == (2, 3, 2) and torch.equal(q.view(6, 256).float(), q2.float()) and torch.equal(s.view(6, 2), s2)
    flat = normal(gen_of(dev, 3), 1 + 6 * 256)[1:].view(6, 256)          # two bytes off a 16-byte border
    check_quantized(flat, *ops.fp8_quantize(flat), False)


@pytest.mark.parametrize("rows,k", [((1 << 26) + 6, 1), ((1 << 25) + 9, 130), ((1 << 29) + 40, 16)])
def test_quantize_more_rows_than_a_launch_takes(dev, rows, k):
    """Rows on either side of a launch's last one, and the last rows, are as in a call of their own."""
    gen = gen_of(dev, k)
    x = torch.empty((rows, k), dtype=torch.int16, device=dev)
    for part in x.split(1 << 24):
        part.random_(0, 0x7f00, generator=gen)
    x = x.view(torch.bfloat16)
    q, s = ops.fp8_quantize(x)
    a_launch = ((1 << 24) - 1) * (32 if k % 16 == 0 else 4) // s.shape[1]
    assert rows > a_launch
    for at in (0, a_launch - 5, a_launch, rows - 37):
        at = min(at, rows - 37)
        want_q, want_s = ops.fp8_quantize(x[at:at + 37].clone())
        assert torch.equal(q[at:at + 37].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[at:at + 37], want_s)


# ---------------------------------------------------------------- product


def rows_of(gen, m, k):
    return ops.fp8_quantize(normal(gen, m, k))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (1, 128, 16), (2, 144, 17), (5, 1040, 130), (16, 4096, 256), (17, 512, 64),
                                   (33, 272, 500), (64, 2048, 384), (65, 640, 100), (130, 1536, 260), (257, 256, 1024),
                                   (300, 1168, 513), (513, 384, 768)])
def test_gemm(dev, m, k, n, out):
    gen = gen_of(dev, m * 7 + k + n)
    a, sa = rows_of(gen, m, k)
    w, sw = R.matrix(gen, n, k)
    within(ops.fp8_gemm(a, sa, w, sw, out_dtype=out), *R.gemm(a, sa, w, sw, out), f"{m}x{k}x{n}")


@pytest.mark.parametrize("m", [1, 2, 4, 8, 9, 31, 47, 96, 128, 200, 256, 384, 640, 1024, 1100])
def test_gemm_row_counts(dev, m):
    """Every variant that the row count chooses, on one matrix: a row does not depend on the others beside it beyond rounding."""
    gen = gen_of(dev, m)
    a, sa = rows_of(gen, m, 1024)
    w, sw = R.matrix(gen, 640, 1024)
    within(ops.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32), *R.gemm(a, sa, w, sw, torch.float32), str(m))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(5, 4084), (16, 4090), (15, 12200), (33, 4084), (50, 4090), (120, 4084), (250, 4090),
                                 (500, 4084), (500, 4090), (1000, 4090), (2000, 8180), (4000, 4090)])
def test_gemm_tile_shapes(dev, m, n, out):
    """Rows and columns that every tile shape is chosen for, ragged in both, and a last block of 16."""
    gen = gen_of(dev, m + n)
    a, sa = rows_of(gen, m, 272)
    w, sw = R.matrix(gen, n, 272)
    within(ops.fp8_gemm(a, sa, w, sw, out_dtype=out), *R.gemm(a, sa, w, sw, out), f"{m}x{n}")


@pytest.mark.parametrize("m,k,n", [(3, 400, 40), (40, 400, 200), (300, 400, 330), (600, 1040, 600)])
def test_gemm_writes_its_rows_only_and_keeps_nan_in_them(dev, m, k, n):
    """Rows around c stay; a NaN in one row of a, or of w, reaches that row, or column, only; bytes past k are not used."""
    gen = gen_of(dev, 4)
    a, sa = rows_of(gen, m, k)
    w, sw = R.matrix(gen, n, k)
    plain = ops.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32)
    a.view(torch.uint8)[m - 2, 7] = 0x7f
    w.view(torch.uint8)[n - 3, k - 1] = 0xff
    buf = torch.full((m + 4, n), 7.0, device=dev)
    pad = 2 * n * 4 % 16 == 0
    c = ops.fp8_gemm_into(a, sa, w, sw, buf[2:m + 2] if pad else torch.empty((m, n), device=dev))
    assert (buf[:2] == 7).all() and (buf[m + 2:] == 7).all()
    bad = torch.zeros((m, n), dtype=torch.bool, device=dev)
    bad[m - 2], bad[:, n - 3] = True, True
    assert torch.equal(torch.isnan(c), bad) and torch.equal(c[~bad], plain[~bad])


@pytest.mark.parametrize("m,k,n", [(5, 4368, 330), (20, 9552, 500), (50, 9552, 4084), (60, 4784, 5002), (120, 9232, 4084),
                                   (250, 4368, 4090), (120, 4784, 8000), (500, 4368, 4084), (1000, 2320, 4090),
                                   (4000, 2320, 4090)])
def test_gemm_long_rows_of_every_tile(dev, m, k, n):
    """More than two groups of staged scales for every tile shape, their number no multiple of a group, a ragged last
    block, scales far apart: the fp32 result against the reference, a 16-bit one against its rounding."""
    gen = gen_of(dev, m + k)
    a, sa = rows_of(gen, m, k)
    w, sw = R.matrix(gen, n, k)
    sw = sw * torch.exp2(torch.randint(-6, 7, sw.shape, generator=gen, device=dev).float())
    c = ops.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32)
    ref, tol = R.gemm(a, sa, w, sw, torch.float32)
    within(c, ref, tol, f"{m}x{k}x{n}")
    # Partial sums of terms of either sign are no larger than the whole in the mean, and their roundings (one step at
    # most each) no more alike than the terms: the 2-norm grows with the root of their number.
    assert torch.linalg.norm(c.double() - ref) <= torch.linalg.norm(ref) * R.steps(k) ** 0.5 * R.U
    for dtype in (torch.float16, torch.bfloat16):
        s = 2.0 ** -8 if dtype is torch.float16 else 1.0          # into fp16's range
        assert torch.equal(ops.fp8_gemm(a, sa * s, w, sw, out_dtype=dtype), (c * s).to(dtype))


@pytest.mark.parametrize("m", [1, 3, 8, 9, 16, 40, 77, 300])
@pytest.mark.parametrize("wide", [1.0, 20.0])
def test_16_bit_results_are_the_fp32_sum_rounded_once(dev, m, wide):
    """Whatever the row count, with and without channels that stand out."""
    gen = gen_of(dev, m)
    x = torch.randn((m, 1024), generator=gen, device=dev)
    x[:, torch.rand(1024, generator=gen, device=dev) < 0.005] *= wide
    x = x.to(torch.bfloat16)
    w, sw = R.matrix(gen, 512, 1024)
    sw = sw * 2.0 ** -8
    a, sa = ops.fp8_quantize(x)
    for dtype in (torch.float16, torch.bfloat16):
        assert torch.equal(ops.fp8_gemm(a, sa, w, sw, out_dtype=dtype),
                           ops.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32).to(dtype))
        assert torch.equal(ops.fp8_linear(x, w, sw, out_dtype=dtype), ops.fp8_linear(x, w, sw, out_dtype=torch.float32).to(dtype))


@pytest.mark.parametrize("m", [3, 20, 50, 100, 300])
@pytest.mark.parametrize("out", TYPES)
def test_gemm_infinite_scales(dev, m, out):
    """An infinite scale makes its products infinite, none of them a NaN, wherever the blocks of k end."""
    gen = gen_of(dev, m)
    for k in (272, 640):
        a, w = (torch.randint(0x30, 0x40, s, generator=gen, device=dev, dtype=torch.uint8).view(R.E4M3) for s in ((m, k), (200, k)))
        sa, sw = torch.ones((m, -(-k // 128)), device=dev), torch.ones((2, -(-k // 128)), device=dev)
        good = ops.fp8_gemm(a, sa, w, sw, out_dtype=out)
        sa[1, -1], sw[1, -1] = torch.inf, torch.inf
        c = ops.fp8_gemm(a, sa, w, sw, out_dtype=out)
        assert (c[1] == torch.inf).all() and (c[:, 128:] == torch.inf).all()
        keep = [r for r in range(m) if r != 1]
        assert torch.equal(c[keep, :128], good[keep, :128])


def test_gemm_is_repeatable(dev):
    gen = gen_of(dev, 9)
    for m in (1, 20, 100, 700):
        a, sa = rows_of(gen, m, 2048)
        w, sw = R.matrix(gen, 512, 2048)
        first = ops.fp8_gemm(a, sa, w, sw)
        assert all(torch.equal(first, ops.fp8_gemm(a, sa, w, sw)) for _ in range(3))


def test_gemm_empty(dev):
    gen = gen_of(dev, 1)
    w, sw = R.matrix(gen, 48, 256)
    a, sa = ops.fp8_quantize(torch.empty((0, 256), dtype=torch.float16, device=dev))
    assert ops.fp8_gemm(a, sa, w, sw).shape == (0, 48)
    assert ops.fp8_linear(torch.empty((2, 0, 256), dtype=torch.float16, device=dev), w, sw).shape == (2, 0, 48)


@pytest.mark.parametrize("m,k,n", [(300, 1 << 17, 33000), (70000, 256, 33000)])
def test_gemm_past_32_bit_offsets(dev, m, k, n):
    """A matrix of more than 2^32 bytes, an output of more than 2^31 values; the last corner against the reference."""
    gen = gen_of(dev, 2)
    a, sa = rows_of(gen, m, k)
    w = torch.randint(0, 127, (n, k), generator=gen, device=dev, dtype=torch.uint8).view(R.E4M3)
    sw = torch.rand((-(-n // 128), k // 128), generator=gen, device=dev) * 2.0 ** -6
    c = ops.fp8_gemm(a, sa, w, sw)
    last = slice((n - 1) // 128 * 128, n)
    within(c[-40:, last], *R.gemm(a[-40:], sa[-40:], w[last], sw[-1:], torch.bfloat16), "corner")


@pytest.mark.parametrize("out", [torch.float16, torch.float32])
def test_gemm_longest_rows(dev, out):
    """Rows too long for a tile's 32-bit offsets; no value is negative, so that the sum's size is its own."""
    gen = gen_of(dev, 8)
    m, k, n = 17, (1 << 22) + 16, 20
    a, w = (torch.randint(0, 0x40, shape, generator=gen, device=dev, dtype=torch.uint8).view(R.E4M3)
            for shape in ((m, k), (n, k)))
    sa = torch.rand((m, -(-k // 128)), generator=gen, device=dev)
    sw = torch.rand((1, -(-k // 128)), generator=gen, device=dev) * 2.0 ** -10
    c = ops.fp8_gemm(a, sa, w, sw, out_dtype=out)
    ref = torch.zeros((m, n), dtype=torch.float64, device=dev)
    for at in range(0, k, 1 << 20):
        part = slice(at, min(at + (1 << 20), k))
        b = slice(at // 128, -(-part.stop // 128))
        ref += R.rows(a[:, part], sa[:, b]) @ R.weight(w[:, part], sw[:, b]).t()
    # an eighth of the blocks is a wave's sum, and eight of them are joined
    within(c, ref, ref * (R.steps(k // 8) * R.U + R.half_step(out)), "longest")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 13, 16, 17, 40, 300])
@pytest.mark.parametrize("k,n", [(1536, 384), (272, 70)])
def test_linear_is_quantize_then_gemm(dev, dtype, rows, k, n):
    gen = gen_of(dev, rows)
    x = normal(gen, rows, k, dtype=dtype)
    w, sw = R.matrix(gen, n, k)
    q, s = ops.fp8_quantize(x)
    for out in (None, torch.float32):
        ref, tol = R.gemm(q, s, w, sw, out or dtype)
        within(ops.fp8_linear(x, w, sw, out_dtype=out), ref, tol, f"{rows} {out}")
    x3 = x.view(1, rows, k)
    assert torch.equal(ops.fp8_linear(x3, w, sw)[0], ops.fp8_linear(x, w, sw))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 7168), (2, 7168), (1, 12288), (2, 12288), (1, 4224), (1, 8208)])
def test_linear_long_rows(dev, dtype, rows, k):
    """More blocks than a wave has on their way at once."""
    gen = gen_of(dev, rows + k)
    x = normal(gen, rows, k, dtype=dtype)
    w, sw = R.matrix(gen, 84, k)
    sw = sw * torch.exp2(torch.randint(-3, 4, sw.shape, generator=gen, device=dev).float()) * 2.0 ** -6
    q, s = ops.fp8_quantize(x)
    y = ops.fp8_linear(x, w, sw, out_dtype=torch.float32)
    ref, tol = R.gemm(q, s, w, sw, torch.float32)
    within(y, ref, tol, f"{rows}x{k}")
    assert torch.equal(ops.fp8_linear(x, w, sw, out_dtype=torch.bfloat16), y.to(torch.bfloat16))


@pytest.mark.parametrize("rows", [1, 4, 12])
def test_linear_nan_infinity_and_zero_rows(dev, rows):
    gen = gen_of(dev, 6)
    x = normal(gen, rows + 2, 512)
    w, sw = R.matrix(gen, 96, 512)
    good = ops.fp8_linear(x, w, sw, out_dtype=torch.float32)
    x[0, 3], x[1, 400] = float("nan"), float("inf")
    x[rows + 1] = 0
    y = ops.fp8_linear(x, w, sw, out_dtype=torch.float32)
    assert torch.isnan(y[:2]).all() and (y[rows + 1] == 0).all()
    assert torch.equal(y[2:rows + 1], good[2:rows + 1])


# ---------------------------------------------------------------- router


def check_route(logits, topk, scoring, bias=None, renormalize=True, scale=1.0, ids_dtype=torch.int32):
    ids, wts = ops.moe_route(logits, topk, scoring=scoring, bias=bias, renormalize=renormalize, scale=scale,
                             ids_dtype=ids_dtype)
    want_ids, want = R.route(logits, topk, scoring, bias, renormalize, scale)
    assert ids.dtype == ids_dtype and torch.equal(ids.long(), want_ids)
    # the softmax's sum over a row is fp32: some roundings of each lane and six joins; all else is 64-bit, rounded once
    rel = 2.0 ** -24 + (64 * 2.0 ** -24 if scoring == "softmax" and not renormalize else 0.0)
    assert ((wts.double() - want).abs() <= want.abs() * rel * 1.001 + 1e-300 + 2.0 ** -149).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("rows,experts,topk", [(1, 1, 1), (3, 5, 5), (2, 64, 8), (17, 65, 6), (16, 256, 8), (1000, 256, 8),
                                               (9, 384, 64), (5, 512, 10), (4, 1000, 16), (3, 2048, 9)])
def test_route(dev, scoring, biased, rows, experts, topk):
    gen = gen_of(dev, rows + experts)
    bias = torch.randn(experts, generator=gen, device=dev) * 0.1 if biased else None
    for dtype in TYPES:        # 16-bit logits bring ties
        logits = (torch.randn((rows, experts), generator=gen, device=dev) * 2).to(dtype)
        check_route(logits, topk, scoring, bias)
        check_route(logits, topk, scoring, bias, renormalize=False, scale=2.5, ids_dtype=torch.int64)


@pytest.mark.parametrize("rows,experts,topk", [(40, 64, 8), (40, 300, 8), (200, 2048, 16)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_softmax_over_the_row_is_64_bit(dev, rows, experts, topk, biased):
    gen = gen_of(dev, experts)
    bias = torch.randn(experts, generator=gen, device=dev) * 0.1 if biased else None
    logits = torch.randn((rows, experts), generator=gen, device=dev) * 3
    ids, wts = ops.moe_route(logits, topk, bias=bias, renormalize=False)
    want_ids, want = R.route(logits, topk, "softmax", bias, False, 1.0)
    assert torch.equal(ids.long(), want_ids)
    assert ((wts.double() - want).abs() <= want * 2.0 ** -24 * 1.001 + 2.0 ** -150).all()     # one rounding


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_route_ties_and_near_ties(dev, scoring):
    """Equal logits go by index; scores that fp32 cannot tell apart go by their exact order."""
    gen = gen_of(dev, 3)
    check_route(torch.zeros((4, 300), device=dev), 9, scoring)
    check_route(torch.zeros((4, 300), device=dev), 9, scoring, torch.zeros(300, device=dev))
    near = 1.0 + torch.randint(0, 64, (200, 256), generator=gen, device=dev).float() * 2.0 ** -22
    bias = torch.randint(0, 3, (256,), generator=gen, device=dev).float() * 2.0 ** -23
    check_route(near, 8, scoring, bias)
    far = torch.randn((64, 256), generator=gen, device=dev) * 3 + 30          # sigmoids next to one
    check_route(far, 8, scoring, torch.randn(256, generator=gen, device=dev) * 1e-7)


def test_route_scores_that_a_bias_takes_back(dev):
    """A key's error is that of its score, which may be far above the key."""
    gen = gen_of(dev, 11)
    logits = torch.randn((500, 6), generator=gen, device=dev)
    logits[:, ::2] = 1e6 + torch.randint(-32, 32, (500, 3), generator=gen, device=dev) * 0.0625
    score = torch.sqrt(logits.double().clamp(min=0) + torch.log1p(torch.exp(-logits.double().abs())))
    for shift in (0.0, 0.5):
        for row in range(0, 500, 10):
            bias = (shift - score[row]).float()             # this row's keys lie within fp32's error of each other
            check_route(logits[row:row + 10].contiguous(), 2, "sqrtsoftplus", bias)
            check_route(logits[row:row + 10].contiguous(), 6, "sqrtsoftplus", bias + torch.randint(
                -8, 8, (6,), generator=gen, device=dev) * 2.0 ** -16)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_route_more_rows_than_a_launch_takes(dev, ids_dtype):
    rows = (1 << 26) + 5
    logits = torch.empty((rows, 2), dtype=torch.bfloat16, device=dev).normal_(generator=gen_of(dev, 7))
    ids, wts = ops.moe_route(logits, 1, scoring="sigmoid", renormalize=False, ids_dtype=ids_dtype)
    assert torch.equal(ids[:, 0], (logits[:, 1] > logits[:, 0]).to(ids_dtype))
    for at in (0, 4 * ((1 << 24) - 1) - 9, rows - 20):
        want = R.route(logits[at:at + 20], 1, "sigmoid", None, False, 1.0)[1]
        assert ((wts[at:at + 20].double() - want).abs() <= want * 2.0 ** -24 * 1.001).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_masked_and_extreme_logits(dev, scoring, biased):
    gen = gen_of(dev, 8)
    logits = torch.randn((6, 100), generator=gen, device=dev)
    logits[0] = -torch.inf                                   # nothing to choose
    logits[1, 3:] = -torch.inf                               # fewer than k
    logits[2, ::2] = torch.nan
    logits[3] = torch.finfo(torch.float32).min               # the type's lowest value is a logit as any other
    logits[3, 40] = 1.0
    logits[4] *= 40.0                                        # scores far below fp32's range
    bias = torch.randn(100, generator=gen, device=dev) * 0.1 if biased else None
    for renormalize in (True, False):
        ids, wts = ops.moe_route(logits, 8, scoring=scoring, bias=bias, renormalize=renormalize)
        assert torch.isfinite(wts).all() and (ids[0] == -1).all() and (wts[0] == 0).all()
        assert (ids[1, 3:] == -1).all() and sorted(ids[1, :3].tolist()) == [0, 1, 2]
        assert (ids[2] % 2 == 1).all()
        want_ids, _ = R.route(logits, 8, scoring, bias, renormalize, 1.0)
        assert torch.equal(ids.long()[:5], want_ids[:5])
        check_route(logits[5:].contiguous(), 8, scoring, bias, renormalize)
    assert ops.moe_route(torch.empty((0, 8), device=dev), 2)[0].shape == (0, 2)


# ---------------------------------------------------------------- expert layer


def layer(gen, experts, hidden, inter, size=2.0 ** -6):
    """With size 1 the gate is of the order of one, and the output too; with less the fp16 values are subnormal."""
    w13, s13 = R.matrix(gen, experts, 2 * inter, hidden)
    w2, s2 = R.matrix(gen, experts, hidden, inter)
    return w13, s13 * (size / hidden ** 0.5), w2, s2 * (size / inter ** 0.5)


def routed(gen, rows, experts, topk, dtype=torch.int32):
    logits = torch.randn((rows, experts), generator=gen, device=gen.device)
    return ops.moe_route(logits, topk, ids_dtype=dtype)


def check_moe(x, mats, ids, wts, limit=None, emap=None, out=None):
    y = ops.fp8_moe(x, *mats, ids, wts, swiglu_limit=limit, expert_map=emap, out=out)
    ref, tol = R.moe(x, *mats, ids.cpu(), wts.cpu(), limit, None if emap is None else emap.cpu(), y.dtype)
    within(y, ref, tol, "moe")
    # in the 2-norm: the output's half step (2^-25 where fp16 is subnormal) and little else
    low = ref.numel() ** 0.5 * 2.0 ** -25 if y.dtype is torch.float16 else 0.0
    norm = torch.linalg.norm
    assert norm(y.double() - ref) <= norm(ref) * (R.half_step(y.dtype) + 2.0 ** -16) + low
    return y


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("limit", [None, 0.5])
@pytest.mark.parametrize("rows,experts,topk,hidden,inter", [(1, 1, 1, 128, 128), (1, 8, 8, 512, 256), (2, 4, 3, 256, 384),
                                                            (13, 16, 4, 1024, 128), (16, 6, 2, 384, 512), (17, 40, 6, 256, 256),
                                                            (32, 3, 1, 128, 640), (33, 64, 8, 256, 128), (64, 5, 3, 256, 256),
                                                            (64, 70, 16, 128, 128)])
def test_moe(dev, dtype, limit, rows, experts, topk, hidden, inter):
    gen = gen_of(dev, rows + experts)
    mats = layer(gen, experts, hidden, inter)
    x = normal(gen, rows, hidden, dtype=dtype, spread=False)
    ids, wts = routed(gen, rows, experts, min(topk, experts))
    check_moe(x, mats, ids, wts, limit)
    mats = (mats[0], mats[1] * 64, mats[2], mats[3] * 64)
    check_moe(x, mats, ids, wts, limit)
    check_moe(x, mats, ids.long(), wts.to(torch.bfloat16), limit, out=torch.empty(x.shape, dtype=torch.float32, device=dev))


def test_moe_skipped_repeated_and_mapped_ids(dev):
    gen = gen_of(dev, 11)
    mats = layer(gen, 6, 256, 256)
    x = normal(gen, 20, 256, spread=False)
    ids, wts = routed(gen, 20, 6, 4)
    ids[0] = -1                                             # a row without an expert
    ids[1, 2:] = 6                                          # outside
    ids[2] = 3                                              # one expert in every slot
    ids[3, 3] = ids[3, 0]
    ids[7:, 1] = 2                                          # an expert of many rows
    wts[4, 1] = 0.0
    y = check_moe(x, mats, ids, wts)
    assert (y[0] == 0).all()
    emap = torch.tensor([-1, 4, 0, 99, -7, 1, 2, 5, 3], device=dev)
    g = torch.randint(-2, 12, (20, 4), generator=gen, device=dev)
    check_moe(x, mats, g, wts, 2.0, emap)
    none = torch.full((20, 4), -1, dtype=torch.int32, device=dev)
    assert (ops.fp8_moe(x, *mats, none, wts) == 0).all()
    assert ops.fp8_moe(x[:0], *mats, none[:0], wts[:0]).shape == (0, 256)


@pytest.mark.parametrize("ids", [[3, 3, 0, -1, 7, 3], [-1, -1, 5], [9, 5000, -7], [2], list(range(16))])
@pytest.mark.parametrize("mapped", [False, True])
def test_moe_one_row(dev, ids, mapped):
    """A single token: an expert named twice, none at all, ids out of range, every slot that there may be."""
    gen = gen_of(dev, 18)
    mats = layer(gen, 8, 256, 384, size=1.0)
    emap = torch.tensor([4, -1, 0, 7, 7, 2], device=dev) if mapped else None
    wts = torch.rand((1, len(ids)), generator=gen, device=dev)
    y = check_moe(normal(gen, 1, 256, spread=False), mats, torch.tensor([ids], device=dev, dtype=torch.int32), wts, emap=emap)
    if ids[0] == 9:
        assert (y == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_moe_small_and_large_inputs(dev, dtype):
    """Inputs in fp16's subnormal range, and activations past fp16's largest value."""
    gen = gen_of(dev, 17)
    mats = layer(gen, 8, 256, 256, size=1.0)
    x = normal(gen, 6, 256, dtype=torch.float32, spread=False)
    ids, wts = routed(gen, 6, 8, 2)
    out = torch.empty((6, 256), dtype=torch.float32, device=dev)
    check_moe((x * 2.0 ** -19).to(dtype), mats, ids, wts, out=out)
    check_moe((x * 64).to(dtype), (mats[0], mats[1] * 64, mats[2], mats[3]), ids, wts, out=out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,experts,topk", [(1, 4, 3), (5, 16, 2), (20, 3, 2), (40, 64, 2), (64, 4, 3)])
def test_moe_activation_is_fp32(dev, dtype, rows, experts, topk):
    """One input and one value of each down row other than zero: the output is a sum of the activations themselves."""
    gen = gen_of(dev, rows)
    n = 256
    w13, s13 = R.matrix(gen, experts, 2 * n, n)
    w13 = (w13.float() / 448).clamp(-1, 1).to(R.E4M3)
    s13 = s13 * 64
    w2 = torch.eye(n, device=dev).expand(experts, n, n).contiguous().to(R.E4M3)
    s2 = torch.ones((experts, 2, 2), device=dev)
    x = torch.zeros((rows, n), dtype=dtype, device=dev)
    at = torch.randint(0, n, (rows,), generator=gen, device=dev)
    x[torch.arange(rows, device=dev), at] = (torch.rand(rows, generator=gen, device=dev) * 4 + 0.5).to(dtype)
    ids = torch.rand((rows, experts), generator=gen, device=dev).argsort(1)[:, :topk].contiguous()
    wts = torch.ones((rows, topk), device=dev)
    out = ops.fp8_moe(x, w13, s13, w2, s2, ids, wts, swiglu_limit=8.0, out=torch.empty((rows, n), device=dev))
    ref, tol = torch.zeros((rows, n), dtype=torch.float64, device=dev), 0.0
    full = R.weight(w13, s13)
    for j in range(topk):
        h = (full[ids[:, j]] @ x.double().unsqueeze(2)).squeeze(2)
        g, u = h[:, :n].clamp(max=8.0), h[:, n:].clamp(-8.0, 8.0)
        act = g * torch.sigmoid(g) * u
        ref += act
        # half steps: a rounding each of g (which silu's slope makes 1 + |g| of at most), u, 1 + e^-g, the quotient, the
        # product, the scaled sum and the joined one, four of the exponential
        tol = tol + act.abs() * (11 + g.abs()) * 2.0 ** -24
    within(out, ref, tol + 2.0 ** -126, "act")


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_moe_infinite_activations(dev, rows):
    """An activation past fp32 is infinite, and so is what positive weights make of it: no NaN, and no other row's."""
    gen = gen_of(dev, rows)
    w13 = torch.randint(0x30, 0x40, (3, 512, 128), generator=gen, device=dev, dtype=torch.uint8).view(R.E4M3)
    w2 = torch.randint(0x30, 0x40, (3, 128, 256), generator=gen, device=dev, dtype=torch.uint8).view(R.E4M3)
    s13, s2 = torch.ones((3, 4, 1), device=dev), torch.ones((3, 1, 2), device=dev) * 2.0 ** -20
    x = torch.rand((rows, 128), generator=gen, device=dev).to(torch.bfloat16)
    ids = torch.arange(rows, device=dev).reshape(-1, 1) % 3
    want = ops.fp8_moe(x, w13, s13, w2, s2, ids, torch.ones((rows, 1), device=dev))
    x[rows // 2] = 2.0 ** 80
    y = ops.fp8_moe(x, w13, s13, w2, s2, ids, torch.ones((rows, 1), device=dev))
    assert (y[rows // 2] == torch.inf).all() and torch.isfinite(want).all()
    keep = [r for r in range(rows) if r != rows // 2]
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("rows,experts,topk", [(16, 64, 4), (31, 64, 3), (64, 64, 3), (64, 9, 2)])
def test_moe_crowded_expert(dev, rows, experts, topk):
    """One expert that every row names, more rows than are taken at once, among experts of few rows."""
    gen = gen_of(dev, rows)
    mats = layer(gen, experts, 256, 128, size=1.0)
    x = normal(gen, rows, 256, spread=False)
    ids, wts = routed(gen, rows, experts, topk)
    ids[:, 0] = 5
    ids[:5, 1] = 7
    check_moe(x, mats, ids, wts, 8.0)


def test_unaligned_inputs_and_own_output(dev):
    """x two bytes off a 16-byte border; the layer's output over its input."""
    gen = gen_of(dev, 21)
    w, sw = R.matrix(gen, 64, 256)
    mats = layer(gen, 4, 256, 128, size=1.0)
    for rows in (2, 20):
        flat = normal(gen, 1 + rows * 256, spread=False)
        x = flat[1:].view(rows, 256)
        assert torch.equal(ops.fp8_linear(x, w, sw), ops.fp8_linear(x.clone(), w, sw))
        ids, wts = routed(gen, rows, 4, 2)
        want = ops.fp8_moe(x.clone(), *mats, ids, wts)
        assert torch.equal(ops.fp8_moe(x, *mats, ids, wts), want)
        y = x.clone()
        assert ops.fp8_moe(y, *mats, ids, wts, out=y) is y and torch.equal(y, want)


def test_unaligned_matrices_and_outputs_are_refused(dev):
    """What a kernel reads or writes by 16 bytes and is too large to copy for a call."""
    off = lambda t: torch.cat([t.flatten().view(torch.uint8)[:8], t.flatten().view(torch.uint8)])[8:].view(t.dtype).view(t.shape)  # noqa: E731
    gen = gen_of(dev, 22)
    w, sw = R.matrix(gen, 64, 256)
    a, sa = rows_of(gen, 20, 256)
    x = normal(gen, 20, 256, spread=False)
    mats = layer(gen, 4, 256, 128)
    ids, wts = routed(gen, 20, 4, 2)
    c = torch.empty((20, 64), dtype=torch.bfloat16, device=dev)
    for call in (lambda: ops.fp8_gemm(off(a), sa, w, sw), lambda: ops.fp8_gemm(a, sa, off(w), sw),
                 lambda: ops.fp8_gemm_into(a, sa, w, sw, off(c)), lambda: ops.fp8_linear(x, off(w), sw),
                 lambda: ops.fp8_moe(x, off(mats[0]), *mats[1:], ids, wts),
                 lambda: ops.fp8_moe(x, *mats[:2], off(mats[2]), mats[3], ids, wts),
                 lambda: ops.fp8_moe(x, *mats, ids, wts, out=off(x))):
        with pytest.raises(RuntimeError, match="16-byte aligned"):
            call()


def test_moe_rows_are_apart(dev):
    """NaN and infinities of a row, or of an expert that only it names, stay in it."""
    gen = gen_of(dev, 12)
    mats = layer(gen, 5, 256, 256)
    x = normal(gen, 18, 256, spread=False)
    ids = torch.randint(0, 4, (18, 2), generator=gen, device=dev, dtype=torch.int32)
    ids[:, 1] = (ids[:, 0] + 1) % 4
    wts = torch.rand((18, 2), generator=gen, device=dev)
    clean = ops.fp8_moe(x, *mats, ids, wts)
    x[3, 7], x[17, 0] = torch.nan, torch.inf
    ids[5, 1] = 4
    mats[0].view(torch.uint8)[4, 3, 9] = 0x7f
    mats[2].view(torch.uint8)[4, 200, 9] = 0x7f
    y = ops.fp8_moe(x, *mats, ids, wts)
    assert torch.isnan(y[3]).all() and torch.isnan(y[17]).any() and torch.isnan(y[5]).any()
    keep = [r for r in range(18) if r not in (3, 5, 17)]
    assert torch.equal(y[keep], clean[keep])


def test_moe_full_size_layer(dev):
    """256 experts of 4096 x 2048: byte offsets past 2^32, and an act row for each of 16 x 8 slots."""
    gen = gen_of(dev, 13)
    e, h, i = 256, 4096, 2048
    bytes_of = lambda *s: torch.randint(0, 120, s, generator=gen, device=dev, dtype=torch.uint8)  # noqa: E731
    w13 = torch.empty((e, 2 * i, h), dtype=torch.uint8, device=dev)
    w2 = torch.empty((e, h, i), dtype=torch.uint8, device=dev)
    for j in range(e):
        w13[j] = bytes_of(2 * i, h) | (bytes_of(2 * i, h) & 1) << 7
        w2[j] = bytes_of(h, i) | (bytes_of(h, i) & 1) << 7
    s13 = torch.rand((e, 2 * i // 128, h // 128), generator=gen, device=dev) * 2.0 ** -13
    s2 = torch.rand((e, h // 128, i // 128), generator=gen, device=dev) * 2.0 ** -13
    x = normal(gen, 16, h, spread=False)
    ids, wts = routed(gen, 16, e, 8)
    ids[0, 0] = 255
    y = ops.fp8_moe(x, w13.view(R.E4M3), s13, w2.view(R.E4M3), s2, ids, wts, swiglu_limit=10.0)
    pick = [0, 9, 15]
    ref, tol = R.moe(x[pick], w13.view(R.E4M3), s13, w2.view(R.E4M3), s2, ids[pick].cpu(), wts[pick].cpu(), 10.0, None,
                     y.dtype)
    within(y[pick], ref, tol, "full size")


# ---------------------------------------------------------------- together, streams, graphs


def block(x, gate, proj, mats):
    """A layer's tail as a program runs it: projection, router, experts."""
    h = ops.fp8_linear(x, *proj)
    q, s = ops.fp8_quantize(h)
    ids, wts = ops.moe_route(ops.fp8_gemm(q, s, *gate, out_dtype=torch.float32), 3, scoring="sigmoid")
    return ops.fp8_moe(h, *mats, ids, wts, swiglu_limit=4.0), ids, h


@pytest.mark.parametrize("rows", [1, 6, 24, 64])
def test_together_captured_and_on_another_stream(dev, rows):
    gen = gen_of(dev, rows)
    gate, proj, mats = R.matrix(gen, 12, 256), R.matrix(gen, 256, 512), layer(gen, 12, 256, 384)
    proj = (proj[0], proj[1] * 2.0 ** -10)
    xs = [normal(gen, rows, 512, spread=False) for _ in range(4)]
    want = [block(x, gate, proj, mats) for x in xs]
    for y, ids, h in want:
        q, s = ops.fp8_quantize(h)
        logits = ops.fp8_gemm(q, s, *gate, out_dtype=torch.float32)
        ref_ids, ref_w = R.route(logits, 3, "sigmoid", None, True, 1.0)
        assert torch.equal(ids.long(), ref_ids)
        within(y, *R.moe(h, *mats, ref_ids.cpu(), ref_w.cpu(), 4.0, None, y.dtype), "block")
    static = xs[0].clone()
    graphs = []
    for _ in range(2):                                     # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(static, gate, proj, mats)
        graphs.append((g, out))
    for k, x in enumerate(xs):
        static.copy_(x)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])
        eager = block(xs[(k + 1) % 4], gate, proj, mats)
        assert torch.equal(eager[0], want[(k + 1) % 4][0])
    side = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    torch.cuda.synchronize()
    got = []
    for n in range(8):                                     # two streams at once
        with torch.cuda.stream(side[n % 2]):
            got.append(block(xs[n % 4], gate, proj, mats))
    torch.cuda.synchronize()
    assert all(torch.equal(got[n][0], want[n % 4][0]) for n in range(8))


def test_router_feeds_the_packed_experts(dev):
    """moe_route's outputs go into the trellis-packed layer as they are: a slot with id -1 adds nothing there either."""
    from dsv4_carve_amd import synth
    from oracle import oracle as O

    E, H, I, m = 8, 512, 256, 5
    experts = [synth.expert(e, H, I, 3, seed=8) for e in range(E)]
    keep, cols = [], {k: [] for k in ops.MOE_TABLE_KEYS}
    for ex in experts:
        for p in ("gate", "up", "down"):
            for part in ("trellis", "suh", "svh"):
                keep.append(torch.from_numpy(ex[p][part]).to(dev))
                cols[f"{p}_{part}"].append(int(keep[-1].data_ptr()))
    tables = {k: torch.tensor(v, dtype=torch.int64, device=dev) for k, v in cols.items()}
    logits = torch.randn((m, E), generator=gen_of(dev, 3), device=dev)
    logits[1, 1:] = -torch.inf
    ids, wts = ops.moe_route(logits, 2)
    assert ids[1].tolist()[1] == -1
    xm = synth.activations(m, H, seed=10)
    out = torch.empty((m, H), dtype=torch.float32, device=dev)
    ops.moe_decode(torch.from_numpy(xm).to(dev), out, tables, ids, wts, intermediate=I, bits=3, swiglu_limit=10.0)
    ids_np = ids.cpu().numpy()
    wts_np = wts.cpu().numpy()
    ids_np[1, 1] = 0                                       # weight 0: the oracle's way to skip the slot
    assert wts_np[1, 1] == 0
    ref = O.moe(xm, ids_np, wts_np, experts, 10.0)
    got = out.cpu().numpy()
    assert abs(got - ref).max() <= 2e-2
