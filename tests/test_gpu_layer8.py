"""The norm, the 8-bit cache and the attention over it on the GPU, against 64-bit references."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import _lib, ops
from tests import fp8_ref as R
from tests import layer8_ref as L8
from tests.test_gpu_fp8 import gen_of, normal, within

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


# ---------------------------------------------------------------- norm


def near(got, ref, dtype, least=0.0):
    """One rounding to fp32 and one to dtype; past dtype's largest value by half a step an infinity."""
    past = ref.abs() >= torch.finfo(dtype).max * (1 + R.half_step(dtype))
    assert torch.equal(got[past].double(), torch.copysign(torch.full_like(ref[past], torch.inf), ref[past]))
    tol = ref.abs() * (R.half_step(dtype) + 2.0 ** -24) + least
    within(got[~past], ref[~past], tol[~past], str(dtype)) if not past.all() else None


def check_norm(x, weight, residual=None, eps=1e-6, pow2=False, normed_dtype=None):
    k = x.shape[-1]
    got = ops.fp8_norm(x, weight, residual=residual, eps=eps, pow2=pow2, normed_dtype=normed_dtype)
    flat = lambda t: None if t is None else t.reshape(-1, k)  # noqa: E731
    q, scale, h, y = L8.norm(flat(x), weight, flat(residual), eps, pow2)
    assert got.q.shape == x.shape and got.q.dtype == R.E4M3 and got.scale.shape == (*x.shape[:-1], -(-k // 128))
    assert torch.equal(flat(got.q).double(), q)
    within(got.scale.reshape(scale.shape), scale, scale * 2.0 ** -24 * (0 if pow2 else 1 + 2.0 ** -20), "scale")
    assert (got.residual is None) == (residual is None) and (got.normed is None) == (normed_dtype is None)
    if residual is not None:
        assert got.residual.dtype == residual.dtype
        near(flat(got.residual), h, residual.dtype, 2.0 ** -25 * (residual.dtype == torch.float16))
    if normed_dtype is not None:
        assert got.normed.dtype == normed_dtype
        near(flat(got.normed), y, normed_dtype, 2.0 ** -25 * (normed_dtype == torch.float16))
    return got


SHAPES = [(1, 1), (2, 16), (3, 127), (5, 128), (7, 144), (9, 1008), (6, 1024), (33, 1536), (3, 2048), (7, 4096), (300, 250),
          (2, 5120), (3, 8192), (2, 12304), (2, 16384), (2, 16400), (1, 40000)]


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pow2", [False, True])
def test_norm(dev, dtype, rows, k, pow2):
    gen = gen_of(dev, rows * k)
    x = normal(gen, rows, k, dtype=dtype)
    weight = normal(gen, k, dtype=dtype, spread=False)
    residual = normal(gen, rows, k, dtype=dtype)
    check_norm(x, weight, pow2=pow2)
    check_norm(x, weight.float(), residual, pow2=pow2, normed_dtype=dtype)
    check_norm(x, weight.to(torch.float16), residual.float(), pow2=pow2, normed_dtype=torch.float32)


@pytest.mark.parametrize("k", [256, 250])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_keeps_ties(dev, dtype, k):
    """Few-bit values: many quotients of a value and its group's largest lie on a rounding border of e4m3."""
    gen = gen_of(dev, 4)
    most = torch.arange(1, 129, device=dev).float().reshape(-1, 1) / 64
    x = (most * (torch.randint(0, 897, (128, k), generator=gen, device=dev) / 896.0)).to(dtype)
    x[:, 0::128] = most.to(dtype)
    weight = torch.full((k,), 1.25, device=dev)
    q, _, _, _ = L8.norm(x, weight, None, 1e-6, False)
    quotient = x.double() * 448 / most.to(dtype).double()
    assert (2 * (quotient - q).abs() == R.power(torch.frexp(quotient.clamp(min=2.0 ** -6)).exponent - 4)).sum() > 20
    check_norm(x, weight)
    check_norm(x, weight, pow2=True)


@pytest.mark.parametrize("k", [256, 200, 20000])
def test_norm_extremes(dev, k):
    for dtype in TYPES:
        f = torch.finfo(dtype)
        for v in (0.0, f.smallest_normal * 2.0 ** -4, f.tiny, f.max, -f.max):
            x = torch.zeros((2, k), dtype=dtype, device=dev)
            x[0, 3:9] = v
            x[1, :] = v
            for eps in (1e-6, 1e-30):
                check_norm(x, torch.ones(k, dtype=dtype, device=dev), eps=eps)
                check_norm(x, torch.ones(k, dtype=dtype, device=dev), x.clone(), eps=eps, pow2=True)


@pytest.mark.parametrize("k", [384, 380])
@pytest.mark.parametrize("pow2", [False, True])
def test_norm_groups_of_any_size(dev, k, pow2):
    """Groups of a row whose largest values are 2^250 apart, and products with the weight past fp32's range."""
    gen = gen_of(dev, k + 1)
    x, w = normal(gen, 90, k, dtype=torch.float32, spread=False), normal(gen, k, dtype=torch.float32, spread=False)
    for exponents in ((-120, 60, 0), (60, -130, 10), (-100, -101, -99), (100, 99, 101), (40, 40, 40)):
        size = torch.tensor(exponents, device=dev).repeat_interleave(128)[:k]
        check_norm(torch.ldexp(x, size), w, pow2=pow2, eps=1e-30)
        check_norm(x, torch.ldexp(w, size), pow2=pow2)
        check_norm(torch.ldexp(x, size // 2), torch.ldexp(w, size), pow2=pow2)


@pytest.mark.parametrize("k", [384, 380])
@pytest.mark.parametrize("pow2", [False, True])
def test_norm_rows_that_are_not_finite(dev, k, pow2):
    """They stay by themselves: a NaN row is NaN under the least scale, a row with an infinity 0 and NaN; 0 / 0 is NaN."""
    gen = gen_of(dev, k)
    x, weight = normal(gen, 4, k), normal(gen, k, spread=False)
    clean = ops.fp8_norm(x, weight, pow2=pow2, normed_dtype=torch.bfloat16)
    x[1, 5], x[2, 300] = torch.nan, -torch.inf
    got = ops.fp8_norm(x, weight, pow2=pow2, normed_dtype=torch.bfloat16)
    for r in (0, 3):
        assert torch.equal(got.q[r].float(), clean.q[r].float()) and torch.equal(got.scale[r], clean.scale[r])
    assert got.q[1].float().isnan().all() and got.normed[1].isnan().all()
    want = torch.zeros(k, device=dev)
    want[300] = torch.nan
    assert torch.equal(got.q[2].float().nan_to_num(7.0), want.nan_to_num(7.0)) and got.normed[2, 300].isnan()
    assert (got.scale[1:3] == 2.0 ** -126).all()
    zero = ops.fp8_norm(torch.zeros((1, k), device=dev), weight, eps=0.0, pow2=pow2)
    assert zero.q.float().isnan().all()


def test_norm_shapes_alignment_and_place(dev):
    gen = gen_of(dev, 8)
    w = normal(gen, 256, spread=False)
    empty = ops.fp8_norm(torch.empty((0, 256), dtype=torch.bfloat16, device=dev), w, normed_dtype=torch.float16)
    assert empty.q.shape == (0, 256) and empty.scale.shape == (0, 2) and empty.normed.dtype == torch.float16
    check_norm(normal(gen, 2, 3, 256), w, normal(gen, 2, 3, 256, dtype=torch.float32))
    off = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    x, r = normal(gen, 5, 256), normal(gen, 5, 256)
    for a, b, c in ((off(x), w, r), (x, off(w), r), (x, w, off(r))):
        check_norm(a, b, c, normed_dtype=torch.bfloat16)
    for k in (256, 250):                                    # the new residual over the old one, through the C ABI
        x, r, w = normal(gen, 9, k), normal(gen, 9, k), normal(gen, k, spread=False)
        want = ops.fp8_norm(x, w, residual=r)
        q, s = torch.empty_like(want.q), torch.empty_like(want.scale)
        _lib.check(_lib.load().exl3_fp8_norm(x.data_ptr(), 1, r.data_ptr(), 1, w.data_ptr(), 1, 9, k, 1e-6, 0, q.data_ptr(),
                                             s.data_ptr(), r.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(r, want.residual) and torch.equal(q.float(), want.q.float()) and torch.equal(s, want.scale)


@pytest.mark.parametrize("rows,k", [((1 << 24) + 40, 2), ((1 << 26) + 40, 16)])
def test_norm_more_rows_than_a_launch_takes(dev, rows, k):
    gen = gen_of(dev, k)
    x = torch.empty((rows, k), dtype=torch.int16, device=dev)
    for part in x.split(1 << 24):
        part.random_(0, 0x7f00, generator=gen)
    x = x.view(torch.bfloat16)
    w = torch.ones(k, dtype=torch.bfloat16, device=dev)
    got = ops.fp8_norm(x, w)
    a_launch = ((1 << 24) - 1) * (4 if k == 16 else 1)
    assert rows > a_launch
    for at in (0, a_launch - 5, rows - 37):
        want = ops.fp8_norm(x[at:at + 37].clone(), w)
        assert torch.equal(got.q[at:at + 37].view(torch.uint8), want.q.view(torch.uint8))
        assert torch.equal(got.scale[at:at + 37], want.scale)


# ---------------------------------------------------------------- cache


def cache_on(gen, pages, kv, page, dim, octaves=2):
    return ops.Fp8Cache(*L8.make_cache(gen, pages, kv, page, dim, octaves))


def starts_of(dev, counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=dev)


def lengths_of(dev, lengths):
    return torch.tensor(lengths, dtype=torch.int32, device=dev)


def check_append(k, v, cache, table, lengths, starts=None):
    want = L8.append(k.cpu(), v.cpu(), [t.cpu() for t in cache], table.cpu(), lengths.cpu(), None if starts is None else starts.cpu())
    back = ops.fp8_cache_append(k, v, cache, table, lengths, starts)
    assert back is cache
    for name, got, ref in zip(cache._fields, cache, want):
        got = got.cpu().double()
        assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0)), name


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,kv,dim", [(torch.bfloat16, 2, 128), (torch.float16, 1, 80), (torch.float32, 3, 16),
                                          (torch.bfloat16, 1, 256)])
def test_append(dev, page, dtype, kv, dim):
    """Fresh and begun pages, chunks that end inside one, sequences without new tokens; what is not written stays."""
    gen = gen_of(dev, page + dim)
    counts, lengths = [1, 5, 0, 40, page, 300, 1], [1, 9, 33, 40, page + 3, 300 + page // 2, 2 * page]
    table, pages = L8.make_table(gen, lengths, page)
    k, v = normal(gen, sum(counts), kv, dim, dtype=dtype), normal(gen, sum(counts), kv, dim, dtype=dtype)
    k *= torch.exp2(torch.randint(-12, 6, (sum(counts), 1, 1), generator=gen, device=dev)).to(dtype)
    check_append(k, v, cache_on(gen, pages, kv, page, dim, 6), table, lengths_of(dev, lengths), starts_of(dev, counts))


@pytest.mark.parametrize("page,dim,dtype", [(16, 32, torch.bfloat16), (256, 256, torch.float32), (256, 240, torch.float16),
                                            (128, 144, torch.bfloat16)])
def test_append_many_sequences(dev, page, dim, dtype):
    """More sequences than a wave has lanes, most of few tokens, some of whole pages."""
    gen = gen_of(dev, page + dim)
    counts = [(0, 1, 2, 5)[i % 4] for i in range(150)]
    counts[70], counts[131] = page + 7, 2 * page
    lengths = [c + (i * 13) % 20 for i, c in enumerate(counts)]
    table, pages = L8.make_table(gen, lengths, page)
    k, v = normal(gen, sum(counts), 1, dim, dtype=dtype), normal(gen, sum(counts), 1, dim, dtype=dtype)
    check_append(k, v, cache_on(gen, pages, 1, page, dim, 6), table, lengths_of(dev, lengths), starts_of(dev, counts))


@pytest.mark.parametrize("page,kv,dim", [(16, 7, 128), (64, 3, 80), (128, 8, 16), (256, 5, 32)])
def test_append_a_wave_a_page(dev, page, kv, dim):
    """Many sequences of few tokens, and heads that are no multiple of a workgroup's waves; one with pages of tokens."""
    gen = gen_of(dev, page + kv)
    for counts in ([1] * 400, [1 + i % 3 for i in range(399)] + [2 * page + 5], [6 * (i % 2) for i in range(300)]):
        lengths = [c + (i * 29) % (2 * page) for i, c in enumerate(counts)]
        table, pages = L8.make_table(gen, lengths, page)
        k, v = normal(gen, sum(counts), kv, dim), normal(gen, sum(counts), kv, dim)
        starts = None if max(counts) == 1 else starts_of(dev, counts)
        check_append(k, v, cache_on(gen, pages, kv, page, dim, 6), table, lengths_of(dev, lengths), starts)


@pytest.mark.parametrize("page", [16, 64])
def test_append_token_by_token(dev, page):
    """Scales grow and stay as the tokens come, and each page begins anew."""
    gen = gen_of(dev, page)
    table, pages = L8.make_table(gen, [2 * page + 3, 2 * page + 8], page)
    cache = cache_on(gen, pages, 2, page, 32)
    for i in range(2 * page + 3):
        k, v = normal(gen, 2, 2, 32), normal(gen, 2, 2, 32, dtype=torch.bfloat16)
        if i % 5 == 0:
            k *= 2.0 ** (i % 7)
        check_append(k, v, cache, table, lengths_of(dev, [i + 1, i + 6]))


def test_append_values_that_are_not_finite(dev):
    gen = gen_of(dev, 3)
    table, pages = L8.make_table(gen, [20, 3], 16)
    for dtype in TYPES:
        k, v = normal(gen, 23, 2, 16, dtype=dtype), normal(gen, 23, 2, 16, dtype=dtype)
        k[0, 0, 3], k[17, 1, 5], v[2, 1, 0], v[20] = torch.nan, torch.inf, -torch.inf, torch.nan
        k[1, :, 4] = 0.0
        cache = cache_on(gen, pages, 2, 16, 16)
        check_append(k, v, cache, table, lengths_of(dev, [20, 3]), starts_of(dev, [20, 3]))
        big = torch.full_like(k[:2], torch.finfo(dtype).max)
        check_append(big, -big, cache, table, lengths_of(dev, [21, 4]))
        check_append(big * 0, big * 0, cache, table, lengths_of(dev, [22, 1]))


def test_append_inputs_of_a_fused_projection(dev):
    """Heads of a wider row as they are, rows off their borders or turned by a copy."""
    gen = gen_of(dev, 5)
    lengths = [70, 4]
    table, pages = L8.make_table(gen, lengths, 16)
    for dtype in TYPES:
        qkv = normal(gen, 74, 8 * 32 + 32, dtype=dtype)
        k, v = qkv[:, 128:192].view(74, 2, 32), qkv[:, 192:256].view(74, 2, 32)
        assert not k.is_contiguous()
        check_append(k, v, cache_on(gen, pages, 2, 16, 32), table, lengths_of(dev, lengths), starts_of(dev, [70, 4]))
        k, v = qkv[:, 1:65].view(74, 2, 32), qkv[:, :64].view(74, 32, 2).transpose(1, 2)
        check_append(k, v, cache_on(gen, pages, 2, 16, 32), table, lengths_of(dev, lengths), starts_of(dev, [70, 4]))


def test_append_what_the_tables_name_out_of_range(dev):
    """Tokens before position 0, behind the table's room, pages outside the cache, starts outside the call."""
    gen = gen_of(dev, 6)
    k, v = normal(gen, 90, 2, 32), normal(gen, 90, 2, 32)
    wide = torch.full((5, 9), -3, dtype=torch.int32, device=dev)
    wide[:, :3] = torch.arange(15, device=dev).view(5, 3)
    wide[1, 1], wide[2, 0] = 15, 1 << 30
    table = wide[:, :3]                                     # a slice of a wider table; room for 48 tokens
    for lengths, starts in (([5, 48, 40, 1000, 0], [0, 20, 40, 60, 80, 90]), ([-4, 30, 2 ** 31 - 1, 48, 47], [-9, 20, 15, 50, 95, 200]),
                            ([48] * 5, [80, 90, 90, 10, 20, 3])):
        cache = cache_on(gen, 15, 2, 16, 32)
        check_append(k, v, cache, table, lengths_of(dev, lengths), lengths_of(dev, starts))


def test_append_nothing(dev):
    gen = gen_of(dev, 7)
    cache = cache_on(gen, 3, 1, 16, 16)
    before = [t.clone() for t in cache]
    none = torch.empty((0, 1, 16), dtype=torch.bfloat16, device=dev)
    table = torch.zeros((2, 2), dtype=torch.int32, device=dev)
    ops.fp8_cache_append(none, none, cache, table, lengths_of(dev, [3, 4]), lengths_of(dev, [0, 0, 0]))
    ops.fp8_cache_append(none, none, cache, table[:0], lengths_of(dev, []))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))


# ---------------------------------------------------------------- attention


def check_attention(q, cache, table, lengths, starts=None, **kw):
    out, lse = ops.fp8_attention(q, cache, table, lengths, starts, return_lse=True, **kw)
    kw.pop("out", None)
    ref, tol, ref_lse, lse_tol, mine = L8.attention(q, cache, table, lengths, starts, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:2]
    within(out[mine], ref[mine], tol[mine], "out")
    empty = ref_lse == -torch.inf
    assert torch.equal(lse == -torch.inf, empty) and (out[empty] == 0).all()
    within(lse[mine & ~empty.any(1)], ref_lse[mine & ~empty.any(1)], lse_tol[mine & ~empty.any(1)], "lse")
    return out, lse


def problem(gen, counts, lengths, *, heads, kv, dim, page, dtype=torch.bfloat16, octaves=2, size=1.0):
    dev = gen.device
    table, pages = L8.make_table(gen, lengths, page)
    q = (torch.randn((sum(counts), heads, dim), generator=gen, device=dev) * size).to(dtype)
    return q, cache_on(gen, pages, kv, page, dim, octaves), table, lengths_of(dev, lengths), starts_of(dev, counts)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 144, 192, 208, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_single_tokens(dev, dim, page, dtype):
    gen = gen_of(dev, dim * page)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 300, 1000, 37, 129]
    q, cache, table, n, _ = problem(gen, [1] * 12, lengths, heads=6, kv=2, dim=dim, page=page, dtype=dtype)
    check_attention(q, cache, table, n)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 12, 16, 20, 40])
@pytest.mark.parametrize("counts,lengths", [([3, 1, 2], [70, 1, 333]), ([5, 60, 1, 0], [5, 130, 200, 9]), ([200], [1000])])
def test_attention_groups_and_several_queries(dev, group, counts, lengths):
    """Every size of a tile, tiles that end inside a query's heads, more queries than one tile."""
    gen = gen_of(dev, group)
    for dtype, dim, kv in ((torch.bfloat16, 64, 2), (torch.float16, 128, 1), (torch.bfloat16, 192, 1)):
        check_attention(*problem(gen, counts, lengths, heads=group * kv, kv=kv, dim=dim, page=16, dtype=dtype))


@pytest.mark.parametrize("window", [1, 7, 64, 100, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_window_sinks_and_scale(dev, window, dtype):
    gen = gen_of(dev, window)
    p = problem(gen, [1, 4, 90, 7], [1, 500, 90, 3000], heads=8, kv=2, dim=64, page=32, dtype=dtype)
    sinks = torch.randn(8, generator=gen, device=dev) * 4
    sinks[3], sinks[5] = -torch.inf, 30.0
    check_attention(*p, window=window)
    check_attention(*p, window=window, sinks=sinks, scale=0.3)
    check_attention(*p, sinks=sinks, scale=-0.05)


def test_attention_many_sequences_share_the_work(dev):
    """More tiles than workgroups, shares that begin and end inside them, sequences of one and of thousands of keys."""
    gen = gen_of(dev, 1)
    lengths = [1 + (i * 7919) % 700 for i in range(300)] + [9000, 1, 4500]
    check_attention(*problem(gen, [1] * 303, lengths, heads=4, kv=2, dim=64, page=16))
    counts = [1 + i % 3 for i in range(303)]
    lengths = [max(c, n) for c, n in zip(counts, lengths)]
    check_attention(*problem(gen, counts, lengths, heads=8, kv=2, dim=128, page=64, dtype=torch.float16))


@pytest.mark.parametrize("dim,heads,kv,seqs", [(64, 64, 32, 40), (64, 320, 16, 40), (128, 48, 24, 50), (128, 32, 32, 40),
                                               (208, 64, 16, 70)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_a_workgroup_a_sequence(dev, dim, heads, kv, seqs, dtype):
    """As many tokens as sequences, one each or not, where a workgroup has a tile; some sequences without keys."""
    gen = gen_of(dev, dim + kv)
    lengths = [(i * 37) % 200 for i in range(seqs)]
    q, cache, table, n, _ = problem(gen, [1] * seqs, lengths, heads=heads, kv=kv, dim=dim, page=32, dtype=dtype)
    assert ops._fp8_attention_scratch_bytes(dev.index or 0, seqs, heads, kv, dim, seqs, table.shape[1], 32, 0) == 0
    sinks = torch.randn(heads, generator=gen, device=dev)
    alone, _ = check_attention(q, cache, table, n, sinks=sinks)
    counts = [(2, 0, 1, 1)[i % 4] for i in range(seqs - seqs % 4)] + [1] * (seqs % 4)
    check_attention(q, cache, table, n, starts_of(dev, counts), sinks=sinks, window=40)
    same = ops.fp8_attention(q, cache, table, n, starts_of(dev, [1] * seqs), sinks=sinks)
    assert torch.equal(same, alone)


def test_attention_one_long_sequence(dev):
    gen = gen_of(dev, 2)
    for heads, counts in ((4, [1]), (32, [2]), (8, [40])):
        check_attention(*problem(gen, counts, [50000], heads=heads, kv=1, dim=128, page=128, size=4.0))


def test_attention_prompts(dev):
    """Whole prompts, a workgroup a tile, several heads; chunks behind a context."""
    gen = gen_of(dev, 3)
    check_attention(*problem(gen, [700, 1, 333, 1000], [700, 1, 333, 1300], heads=16, kv=8, dim=64, page=16))
    check_attention(*problem(gen, [900, 500], [900, 2100], heads=8, kv=8, dim=128, page=64, dtype=torch.float16))


@pytest.mark.parametrize("dim", [48, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("counts", [[2, 5, 3], [1 + i % 4 for i in range(70)], [9, 4, 0, 11], [60, 3, 20]])
def test_attention_tiles_of_each_size(dev, dim, counts):
    """About 27, 20, 48 and 221 rows a sequence and cache head, of few such pairs and of many."""
    gen = gen_of(dev, dim + len(counts))
    lengths = [c + (i * 37) % 150 for i, c in enumerate(counts)]
    sinks = torch.randn(16, generator=gen, device=dev)
    for dtype, page in ((torch.bfloat16, 16), (torch.float16, 64)):
        p = problem(gen, counts, lengths, heads=16, kv=2, dim=dim, page=page, dtype=dtype)
        check_attention(*p)
        check_attention(*p, window=30, sinks=sinks)


@pytest.mark.parametrize("heads,kv,dim,tokens", [(8, 1, 16, 17000), (16, 4, 128, 8500), (16, 8, 64, 8500), (16, 16, 96, 8500),
                                                 (6, 3, 128, 22500), (16, 4, 256, 4300)])
def test_attention_a_workgroup_a_tile(dev, heads, kv, dim, tokens):
    """More tiles than four a CU, in each order of heads and tiles; some sequences behind a context, one of one token."""
    gen = gen_of(dev, tokens + kv)
    counts = [1] + [tokens // 16] * 16
    lengths = [1 if i == 0 else c + 40 * (i % 3) for i, c in enumerate(counts)]
    p = problem(gen, counts, lengths, heads=heads, kv=kv, dim=dim, page=64, dtype=torch.bfloat16 if kv != 4 else torch.float16)
    check_attention(*p, window=None if kv % 3 else 70)


@pytest.mark.parametrize("dim,heads,kv", [(64, 32, 8), (128, 32, 8), (256, 16, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_a_chunk_behind_a_long_context(dev, dim, heads, kv, dtype):
    """Shares of about 70 units, of one tile or of two, beside a short sequence."""
    gen = gen_of(dev, dim)
    p = problem(gen, [300, 2], [28000, 500], heads=heads, kv=kv, dim=dim, page=64, dtype=dtype)
    check_attention(*p)
    check_attention(*p, window=20000)


@pytest.mark.parametrize("dim", [128, 256])
def test_attention_queries_of_far_apart_values(dev, dim):
    """Values down to 2^-30 of a row's largest, a largest one that meets zeros only, rows of any size."""
    gen = gen_of(dev, dim + 11)
    q, cache, table, n, starts = problem(gen, [150, 20], [200, 300], heads=4, kv=2, dim=dim, page=32)
    q *= torch.exp2(torch.randint(-30, 1, q.shape, generator=gen, device=dev)).to(q.dtype)
    check_attention(q, cache, table, n, starts)
    q[:, :, 3] = 2.0 ** 9                                     # beside a channel of the keys that is 0
    cache.k.view(torch.uint8)[..., 3] = 0
    check_attention(q, cache, table, n, starts)
    q *= torch.exp2(torch.randint(-100, 1, (170, 4, 1), generator=gen, device=dev)).to(q.dtype)
    q[5], q[6, 1], q[7, :, 5:] = 0.0, 2.0 ** -133, 0.0
    check_attention(q, cache, table, n, starts)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1] * 70, [9, 4, 11], [60, 3, 20]])
def test_attention_pages_that_no_query_sees(dev, dim, counts):
    """The cache's first page and pages of other sequences hold NaNs and NaN scales; so do a sequence's pages before its windows."""
    gen = gen_of(dev, dim + len(counts))
    lengths = [c + 90 + (i * 37) % 60 for i, c in enumerate(counts)]
    q, cache, table, n, starts = problem(gen, counts, lengths, heads=4, kv=2, dim=dim, page=16)
    own = table[table >= 0]
    away = ops.Fp8Cache(*(torch.cat([t.view(torch.uint8)[:1], t.view(torch.uint8), t.view(torch.uint8)[:1]]).view(t.dtype)
                          if t.dtype == R.E4M3 else torch.cat([t[:1], t, t[:1]]) for t in cache))
    moved = torch.where(table >= 0, table + 1, table)
    unseen = torch.ones(away.k.shape[0], dtype=torch.bool, device=dev)
    unseen[own.long() + 1] = False
    for window in (None, 20):
        clean = ops.fp8_attention(q, cache, table, n, starts, window=window)
        for i, (c, length) in enumerate(zip(counts, lengths)):
            if window:
                unseen[moved[i, :max(length - c - window, 0) // 16].long()] = True
        for t in (away.k, away.v):
            t.view(torch.uint8)[unseen] = 0x7f
        for t in (away.k_scale, away.v_scale):
            t[unseen] = torch.nan
        assert torch.equal(ops.fp8_attention(q, away, moved, n, starts, window=window), clean)


def test_attention_rows_without_keys(dev):
    """Lengths of zero, fewer keys than queries, a table without a valid page: 0, and -inf or the sink."""
    gen = gen_of(dev, 4)
    q, cache, table, _, starts = problem(gen, [2, 5, 3, 30, 4], [64] * 5, heads=4, kv=2, dim=64, page=16)
    table[2] = -1
    n = lengths_of(dev, [0, 2, 40, 3, -5])
    out, lse = check_attention(q, cache, table, n, starts)
    assert (out[:2] == 0).all() and (lse[:5] == -torch.inf).all() and torch.isfinite(lse[5:7]).all()
    sinks = torch.tensor([0.5, -1.0, -torch.inf, 3.0], device=dev)
    out, lse = ops.fp8_attention(q, cache, table, n, starts, sinks=sinks, return_lse=True)
    assert (out[:5] == 0).all() and (out[7:10] == 0).all()
    assert torch.allclose(lse[0], sinks, atol=1e-6) and torch.allclose(lse[-1], sinks, atol=1e-6)


def test_attention_what_the_tables_name_out_of_range(dev):
    gen = gen_of(dev, 5)
    q, cache, table, _, _ = problem(gen, [20] * 4, [64] * 4, heads=4, kv=1, dim=64, page=16)
    pages = cache.k.shape[0]
    table = table[:, :4].contiguous()
    table[0, 1], table[1, 0], table[2, 3], table[3] = pages, -1, 1 << 30, -(1 << 31)
    for lengths, starts in (([64, 40, 64, 60], [0, 20, 40, 60, 80]), ([1000, 2 ** 31 - 1, 30, 64], [-5, 30, 25, 70, 1000]),
                            ([64, 64, 64, 64], [70, 80, 10, 5, 0])):
        check_attention(q, cache, table, lengths_of(dev, lengths), lengths_of(dev, starts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_bytes_that_no_query_sees(dev, dtype):
    """NaN codes and NaN scales behind a sequence's end, before its window, and of later tokens of the same call."""
    gen = gen_of(dev, 6)
    counts, lengths, page = [1, 40, 3, 70], [37, 100, 64, 70], 16
    q, cache, table, n, starts = problem(gen, counts, lengths, heads=4, kv=2, dim=64, page=page, dtype=dtype)
    clean = [ops.fp8_attention(q, cache, table, n, starts, window=w) for w in (None, 20)]
    k8, v8 = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    for s, length in enumerate(lengths):
        if length % page:
            p = int(table[s, length // page])
            k8[p, :, length % page:] = 0x7f
            v8[p, :, :, length % page:] = 0xff
    spare = (set(range(cache.k.shape[0])) - set(table[table >= 0].tolist())).pop()
    cache.k_scale[spare], cache.v_scale[spare] = torch.nan, torch.nan
    for w, want in zip((None, 20), clean):
        assert torch.equal(ops.fp8_attention(q, cache, table, n, starts, window=w), want)
    before = int(table[1, 1])                                # keys 16..31 of the second sequence: outside the last queries' windows
    v8[before, 1, 3, 2], k8[before, 0, 7, 5] = 0x7f, 0x7f
    check = ops.fp8_attention(q, cache, table, n, starts, window=20)
    want = clean[1].clone()
    assert torch.equal(check, want)                          # its first query is at 60
    later = int(table[3, 50 // page])
    v8[later, 0, 9, 50 % page], k8[later, 1, 50 % page, 60] = 0xff, 0x7f
    for w in (None, 20):
        got = ops.fp8_attention(q, cache, table, n, starts, window=w)
        first = starts[3]
        assert torch.equal(got[first:first + 50], clean[w is not None][first:first + 50])
        sees = slice(first + 50, first + (70 if w is None else 70))
        assert got[sees, 2:].isnan().all() and got[sees, :2, 9].isnan().all()
        others = [d for d in range(64) if d != 9]
        assert torch.equal(got[sees, :2][:, :, others], clean[w is not None][sees, :2][:, :, others])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_scales_far_apart(dev, dtype):
    """Pages whose scales differ by up to 2**60, seen by rows that weigh them differently: each row is held to its own bound."""
    gen = gen_of(dev, 7)
    q, cache, table, n, starts = problem(gen, [1, 5, 66], [400, 200, 66], heads=8, kv=2, dim=64, page=16, dtype=dtype)
    cache.v_scale.copy_(torch.exp2(torch.randint(-38, 23 if dtype == torch.bfloat16 else 2, cache.v_scale.shape, generator=gen, device=dev)))
    check_attention(q, cache, table, n, starts)
    cache.v_scale.fill_(2.0 ** -12)
    cache.v_scale[int(table[0, 3])] = 2.0 ** -126             # a page of zeros under the least scale
    cache.k_scale.mul_(2.0 ** -3)
    check_attention(q, cache, table, n, starts)
    cache.k_scale.mul_(64.0)                                 # rows with one heavy key
    check_attention(q, cache, table, n, starts)


def test_attention_rows_are_apart(dev):
    gen = gen_of(dev, 8)
    q, cache, table, n, starts = problem(gen, [1, 30, 2], [90, 64, 300], heads=8, kv=2, dim=128, page=32)
    clean = ops.fp8_attention(q, cache, table, n, starts)
    q[4, 1, 7], q[20, 6, 0] = torch.nan, torch.inf
    got = ops.fp8_attention(q, cache, table, n, starts)
    assert got[4, 1].isnan().all() and got[20, 6].isnan().all()
    got[4, 1], got[20, 6] = clean[4, 1], clean[20, 6]
    assert torch.equal(got, clean)


def test_attention_inputs_and_outputs(dev):
    """Heads of a fused projection, copies where rows are off their borders, an output given, rows of no sequence."""
    gen = gen_of(dev, 9)
    q, cache, table, n, starts = problem(gen, [1, 9, 4], [90, 64, 300], heads=8, kv=2, dim=64, page=32)
    want, want_lse = check_attention(q, cache, table, n, starts)
    qkv = torch.cat([normal(gen, 14, 64), q.view(14, 512), normal(gen, 14, 32)], 1)
    assert torch.equal(ops.fp8_attention(qkv[:, 64:576].view(14, 8, 64), cache, table, n, starts), want)
    qkv = torch.cat([qkv[:, :1], q.view(14, 512), qkv[:, :5]], 1)
    assert torch.equal(ops.fp8_attention(qkv[:, 1:513].view(14, 8, 64), cache, table, n, starts), want)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.fp8_attention(turned, cache, table, n, starts), want)
    more = torch.cat([q[:3], q, q[:5]])
    out = torch.full((22, 8, 64), 7.0, dtype=q.dtype, device=dev)
    assert ops.fp8_attention(more, cache, table, n, starts + 3, out=out) is out
    assert torch.equal(out[3:17], want) and (out[:3] == 7).all() and (out[17:] == 7).all()
    out, lse = ops.fp8_attention(more, cache, table, n, starts + 3, return_lse=True)
    assert torch.equal(out[3:17], want) and torch.equal(lse[3:17], want_lse)
    assert (out[:3] == 0).all() and (out[17:] == 0).all() and (lse[:3] == -torch.inf).all() and (lse[17:] == -torch.inf).all()
    off = torch.empty(14 * 512 + 8, dtype=q.dtype, device=dev)[1:1 + 14 * 512].view(14, 8, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.fp8_attention(q, cache, table, n, starts, out=off)
    none = ops.fp8_attention(q[:0], cache, table[:0], n[:0], return_lse=True)
    assert none[0].shape == (0, 8, 64) and none[1].shape == (0, 8)
    alone, lse = ops.fp8_attention(q, cache, table[:0], n[:0], starts[:1], return_lse=True)
    assert (alone == 0).all() and (lse == -torch.inf).all()


def test_attention_offsets_past_32_bits(dev):
    """Pages on either side of 2**32 bytes of a cache."""
    gen = gen_of(dev, 10)
    pages, page, dim = 560000, 64, 128
    assert pages * page * dim > 1 << 32
    cache = ops.fp8_cache(pages, 1, page, dim, device=dev)
    n = 200
    table = torch.tensor([[pages - 1, 3, 524288, 524287]], dtype=torch.int32, device=dev)
    k, v = normal(gen, n, 1, dim, spread=False), normal(gen, n, 1, dim, spread=False)
    ops.fp8_cache_append(k, v, cache, table, lengths_of(dev, [n]), lengths_of(dev, [0, n]))
    small = ops.Fp8Cache(*(t[table[0].long()] if t.dtype == torch.float32 else t.view(torch.uint8)[table[0].long()].view(R.E4M3) for t in cache))
    own = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    want = ops.fp8_cache_append(k, v, ops.fp8_cache(4, 1, page, dim, device=dev), own, lengths_of(dev, [n]), lengths_of(dev, [0, n]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(small, want))
    q = normal(gen, 1, 4, dim, spread=False)
    assert torch.equal(ops.fp8_attention(q, cache, table, lengths_of(dev, [n])), ops.fp8_attention(q, small, own, lengths_of(dev, [n])))


# ---------------------------------------------------------------- together, streams, graphs


class Layer:
    """A decoder layer's attention as a program runs it: norm, projections, cache, attention, output projection, next norm."""

    def __init__(self, gen, heads=8, kv=2, dim=64, hidden=512, page=16):
        self.heads, self.kv, self.dim = heads, kv, dim
        scaled = lambda m, f: (m[0], m[1] * f)  # noqa: E731
        self.qkv = scaled(R.matrix(gen, (heads + 2 * kv) * dim, hidden), 2.0 ** -8)
        self.proj = scaled(R.matrix(gen, hidden, heads * dim), 2.0 ** -9)
        self.w = [normal(gen, hidden, spread=False) for _ in range(2)]

    def __call__(self, x, residual, cache, table, lengths, starts=None):
        a = ops.fp8_norm(x, self.w[0], residual=residual)
        qkv = ops.fp8_gemm(a.q, a.scale, *self.qkv).view(x.shape[0], -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv, self.kv), dim=1)
        ops.fp8_cache_append(k, v, cache, table, lengths, starts)
        o = ops.fp8_attention(q, cache, table, lengths, starts)
        y = ops.fp8_linear(o.view(x.shape[0], -1), *self.proj)
        return (*ops.fp8_norm(y, self.w[1], residual=a.residual, normed_dtype=torch.bfloat16), qkv, o, y, a)


@pytest.mark.parametrize("chunk", [1, 5, 70])
def test_together(dev, chunk):
    """A prompt and the tokens behind it, each step against the references on what it was given."""
    gen = gen_of(dev, chunk)
    layer = Layer(gen)
    lengths = [chunk * 3, chunk * 3 + 11]
    table, pages = L8.make_table(gen, lengths, 16)
    cache = ops.fp8_cache(pages, 2, 16, 64, device=dev)
    first = normal(gen, 11, 512, spread=False)
    layer(first, first, cache, table[1:], lengths_of(dev, [11]), lengths_of(dev, [0, 11]))
    starts = starts_of(dev, [chunk, chunk])
    for step in range(3):
        x, r = normal(gen, 2 * chunk, 512, spread=False), normal(gen, 2 * chunk, 512, spread=False)
        n = lengths_of(dev, [chunk * (step + 1), chunk * (step + 1) + 11])
        before = [t.cpu() for t in cache]
        q2, s2, r2, y2, qkv, o, y, a = layer(x, r, cache, table, n, starts if chunk > 1 else None)
        assert torch.equal(a.q.double(), L8.norm(x, layer.w[0], r, 1e-6, False)[0])
        k, v = qkv[:, 8:10], qkv[:, 10:]
        want = L8.append(k.cpu(), v.cpu(), before, table.cpu(), n.cpu(), starts.cpu() if chunk > 1 else None)
        assert all(torch.equal(t.cpu().double(), w) for t, w in zip(cache, want))
        ref, tol, _, _, _ = L8.attention(qkv[:, :8], cache, table, n, starts if chunk > 1 else None)
        within(o, ref, tol, "attention")
        assert torch.equal(q2.double(), L8.norm(y, layer.w[1], a.residual, 1e-6, False)[0])


def test_captured_and_on_other_streams(dev):
    """Two graphs of a decode step over one cache, replayed in turn with eager steps between; two streams at once."""
    gen = gen_of(dev, 30)
    layer = Layer(gen)
    seqs, room = 5, 96
    table, pages = L8.make_table(gen, [room] * seqs, 16)
    base = [7, 30, 1, 64, 50]
    xs = [normal(gen, seqs, 512, spread=False) for _ in range(8)]
    start = cache_on(gen, pages, 2, 16, 64)

    def fresh():
        return ops.Fp8Cache(*(t.clone() for t in start))

    cache, want = fresh(), []
    for i, x in enumerate(xs):
        want.append([t.clone() for t in layer(x, x, cache, table, lengths_of(dev, [b + i for b in base]))[:4]])
    end = [t.clone() for t in cache]

    cache = fresh()
    sx, sn = xs[0].clone(), lengths_of(dev, base)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(sx, sx, cache, table, sn)
        graphs.append((g, out))
    for i, x in enumerate(xs):
        sx.copy_(x)
        sn.copy_(lengths_of(dev, [b + i for b in base]))
        if i % 3 == 2:
            out = layer(sx, sx, cache, table, sn)
        else:
            g, out = graphs[i % 2]
            g.replay()
            g.replay()                                       # the same tokens again: the same cache and results
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out[:4], want[i])), i
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, end))

    torch.cuda.synchronize()
    side, caches, got = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)], [fresh(), fresh()], [[], []]
    torch.cuda.synchronize()
    for i, x in enumerate(xs):
        for j in (0, 1):
            with torch.cuda.stream(side[j]):
                got[j].append(layer(x, x, caches[j], table, lengths_of(dev, [b + i for b in base]))[:4])
    torch.cuda.synchronize()
    for j in (0, 1):
        for i in range(len(xs)):
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[j][i], want[i]))


def test_results_do_not_depend_on_the_run(dev):
    gen = gen_of(dev, 31)
    p = problem(gen, [1] * 40, [1 + 97 * i for i in range(40)], heads=16, kv=2, dim=128, page=64)
    want = ops.fp8_attention(*p)
    assert all(torch.equal(ops.fp8_attention(*p), want) for _ in range(5))
