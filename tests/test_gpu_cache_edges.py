"""Borders of the 8-bit cache and the attention over it on the GPU, against 64-bit references."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import ops
from tests import layer8_ref as L8
from tests.test_gpu_fp8 import gen_of, normal, within
from tests.test_gpu_layer8 import cache_on, check_append, check_attention, lengths_of, problem, starts_of

pytestmark = pytest.mark.gpu


def rounded_from(got, ref, tol):
    """got is what some value within tol of ref rounds to; 2^-22 of ref for fp32 on the way to a bf16 bound."""
    tol = tol + ref.abs() * 2.0 ** -22
    lo, hi = (ref - tol).to(got.dtype).double(), (ref + tol).to(got.dtype).double()
    off = int(((got.double() < lo) | (got.double() > hi)).sum())
    assert off == 0, f"{off} of {got.numel()} values are rounded from elsewhere"


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("count", [1, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_few_rows_keep_the_weights_bits(dev, dim, count, dtype):
    """A result of few rows is the fp32 one rounded.

    One channel of the query is not zero and is 1/4 at most, keys are 3.5 at most: the bound of an fp32 query counts
    dim + 2 steps of 2^-23 of the product and 6 more, twice, for a weight's logit, 1.1e-4 for 256 channels at most, and
    the sums' 60 steps: 2^-13.  An 11-bit weight is off by up to 2^-12, so that with 64 channels, where the bound is
    2^-14.6, some results of bf16 would be rounded from outside it."""
    gen = gen_of(dev, dim + count)
    counts = [count] * 48
    lengths = [count + 1 + i % 15 for i in range(48)]
    q, cache, table, n, starts = problem(gen, counts, lengths, heads=8, kv=2, dim=dim, page=16, dtype=dtype, octaves=0)
    q[..., 1:] = 0
    q.clamp_(-0.25, 0.25)
    out = ops.fp8_attention(q, cache, table, n, starts, scale=1.0)
    ref, tol, *_ = L8.attention(q.float(), cache, table, n, starts, scale=1.0)
    if dim > 128 and count > 1 and dtype == torch.bfloat16:
        # 20 rows of a wide head go through the kernel for many rows, whose weights have 11 bits for a bf16 result: each
        # is off by up to 2^-12 of itself, so the result by that of its weighted magnitudes, which are the largest value's
        # at most
        tol = tol + 2.0 ** -12 * 448 * float(cache.v_scale.max())
    rounded_from(out, ref, tol + 2.0 ** -25 * (dtype == torch.float16))


@pytest.mark.parametrize("counts,heads,kv,dim", [([1, 1, 1], 4, 2, 64), ([40, 7], 8, 1, 128), ([300, 1], 4, 4, 256)])
def test_attention_logarithms_of_rows_that_no_sequence_has(dev, counts, heads, kv, dim):
    """With an `out` given, whose rows stay, the logarithms are the call's own: -inf before, behind and without sequences."""
    gen = gen_of(dev, dim)
    q, cache, table, n, starts = problem(gen, [5, *counts, 9], [5, *(c + 60 for c in counts), 9], heads=heads, kv=kv, dim=dim,
                                         page=16)
    table, n, starts = table[1:-1], n[1:-1].contiguous(), starts[1:-1].contiguous()
    mine = slice(5, 5 + sum(counts))
    want, want_lse = ops.fp8_attention(q, cache, table, n, starts, return_lse=True)
    none = torch.ones(q.shape[0], dtype=torch.bool, device=dev)
    none[mine] = False
    assert (want[none] == 0).all() and (want_lse[none] == -torch.inf).all()
    for given in (starts, torch.zeros_like(starts)):
        for _ in range(3):
            out = torch.full_like(q, 7.0)
            torch.full((q.shape[0], heads), 3.0, device=dev)          # what the logarithms' place held before
            got, lse = ops.fp8_attention(q, cache, table, n, given, out=out, return_lse=True)
            assert got is out
            left = none if given is starts else torch.ones_like(none)
            assert (out[left] == 7.0).all() and (lse[left] == -torch.inf).all()
            assert torch.equal(out[~left], want[~left]) and torch.equal(lse[~left], want_lse[~left])
            assert torch.equal(ops.fp8_attention(q, cache, table, n, given, out=torch.full_like(q, 7.0)), out)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("counts", [[1, 1, 1], [20, 70, 3], [1] * 70, [300, 2]])
def test_lengths_past_the_tables_room(dev, page, counts):
    """Tokens behind the room have no place: nothing is written for them, and they do not take the place of others."""
    gen = gen_of(dev, page)
    seqs, room, kv, dim = len(counts), 3 * page, 2, 64
    table = torch.randperm(3 * seqs, generator=gen, device=dev).to(torch.int32).view(seqs, 3)
    starts = None if max(counts) == 1 else starts_of(dev, counts)
    k, v = normal(gen, sum(counts), kv, dim), normal(gen, sum(counts), kv, dim)
    q = normal(gen, sum(counts), 4, dim, spread=False)
    # all new tokens behind the room, the first of them its last place, some of them in it, none
    for at, past in enumerate((lambda n: room + n, lambda n: room + n - 1, lambda n: room + n // 2, lambda n: room)):
        lengths = lengths_of(dev, [past(n) for n in counts])
        cache = cache_on(gen, 3 * seqs, kv, page, dim)
        before = [t.clone() for t in cache]
        check_append(k, v, cache, table, lengths, starts)
        live = [(s, j) for s, n in enumerate(counts) for j in range(min(past(n) - n, room))]     # keys from before the call
        ids = torch.tensor([int(table[s, j // page]) for s, j in live], device=dev)
        slot = torch.tensor([j % page for _, j in live], device=dev)
        full = ids[slot == page - 1]
        for was, now in zip(before, cache):
            assert torch.equal(now.view(torch.uint8)[full], was.view(torch.uint8)[full])
        if at == 0:
            assert all(torch.equal(now.view(torch.uint8), was.view(torch.uint8)) for was, now in zip(before, cache))
        for window in (None, 5, page):
            check_attention(q, cache, table, lengths, starts, window=window)
    lengths = lengths_of(dev, [2 ** 31 - 1] * seqs)
    check_append(k, v, cache, table, lengths, starts)
    check_attention(q, cache, table, lengths, starts)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1] * 70, [9, 4, 11], [300, 20]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_scales_that_are_none(dev, dim, counts, dtype):
    """A page whose scale is NaN, infinite or negative: the rows that see a key of it are NaN, and nobody else."""
    gen = gen_of(dev, dim + len(counts))
    heads, kv, page = 8, 2, 16
    lengths = [c + 130 + 17 * (i % 3) for i, c in enumerate(counts)]
    q, cache, table, n, starts = problem(gen, counts, lengths, heads=heads, kv=kv, dim=dim, page=page, dtype=dtype)
    for case, bad in enumerate((torch.nan, torch.inf, -torch.inf, -0.5, -2.0 ** -130)):
        for window in (None, 40):
            ref, tol, ref_lse, lse_tol, _ = L8.attention(q, cache, table, n, starts, window=window)
            s, c = case % len(counts), case % kv
            place = (1, 3, (lengths[s] - 1) // page, max(lengths[s] - counts[s] - 20, 0) // page, 0)[case]
            p = int(table[s, place])
            position = torch.arange(lengths[s] - counts[s], lengths[s], device=dev)
            sees = position >= place * page
            if window:
                sees &= position - window < (place + 1) * page - 1
            hit = torch.zeros((sum(counts), heads), dtype=torch.bool, device=dev)
            hit[int(starts[s]):int(starts[s + 1]), c * heads // kv:(c + 1) * heads // kv] = sees[:, None]
            for scales in (cache.k_scale, cache.v_scale):
                was = scales[p, c].clone()
                scales[p, c] = bad
                out, lse = ops.fp8_attention(q, cache, table, n, starts, window=window, return_lse=True)
                scales[p, c] = was
                assert out[hit].isnan().all()
                within(out[~hit], ref[~hit], tol[~hit], "out")
                if scales is cache.k_scale:
                    assert lse[hit].isnan().all()
                    within(lse[~hit], ref_lse[~hit], lse_tol[~hit], "lse")
                else:
                    within(lse, ref_lse, lse_tol, "lse")


@pytest.mark.parametrize("place", [0, 70, 140])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_one_long_sequence_among_many(dev, place, dtype):
    gen = gen_of(dev, place)
    lengths = [1 + (i * 37) % 90 for i in range(140)]
    lengths.insert(place, 20000)
    q, cache, table, n, _ = problem(gen, [1] * 141, lengths, heads=16, kv=8, dim=64, page=32, dtype=dtype)
    assert ops._fp8_attention_scratch_bytes(dev.index or 0, 141, 16, 8, 64, 141, table.shape[1], 32, 0) > 0
    check_attention(q, cache, table, n)
    check_attention(q, cache, table, n, starts_of(dev, [1] * 141), window=33)
    short = torch.arange(141, device=dev) != place
    check_attention(q[short], cache, table[short][:, :3].contiguous(), n[short])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,dim", [(16, 32), (64, 128), (256, 256)])
@pytest.mark.parametrize("seqs", [3, 70])
def test_append_to_pages_with_any_scale(dev, dtype, page, dim, seqs):
    """A begun page's scale may be no power of two: values on a border of e4m3, or next to one, are rounded as quotients."""
    gen = gen_of(dev, page + seqs)
    kv, counts = 2, [1 + i % (page // 2) for i in range(seqs)]
    cache = cache_on(gen, seqs, kv, page, dim)
    table = torch.arange(seqs, device=dev, dtype=torch.int32).view(-1, 1)
    tokens, starts = sum(counts), starts_of(dev, counts)
    held = torch.tensor([(page - n) // 2 + 1 for n in counts], device=dev)
    codes = torch.arange(0, 127, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    border = (codes[1:] + codes[:-1]) / 2
    pick = lambda *shape: border[torch.randint(len(border), shape, generator=gen, device=dev)]  # noqa: E731
    odd = torch.tensor([1.25, 1.5, 1.75], device=dev, dtype=torch.float64)
    scale = odd[torch.randint(3, (seqs, kv), generator=gen, device=dev)] * 0.25
    of = torch.repeat_interleave(torch.arange(seqs, device=dev), torch.tensor(counts, device=dev))
    # few-bit scales: the border times the scale is a 16-bit number, and lies on the border again when it is divided
    cache.k_scale.copy_(scale)
    cache.v_scale.copy_(scale)
    k, v = ((pick(tokens, kv, dim) * scale[of][:, :, None]).to(dtype) for _ in range(2))
    check_append(k, v, cache, table, (held + torch.tensor(counts, device=dev)).int(), starts)
    # 24-bit scales, a new value that makes them grow to a power of two: an old code, a small whole number, comes next to a
    # border, on the one side of it or the other
    cache.k.copy_(cache.k.float().clamp(1, 15).round().to(cache.k.dtype))
    cache.v.copy_(cache.v.float().clamp(1, 15).round().to(cache.v.dtype))
    by = (pick(seqs, kv) / torch.randint(1, 16, (seqs, kv), generator=gen, device=dev)).float()
    by = by / torch.exp2(torch.ceil(torch.log2(by)))                            # a half to one
    cache.k_scale.copy_(by)
    cache.v_scale.copy_(by)
    k, v = (torch.randn((tokens, kv, dim), generator=gen, device=dev) for _ in range(2))
    k[..., 0], v[..., 0] = 448, 448                                             # the scale 1
    check_append(k.to(dtype), v.to(dtype), cache, table, (held + torch.tensor(counts, device=dev)).int(), starts)
    # 24-bit scales that stay
    cache.k_scale.copy_(by * 8)
    cache.v_scale.copy_(by * 8)
    check_append(k.to(dtype), v.to(dtype), cache, table, (held + torch.tensor(counts, device=dev)).int(), starts)
