"""Borders of the 8-bit cache and the attention over it that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dsv4_carve_amd import _lib, build, ops
from tests.test_layer8 import CACHE, P, args, cache_of, i32, refused, z


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("tokens", [0, 3])
def test_attention_without_sequences_fills_the_logarithms(given, tokens):
    """They are the call's own whether `out` is or not: without a sequence all are -inf, and only an `out` given stays."""
    q = z(tokens, 4, 64) + 1
    out = torch.full_like(q, 7.0) if given else None
    torch.use_deterministic_algorithms(True)             # fills what is not initialised with NaN
    try:
        made, lse = ops.fp8_attention(q, *args(table=i32(0, 2), lengths=i32(0), starts=i32(1)), out=out, return_lse=True)
    finally:
        torch.use_deterministic_algorithms(False)
    assert lse.shape == (tokens, 4) and (lse == -torch.inf).all()
    assert (made == (7.0 if given else 0.0)).all() and (not given or made is out)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_a_tables_room_ends_before_the_kernels_32_bit_places_do(page):
    """Blocks of 64 keys, and those that a wave asks for ahead (up to 8 blocks), are counted in 32 bits."""
    L, most = _lib.load(), ((1 << 31) - 1024) // page
    assert most * page + 64 * 9 < 1 << 31
    assert L.exl3_fp8_attention_scratch_bytes(3, 4, 2, 64, 3, most, page, 0) > 0
    refused(L.exl3_fp8_attention_scratch_bytes(3, 4, 2, 64, 3, most + 1, page, 0), "out of range")
    a = {**CACHE, "page": page, "width": most + 1}
    refused(L.exl3_fp8_cache_append(P, 128, 64, P, 128, 64, 1, 3, *cache_of(a), None), "2^31-1024")
    refused(L.exl3_fp8_attention(P, 1, 256, 64, 3, 4, *cache_of(a), 1.0, 0, None, P, None, 0, P, 1 << 40, None), "2^31-1024")


@pytest.mark.parametrize("heads", [1, 2, 3, 4, 5, 7, 8, 9, 16, 24, 32, 40, 128])
def test_every_tile_has_one_workgroup(heads):
    """A workgroup a tile: the launch's padding has no tile a second time, and none is left out."""
    probe = ctypes.CDLL(build.PROBE_LIB)
    for tiles in [*range(1, 42), 127, 128, 129, 300, 1025]:
        grid = probe.exl3_probe_tile_grid(tiles, heads)
        got = [probe.exl3_probe_tile_by_xcd(b, tiles, heads) for b in range(grid)]
        assert sorted(t for t in got if t >= 0) == list(range(tiles * heads)), tiles


def test_workgroups_of_an_xcd_are_neighbours():
    probe = ctypes.CDLL(build.PROBE_LIB)
    for n in [*range(1, 70), 511, 512, 513]:
        assert sorted(probe.exl3_probe_by_xcd(b, n) for b in range(n)) == list(range(n))
        for x in range(min(8, n)):
            mine = [probe.exl3_probe_by_xcd(b, n) for b in range(x, n, 8)]
            assert mine == list(range(mine[0], mine[0] + len(mine)))


@pytest.mark.parametrize("seqs,heads,kv,dim,keys,shared", [
    (300, 32, 8, 128, 512, False), (300, 32, 8, 128, 131072, True), (129, 32, 8, 128, 16384, True), (256, 32, 8, 128, 4096, False),
    (128, 32, 8, 128, 8192, True), (256, 32, 8, 128, 8192, True), (128, 32, 8, 128, 2048, False), (64, 32, 8, 128, 8192, True),
    (4096, 8, 2, 128, 16384, False), (4096, 8, 2, 128, 1 << 20, True), (1 << 20, 8, 8, 64, 1 << 18, True)])
def test_a_long_sequence_among_single_tokens_is_shared_out(seqs, heads, kv, dim, keys, shared):
    """A workgroup a tile, which needs no scratch, only where the longest sequence that the table has room for takes no more
    time than the launch's rounds, and the tiles are a launch (2^20 of 8 heads are not: (2^16 + 2^20) * 8 > 2^23)."""
    need = _lib.load().exl3_fp8_attention_scratch_bytes
    assert (need(seqs, heads, kv, dim, seqs, keys // 64, 64, 0) > 0) == shared
    assert need(seqs, heads, kv, dim, seqs, (1 << 20) // 64, 64, 512) == need(seqs, heads, kv, dim, seqs, (1 << 24) // 64, 64, 512)
