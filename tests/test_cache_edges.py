"""Borders of the 8-bit cache and the attention over it that need no GPU."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import ops
from tests.test_layer8 import args, i32, z


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
