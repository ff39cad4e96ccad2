"""CPU tests of the norm, the 8-bit cache and the attention over it: refusals of the torch entry points and of the C ABI."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import _lib, ops

E4M3 = torch.float8_e4m3fn


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return z(*shape, dtype=torch.int32)


def test_no_cpu_fallback():
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_norm(z(2, 128), z(128))
    cache = ops.fp8_cache(4, 2, 16, 64, device="cpu")
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_cache_append(z(2, 2, 64), z(2, 2, 64), cache, i32(2, 2), i32(2))
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_attention(z(2, 4, 64), cache, i32(2, 2), i32(2))


@pytest.mark.parametrize("kw", [
    {"x": z(2, 128, dtype=torch.float64)}, {"x": z(4, 256)[:, ::2]}, {"x": z(128, 2).t()}, {"x": z(2, 0), "weight": z(0)},
    {"x": torch.tensor(1.0)}, {"weight": z(127)}, {"weight": z(1, 128)}, {"weight": z(256)[::2]},
    {"weight": z(128, dtype=torch.float64)}, {"residual": z(2, 127)}, {"residual": z(2, 128, dtype=torch.float16)},
    {"residual": z(128, 2).t()}, {"eps": -1e-6}, {"eps": float("nan")}, {"eps": float("inf")},
    {"normed_dtype": torch.float64}, {"normed_dtype": E4M3}])
def test_norm_refuses(kw):
    with pytest.raises(RuntimeError):
        ops.fp8_norm(**{"x": z(2, 128), "weight": z(128), **kw})


@pytest.mark.parametrize("kw", [{"page": 8}, {"page": 48}, {"page": 512}, {"dim": 0}, {"dim": 24}, {"dim": 272}, {"pages": 0},
                                {"kv_heads": 0}, {"kv_heads": 1025}])
def test_cache_refuses(kw):
    with pytest.raises(RuntimeError):
        ops.fp8_cache(**{"pages": 4, "kv_heads": 2, "page": 16, "dim": 64, "device": "cpu", **kw})


def args(**change):
    c = ops.fp8_cache(4, 2, 16, 64, device="cpu")
    a = {"k": c.k, "k_scale": c.k_scale, "v": c.v, "v_scale": c.v_scale, "table": i32(3, 2), "lengths": i32(3), "starts": None}
    a.update(change)
    return ops.Fp8Cache(a["k"], a["k_scale"], a["v"], a["v_scale"]), a["table"], a["lengths"], a["starts"]


def f8(*shape):
    return z(*shape, dtype=torch.uint8).view(E4M3)


BAD_CACHES = [
    {"k": z(4, 2, 16, 64)}, {"k": f8(4, 2, 64, 16)}, {"k": f8(4, 2, 16, 128)[..., ::2]}, {"k": f8(0, 2, 16, 64)},
    {"v": f8(4, 2, 16, 64)}, {"v": f8(3, 2, 64, 16)}, {"k_scale": torch.zeros(4, 1)}, {"v_scale": torch.zeros(2, 4).t()},
    {"v_scale": torch.zeros(4, 2).half()}, {"table": i32(3)}, {"table": i32(3, 2).long()}, {"table": i32(3, 4)[:, ::2]},
    {"table": i32(3, 0)}, {"lengths": i32(2)}, {"lengths": i32(3).long()}, {"lengths": i32(6)[::2]},
    {"starts": i32(3)}, {"starts": i32(4).long()}, {"table": i32(2, 2), "lengths": i32(2)}]


@pytest.mark.parametrize("change", BAD_CACHES)
def test_append_refuses_the_cache(change):
    with pytest.raises(RuntimeError, match="must|without"):
        ops.fp8_cache_append(z(3, 2, 64), z(3, 2, 64), *args(**change))


@pytest.mark.parametrize("change", BAD_CACHES)
def test_attention_refuses_the_cache(change):
    with pytest.raises(RuntimeError, match="must|without"):
        ops.fp8_attention(z(3, 4, 64), *args(**change))


@pytest.mark.parametrize("k,v", [(z(3, 2, 48), z(3, 2, 48)), (z(3, 1, 64), z(3, 1, 64)), (z(3, 128), z(3, 128)),
                                 (z(3, 2, 64), z(3, 2, 64, dtype=torch.float16)), (z(3, 2, 64), z(2, 2, 64)),
                                 (z(3, 2, 64, dtype=torch.float64), z(3, 2, 64, dtype=torch.float64))])
def test_append_refuses(k, v):
    with pytest.raises(RuntimeError, match="must"):
        ops.fp8_cache_append(k, v, *args())


@pytest.mark.parametrize("kw", [
    {"q": z(3, 4, 64, dtype=torch.float32)}, {"q": z(3, 256)}, {"q": z(3, 3, 64)}, {"q": z(3, 1, 64)}, {"q": z(3, 4, 48)},
    {"scale": float("nan")}, {"window": 0}, {"window": -1}, {"window": 1 << 31}, {"sinks": torch.zeros(3)},
    {"sinks": torch.zeros(4).half()}, {"out": z(3, 4, 48)}, {"out": z(3, 4, 64, dtype=torch.float16)},
    {"out": z(4, 3, 64).transpose(0, 1)}])
def test_attention_refuses(kw):
    kw = dict(kw)
    with pytest.raises(RuntimeError, match="must"):
        ops.fp8_attention(kw.pop("q", z(3, 4, 64)), *args(), **kw)


P = 1 << 12          # an aligned stand-in for a device address: every call below is refused before a launch


def refused(rc, msg):
    assert rc < 0
    assert msg in (_lib.load().exl3_last_error() or b"").decode()


@pytest.mark.parametrize("change,msg", [
    ({"x": None}, "null"), ({"weight": None}, "null"), ({"residual": P, "total": None}, "null"), ({"x_kind": 3}, "x_kind"),
    ({"w_kind": -1}, "weight_kind"), ({"residual": P, "r_kind": 0}, "residual_kind"), ({"normed": P, "n_kind": 3}, "normed_kind"),
    ({"rows": 0}, "positive"), ({"k": 0}, "positive"), ({"k": (1 << 24) + 1}, "2^24"), ({"rows": 1 << 40}, "too many"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps")])
def test_norm_argument_errors_without_device(change, msg):
    a = {"x": P, "x_kind": 1, "residual": None, "r_kind": 1, "weight": P, "w_kind": 2, "rows": 2, "k": 128, "eps": 1e-6,
         "total": P, "normed": None, "n_kind": 0, **change}
    refused(_lib.load().exl3_fp8_norm(a["x"], a["x_kind"], a["residual"], a["r_kind"], a["weight"], a["w_kind"], a["rows"],
                                      a["k"], a["eps"], 0, P, P, a["total"], a["normed"], a["n_kind"], None), msg)


CACHE = {"pages": 4, "kv": 2, "page": 16, "dim": 64, "table": P, "stride": 2, "width": 2, "lengths": P, "starts": None,
         "seqs": 3, "tokens": 3, "cache": P, "kind": 1}
CACHE_ERRORS = [
    ({"cache": None}, "null"), ({"table": None}, "null"), ({"lengths": None}, "null"), ({"pages": 0}, "pages"),
    ({"pages": 1 << 31}, "pages"), ({"kv": 0}, "kv_heads"), ({"kv": 2000, "heads": 2000}, "kv_heads"), ({"page": 48}, "page_size"),
    ({"page": 8}, "page_size"), ({"dim": 40}, "dim"), ({"dim": 512}, "dim"), ({"width": 0}, "table"),
    ({"width": 1 << 28}, "table"), ({"seqs": 0}, "seqs"), ({"seqs": 2}, "one token"), ({"tokens": 0}, "tokens"),
    ({"tokens": 1 << 23, "starts": P}, "tokens"), ({"cache": P + 8}, "aligned"), ({"kind": 4}, "kind")]


def cache_of(a):
    return (a["cache"], P, a["cache"], P, a["pages"], a["kv"], a["page"], a["dim"], a["table"], a["stride"], a["width"],
            a["lengths"], a["starts"], a["seqs"])


@pytest.mark.parametrize("change,msg", [*CACHE_ERRORS, ({"k": None}, "null"), ({"k": P + 2}, "aligned"), ({"row": 68}, "aligned")])
def test_append_argument_errors_without_device(change, msg):
    a = {**CACHE, "k": P, "row": 128, **change}
    refused(_lib.load().exl3_fp8_cache_append(a["k"], a["row"], 64, P, 128, 64, a["kind"], a["tokens"], *cache_of(a), None), msg)


@pytest.mark.parametrize("change,msg", [
    *CACHE_ERRORS, ({"kind": 2}, "kind"), ({"q": None}, "null"), ({"heads": 3}, "multiple"), ({"heads": 1}, "multiple"),
    ({"scale": float("inf")}, "scale"), ({"window": -1}, "window"), ({"window": 1 << 31}, "window"), ({"q": P + 8}, "aligned"),
    ({"row": 260}, "aligned"), ({"scratch": None}, "null"), ({"scratch": P + 4}, "aligned"), ({"bytes": 64}, "too small"),
    ({"heads": 65536, "kv": 1, "tokens": 40000, "starts": P}, "too many rows")])
def test_attention_argument_errors_without_device(change, msg):
    a = {**CACHE, "q": P, "row": 256, "heads": 4, "scale": 1.0, "window": 0, "scratch": P, "bytes": 1 << 40, **change}
    refused(_lib.load().exl3_fp8_attention(a["q"], a["kind"], a["row"], 64, a["tokens"], a["heads"], *cache_of(a), a["scale"],
                                           a["window"], None, P, None, 0, a["scratch"], a["bytes"], None), msg)


def test_attention_scratch_refuses():
    L = _lib.load()
    good = (3, 4, 2, 64, 3, 2, 16, 0)
    assert L.exl3_fp8_attention_scratch_bytes(*good) > 0
    for i, v in ((0, 0), (0, 1 << 23), (1, 3), (1, 0), (2, 0), (3, 20), (4, 0), (5, 0), (6, 0), (6, 512), (7, -1)):
        refused(L.exl3_fp8_attention_scratch_bytes(*good[:i], v, *good[i + 1:]), "out of range")


def test_attention_scratch_goes_by_the_calls_device(monkeypatch):
    """How the work is shared out depends on the number of CUs: that of the call's own device, whichever is current."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Lib:
        def exl3_fp8_attention_scratch_bytes(self, *_):
            return 1000 + current[-1]

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "load", Lib)
    ops._fp8_attention_scratch_bytes.cache_clear()
    assert [ops._fp8_attention_scratch_bytes(i, 3, 4, 2, 64, 3, 2, 16, 0) for i in (1, 0, 1)] == [1001, 1000, 1001]
    ops._fp8_attention_scratch_bytes.cache_clear()
