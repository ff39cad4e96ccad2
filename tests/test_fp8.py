"""CPU tests of the block-scaled 8-bit operators and the router: refusals of the torch entry points and of the C ABI."""

from __future__ import annotations

import pytest
import torch

from dsv4_carve_amd import _lib, ops

E4M3 = torch.float8_e4m3fn


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def f8(*shape):
    return z(*shape, dtype=torch.uint8).view(E4M3)


@pytest.mark.parametrize("x", [z(2, 128, dtype=torch.float64), z(4, 256)[:, ::2], z(128, 2).t(), z(2, 0), torch.tensor(1.0)])
def test_quantize_refuses(x):
    with pytest.raises(RuntimeError):
        ops.fp8_quantize(x)


def gemm_args(**change):
    a = {"a": f8(3, 256), "a_scale": torch.ones(3, 2), "w": f8(200, 256), "w_scale": torch.ones(2, 2), "c": z(3, 200)}
    return {**a, **change}


@pytest.mark.parametrize("change", [
    {"a": z(3, 256)}, {"a": f8(3, 512)[:, ::2]}, {"a": f8(3, 264), "w": f8(200, 264)}, {"a": f8(256)},
    {"a": f8(3, 240)}, {"a_scale": torch.ones(3, 1)}, {"a_scale": torch.ones(2, 3).t()},
    {"a_scale": torch.ones(3, 2, dtype=torch.float64)}, {"w": f8(200, 128)}, {"w": f8(256, 200).t()}, {"w": z(200, 256)},
    {"w_scale": torch.ones(2, 3)}, {"w_scale": torch.ones(200, 2)}, {"w_scale": torch.ones(2, 2).half()},
    {"c": z(3, 199)}, {"c": z(200, 3).t()}, {"c": z(3, 200, dtype=torch.float64)}])
def test_gemm_refuses(change):
    with pytest.raises(RuntimeError):
        ops.fp8_gemm_into(**gemm_args(**change))


@pytest.mark.parametrize("x,dtype", [(z(2, 264), None), (z(2, 128), None), (z(512, 2).t(), None), (z(2, 256), torch.float64),
                                     (z(2, 256, dtype=torch.float64), None), (f8(2, 256), None)])
def test_linear_refuses(x, dtype):
    with pytest.raises(RuntimeError):
        ops.fp8_linear(x, f8(48, 256), torch.ones(1, 2), out_dtype=dtype)


@pytest.mark.parametrize("kw", [{"topk": 0}, {"topk": 9}, {"scoring": "relu"}, {"ids_dtype": torch.int16},
                                {"scale": float("inf")}, {"scale": float("nan")}, {"bias": torch.zeros(7)},
                                {"bias": torch.zeros(8).half()}, {"logits": torch.zeros(2, 2049)},
                                {"logits": torch.zeros(8)}, {"logits": torch.zeros(8, 2).t()},
                                {"logits": torch.zeros(2, 8, dtype=torch.int32)}, {"logits": torch.zeros(2, 0)}])
def test_route_refuses(kw):
    with pytest.raises(RuntimeError):
        ops.moe_route(**{"logits": torch.zeros(2, 8), "topk": 2, **kw})


def test_no_cpu_fallback():
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_quantize(z(1, 128))
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_gemm_into(**gemm_args())
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.fp8_linear(z(2, 256), f8(48, 256), torch.ones(1, 2))
    with pytest.raises((NotImplementedError, RuntimeError)):
        ops.moe_route(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="HIP"):
        ops.fp8_moe(z(1, 128), f8(2, 256, 128), torch.ones(2, 2, 1), f8(2, 128, 128), torch.ones(2, 1, 1),
                    torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, 1))


P = 1 << 12          # an aligned stand-in for a device address: every call below is refused before a launch


def refused(rc, msg):
    assert rc < 0
    assert msg in (_lib.load().exl3_last_error() or b"").decode()


@pytest.mark.parametrize("change,msg", [({"x": None}, "null"), ({"kind": 3}, "x_kind"), ({"rows": 0}, "positive"),
                                        ({"k": 0}, "positive"), ({"k": (1 << 24) + 1}, "2^24"), ({"rows": 1 << 60}, "too many")])
def test_quantize_argument_errors_without_device(change, msg):
    a = {"x": P, "kind": 1, "rows": 2, "k": 128, **change}
    refused(_lib.load().exl3_fp8_quantize(a["x"], a["kind"], a["rows"], a["k"], 0, P, P, None), msg)


@pytest.mark.parametrize("change,msg", [({"a": None}, "null"), ({"m": 0}, "positive"), ({"n": 0}, "positive"),
                                        ({"k": 8}, "multiple of 16"), ({"k": 24}, "multiple of 16"),
                                        ({"k": (1 << 24) + 16}, "2^24"), ({"m": 1 << 20}, "1048560"), ({"kind": 5}, "c_kind"),
                                        ({"a": P + 1}, "aligned"), ({"w": P + 8}, "aligned"), ({"c": P + 4}, "aligned")])
def test_gemm_argument_errors_without_device(change, msg):
    a = {"a": P, "m": 2, "k": 128, "w": P, "n": 16, "c": P, "kind": 1, **change}
    L = _lib.load()
    refused(L.exl3_fp8_gemm(a["a"], P, a["m"], a["k"], a["w"], P, a["n"], a["c"], a["kind"], None), msg)
    if "a" not in change:
        refused(L.exl3_fp8_linear(P, 1, a["m"], a["k"], a["w"], P, a["n"], a["c"], a["kind"], P, 1 << 40, None), msg)


def test_linear_scratch_is_checked():
    L = _lib.load()
    need = L.exl3_fp8_linear_scratch_bytes(50, 400, 64)
    assert need >= 50 * 400 + 50 * 4 * 4
    refused(L.exl3_fp8_linear(P, 1, 50, 400, P, P, 64, P, 1, P, need - 1, None), "scratch too small")
    refused(L.exl3_fp8_linear(P, 1, 50, 400, P, P, 64, P, 1, P + 4, need, None), "aligned")
    refused(L.exl3_fp8_linear(P, 1, 50, 400, P, P, 64, P, 1, None, need, None), "null")
    refused(L.exl3_fp8_linear(P + 2, 1, 5, 400, P, P, 64, P, 1, P, need, None), "aligned")
    assert L.exl3_fp8_linear_scratch_bytes(1, 4096, 4096) == 0
    refused(L.exl3_fp8_linear_scratch_bytes(5, 40, 64), "multiple of 16")


def test_linear_scratch_goes_by_the_calls_device(monkeypatch):
    """Whether a call needs scratch depends on the number of CUs: that of its own device, whichever is current."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Lib:
        def exl3_fp8_linear_scratch_bytes(self, m, k, n):
            return 1000 + current[-1]

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "load", Lib)
    ops._fp8_linear_scratch_bytes.cache_clear()
    assert [ops._fp8_linear_scratch_bytes(i, 2, 256, 64) for i in (1, 0, 1)] == [1001, 1000, 1001]
    ops._fp8_linear_scratch_bytes.cache_clear()


MOE = {"x": P, "x_kind": 1, "out_kind": 1, "rows": 2, "hidden": 256, "inter": 128, "E": 4, "topk": 2, "ids_kind": 0,
       "w_kind": 2, "emap": None, "n_global": 0, "limit": 1.0, "scratch": P, "bytes": 1 << 20}


@pytest.mark.parametrize("change,msg", [
    ({"x": None}, "null"), ({"x_kind": 2}, "x_kind"), ({"out_kind": 3}, "out_kind"), ({"rows": 0}, "row count"),
    ({"rows": 65}, "row count"), ({"topk": 0}, "topk"), ({"topk": 17}, "topk"), ({"inter": 64}, "intermediate"),
    ({"hidden": 192}, "hidden"), ({"hidden": 1 << 21}, "2^20"), ({"E": 0}, "n_experts"), ({"limit": 0.0}, "swiglu_limit"),
    ({"limit": float("nan")}, "swiglu_limit"), ({"bytes": 2047}, "scratch too small"), ({"scratch": P + 8}, "aligned"),
    ({"x": P + 2}, "aligned"), ({"ids_kind": 2}, "int32 or int64"), ({"w_kind": 3}, "routing weights"),
    ({"emap": P, "n_global": 0}, "expert map")])
def test_moe_argument_errors_without_device(change, msg):
    a = {**MOE, **change}
    refused(_lib.load().exl3_fp8_moe(a["x"], a["x_kind"], P, a["out_kind"], a["rows"], a["hidden"], a["inter"], a["E"],
                                     a["topk"], P, P, P, P, P, a["ids_kind"], P, a["w_kind"], a["emap"], a["n_global"],
                                     a["limit"], a["scratch"], a["bytes"], None), msg)


def test_moe_limits_agree():
    L = _lib.load()
    assert L.exl3_fp8_moe_max_rows() == ops.FP8_MOE_MAX_ROWS
    assert L.exl3_fp8_moe_scratch_bytes(64, ops.FP8_MOE_MAX_TOPK, 128) == 64 * 16 * 128 * 4


@pytest.mark.parametrize("change,msg", [({"logits": None}, "null"), ({"kind": 3}, "logits_kind"), ({"ids": 2}, "ids_kind"),
                                        ({"scoring": 3}, "scoring"), ({"E": 2049}, "2048"), ({"rows": 0}, "rows"),
                                        ({"topk": 0}, "topk"), ({"topk": 9}, "topk"), ({"topk": 65, "E": 100}, "topk"),
                                        ({"scale": float("nan")}, "finite")])
def test_route_argument_errors_without_device(change, msg):
    a = {"logits": P, "kind": 2, "rows": 3, "E": 8, "topk": 2, "scoring": 0, "scale": 1.0, "ids": 0, **change}
    refused(_lib.load().exl3_moe_route(a["logits"], a["kind"], a["rows"], a["E"], a["topk"], a["scoring"], None, 1,
                                       a["scale"], P, a["ids"], P, None), msg)


def test_route_refuses_rows_past_any_memory():
    refused(_lib.load().exl3_moe_route(P, 1, (1 << 36) + 1, 1, 1, 0, None, 1, 1.0, P, 0, P, None), "too many rows")
