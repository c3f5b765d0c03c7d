"""Linears whose weights depend on the row, without a GPU: public names, fake
implementations, refusals of the C entry points before any CUDA call."""
from __future__ import annotations

import ctypes

import pytest
import torch

import fp8linear_b200 as f

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def api():
    from fp8linear_b200.capi import CApi

    return CApi()


def test_public_names():
    for n in ("fp8_grouped_gemm", "fp8_grouped_linear", "fp8_linear_lora",
              "quantize_expert_weights"):
        assert n in f.__all__ and callable(getattr(f, n))


def test_fake_impls():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(40, 256, dtype=torch.float16)
        wq, ws = f.quantize_expert_weights(torch.empty(6, 96, 256, dtype=torch.bfloat16))
        assert wq.shape == (6, 96, 256) and wq.dtype == torch.float8_e4m3fn
        assert ws.shape == (6, 96) and ws.dtype == torch.float32
        off = torch.empty(7, dtype=torch.int32)
        out = f.fp8_grouped_linear(x, wq, ws, off)
        assert out.shape == (40, 96) and out.dtype == torch.float16
        xq, xs = f.quantize_fp8(x)
        assert f.fp8_grouped_gemm(xq, xs, wq, ws, off).dtype == torch.bfloat16
        a, b = torch.empty(3, 16, 256, dtype=x.dtype), torch.empty(3, 96, 16, dtype=x.dtype)
        y = f.fp8_linear_lora(x.view(4, 10, 256), wq[0], ws[0], a, b,
                              torch.empty(40, dtype=torch.int32), torch.empty(3))
        assert y.shape == (4, 10, 96) and y.dtype == torch.float16


def test_cpu_tensors_fail_loudly():
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    wq = torch.zeros(2, 8, 32, dtype=torch.float8_e4m3fn)
    with pytest.raises((RuntimeError, NotImplementedError)):
        f.fp8_grouped_linear(x, wq, torch.ones(2, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises((RuntimeError, NotImplementedError)):
        f.fp8_linear_lora(x, wq[0], torch.ones(8), torch.zeros(1, 8, 32), torch.zeros(1, 8, 8),
                          torch.zeros(4, dtype=torch.int32), torch.ones(1))
    with pytest.raises((RuntimeError, NotImplementedError)):
        f.quantize_expert_weights(torch.zeros(2, 8, 32))


def grouped(api, *, xq=P, xs=P, wq=P, ws=P, off=P, bias=None, bd=-1, out=P, od=0, M=4, N=8, K=32,
            E=2):
    xs, ws, off = (ctypes.cast(v, ctypes.c_void_p) if v else None for v in (xs, ws, off))
    return api.lib.fp8lin_fp8_grouped_gemm(xq, xs, wq, ws, off, bias, bd, out, od, M, N, K, E, None)


def test_grouped_refusals(api):
    assert grouped(api, M=0) == 0 and grouped(api, N=0) == 0
    assert grouped(api, M=-1) == 1 and grouped(api, od=2) == 1
    assert grouped(api, bias=P, bd=9) == 1
    assert grouped(api, K=24) == 2 and grouped(api, K=0) == 2
    assert grouped(api, E=0) == 2 and grouped(api, E=1025) == 2
    assert "experts" in api.last_error()
    for dim in ("M", "N"):
        for size in (2**31, 2**31 - 1023):
            assert grouped(api, **{dim: size}) == 2 and "int32" in api.last_error()
    assert grouped(api, K=2**31 - 16) == 2 and "int32" in api.last_error()
    odd = ctypes.c_void_p(257)
    assert grouped(api, xs=odd) == 2 and grouped(api, ws=odd) == 2
    assert grouped(api, bias=odd, bd=0) == 2 and grouped(api, bias=ctypes.c_void_p(258), bd=2) == 2
    for name in ("xq", "xs", "wq", "ws", "off", "out"):
        assert grouped(api, **{name: None}) == 1, name
    assert grouped(api, xq=ctypes.c_void_p(264)) == 2 and grouped(api, off=ctypes.c_void_p(258)) == 2


def test_grouped_linear_refusals(api):
    def call(x=P, xd=0, ws=P, nbytes=1 << 20, M=4, E=2):
        return api.lib.fp8lin_fp8_grouped_linear(x, xd, P, P, P, None, -1, P, 0, M, 8, 32, E, ws,
                                                 nbytes, None)

    assert call(M=0) == 0
    assert call(xd=2) == 1 and call(x=None) == 1 and call(E=0) == 2
    assert call(ws=None) == 3 and call(nbytes=511) == 3 and call(ws=ctypes.c_void_p(264)) == 3
    assert "workspace" in api.last_error()


def test_lora_refusals(api):
    def call(x=P, xd=0, a=P, b=P, ids=P, sc=P, M=4, K=32, L=2, R=16, ws=P, nbytes=1 << 20):
        return api.lib.fp8lin_fp8_linear_lora(x, xd, P, P, a, b, ids, sc, None, -1, P, 0, M, 8, K,
                                              L, R, ws, nbytes, None)

    assert call(M=0) == 0
    assert call(xd=2) == 1 and call(L=-1) == 1 and call(R=-8) == 1 and call(M=-1) == 1
    assert call(K=40) == 2
    for R in (0, 4, 12, 136):
        assert call(R=R) == 2 and "rank" in api.last_error()
    assert call(M=2**31) == 2 and call(M=2**31 - 1023) == 2 and call(L=2**31) == 2
    assert call(ids=ctypes.c_void_p(258)) == 2 and call(sc=ctypes.c_void_p(258)) == 2
    for name in ("x", "a", "b", "ids", "sc"):
        assert call(**{name: None}) == 1, name
    odd = ctypes.c_void_p(264)
    assert call(x=odd) == 2 and call(a=odd) == 2 and call(b=odd) == 2
    assert call(ws=None) == 3 and call(ws=odd) == 3
    need = api.lora_workspace_size(4, 32, 16)
    assert call(nbytes=need - 1) == 3 and str(need) in api.last_error()


def test_lora_workspace_size(api):
    size = api.lora_workspace_size
    assert size(0, 32, 16) == 0
    assert size(5, 64, 0) == api.workspace_size(5, 64)
    # h in two parts with the rank padded to 16 and a scale per row; above 64 rows the plan of
    # the token tiles (16 bytes each: a header, tiles of 160 and one per 32 rows for the runs'
    # ends, two per 32 rows and one for the gaps); all rounded up to 256 bytes
    base = api.workspace_size(64, 64)
    assert size(64, 64, 24) - base == 64 * 2 * 32 * 2 + 256
    base = api.workspace_size(1000, 64)
    plan = 16 * (1 + 1000 // 160 + 1000 // 32 + 2 * (1000 // 32) + 1)
    assert size(1000, 64, 24) - base == 1000 * 128 + 4096 + (plan + 255) // 256 * 256
