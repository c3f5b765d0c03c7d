"""Calls of the linears whose weights depend on the row that a program makes around them:
traced by torch.compile, and with arguments of another layout than the documented one."""
from __future__ import annotations

import pytest
import torch

import fp8linear_b200 as f
from tests.helpers import require_sm100

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    require_sm100()


def test_compile_fullgraph():
    g = torch.Generator(device="cuda").manual_seed(0)
    M, K, N, E, L, R = 70, 128, 96, 5, 3, 16
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(E, N, K, generator=g, device="cuda").bfloat16()
    offsets = torch.tensor([0, 10, 10, 40, 69, 70], dtype=torch.int32, device="cuda")
    bias = torch.randn(E, N, generator=g, device="cuda").bfloat16()
    a = torch.randn(L, R, K, generator=g, device="cuda").bfloat16()
    b = torch.randn(L, N, R, generator=g, device="cuda").bfloat16()
    ids = (torch.arange(M, device="cuda") % 4 - 1).int()
    scaling = torch.ones(L, device="cuda")

    def fn(x):
        wq, ws = f.quantize_expert_weights(w)
        xq, xs = f.quantize_fp8(x)
        y = f.fp8_linear_lora(x.view(2, 35, K), wq[0], ws[0], a, b, ids, scaling, bias[0])
        return (f.fp8_grouped_linear(x, wq, ws, offsets, bias) * 2.0,
                f.fp8_grouped_gemm(xq, xs, wq, ws, offsets) + 1.0, y, wq.view(torch.uint8), ws)

    eager = fn(x)
    out = torch.compile(fn, fullgraph=True, backend="aot_eager")(x)
    for o, r in zip(out, eager):
        assert o.dtype == r.dtype and o.shape == r.shape
        assert torch.equal(o, r)


def test_scales_of_another_layout_are_refused():
    """As many scales as experts times channels, but not expert by expert."""
    E, N, K = 3, 8, 32
    wq = torch.zeros(E, N, K, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ws = torch.ones(E, N, device="cuda")
    x = torch.zeros(4, K, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    for same in (ws[:, :, None], ws.view(-1)):
        assert f.fp8_grouped_linear(x, wq, same, offsets).shape == (4, N)
    xq, xs = f.quantize_fp8(x)
    for bad in (ws.t(), ws.t().contiguous(), ws.view(1, E * N), ws.view(E * 2, N // 2),
                ws.view(E, 2, N // 2)):
        with pytest.raises(RuntimeError, match="w_scale"):
            f.fp8_grouped_linear(x, wq, bad, offsets)
        with pytest.raises(RuntimeError, match="w_scale"):
            f.fp8_grouped_gemm(xq, xs, wq, bad, offsets)


def test_adapters_of_another_layout_are_refused():
    """As many entries as rows, but not in the rows' order."""
    K, N = 32, 8
    wq = torch.zeros(N, K, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ws = torch.ones(N, device="cuda")
    x = torch.randn(2, 5, K, device="cuda").half()
    a = torch.randn(3, 8, K, device="cuda").half()
    b = torch.randn(3, N, 8, device="cuda").half()
    ids = (torch.arange(10, device="cuda") % 4 - 1).int()
    sc = torch.ones(3, device="cuda")
    ref = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc)
    for same in (ids.view(2, 5), ids.view(2, 5, 1), ids.view(10, 1), ids.view(1, 2, 5)):
        assert torch.equal(f.fp8_linear_lora(x, wq, ws, a, b, same, sc), ref)
    assert torch.equal(f.fp8_linear_lora(x.view(10, K), wq, ws, a, b, ids.view(1, 10), sc),
                       ref.view(10, N))
    for bad in (ids.view(5, 2), ids.view(2, 5).t()):
        with pytest.raises(RuntimeError, match="adapters"):
            f.fp8_linear_lora(x, wq, ws, a, b, bad, sc)
