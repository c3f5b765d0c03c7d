"""The linears whose weights depend on the row, where element offsets pass 32 bits."""
from __future__ import annotations

import pytest
import torch

import fp8linear_b200 as f
from tests.helpers import require_sm100, torch_quant_ref
from tests.rowsel_helpers import base_rows, check, lora_ref, quantized_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    require_sm100()


@pytest.fixture(autouse=True)
def _no_timeouts(capi):
    yield
    assert capi.device_status(clear=True) == 0
    torch.cuda.empty_cache()


K = 16


def sampled(M):
    """Rows at both ends and around the output's 2^31st element."""
    return torch.tensor([0, 1, M // 2, 65535, 65536, 65537, M - 2, M - 1], device="cuda")


def test_grouped_output_past_2_31():
    M, N = 70000, 32770  # 2.29e9 elements
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wq, ws = quantized_weight(g, 2, N, K)
    offsets = torch.tensor([0, 66000, M - 1], dtype=torch.int32, device="cuda")
    out = f.fp8_grouped_linear(x, wq, ws, offsets)
    rows = sampled(M)[:-1]
    xq, xs = torch_quant_ref(x[rows])
    for e in range(2):
        of = (rows >= 66000) == bool(e)
        check(out[rows[of]], *base_rows(xq[of], xs[of], wq[e], ws[e], None))
    assert int(torch.count_nonzero(out[M - 1])) == 0  # of no expert


def test_lora_output_past_2_31():
    M, N = 70000, 32776
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.float16)
    wq, ws = quantized_weight(g, N, K)
    a = torch.randn(3, 8, K, generator=g, device="cuda").half()
    b = (torch.randn(3, N, 8, generator=g, device="cuda") * 0.1).half()
    sc = torch.ones(3, device="cuda")
    ids = (torch.arange(M, device="cuda") // 30000).int()
    ids[65530:65540] = torch.arange(10, device="cuda").int() % 4 - 1
    out = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc)
    rows = sampled(M)
    check(out[rows], *lora_ref(x[rows], wq, ws, a, b, ids[rows], sc))


@pytest.mark.parametrize("M", [1, 40, 300])
def test_experts_past_2_31(M):
    E, N = 1000, 2160
    k = 1024  # 2.2e9 weights
    g = torch.Generator(device="cuda").manual_seed(3)
    wq = torch.empty(E, N, k, dtype=torch.float8_e4m3fn, device="cuda")
    ws = torch.empty(E, N, device="cuda")
    wq[-2:], ws[-2:] = quantized_weight(g, 2, N, k)
    x = torch.randn(M, k, generator=g, device="cuda").to(torch.bfloat16)
    m = M // 3
    offsets = torch.tensor([0] * (E - 1) + [m, M], dtype=torch.int32, device="cuda")
    out = f.fp8_grouped_linear(x, wq, ws, offsets)
    xq, xs = torch_quant_ref(x)
    check(out[:m], *base_rows(xq[:m], xs[:m], wq[-2], ws[-2], None))
    check(out[m:], *base_rows(xq[m:], xs[m:], wq[-1], ws[-1], None))


@pytest.mark.parametrize("M", [1, 40, 300])
def test_adapters_past_2_31(M):
    L, N, R = 2100, 8192, 128  # lora_b: 2.2e9 elements
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wq, ws = quantized_weight(g, N, K)
    a = torch.empty(L, R, K, dtype=torch.bfloat16, device="cuda")
    b = torch.empty(L, N, R, dtype=torch.bfloat16, device="cuda")
    a[-2:] = torch.randn(2, R, K, generator=g, device="cuda").bfloat16()
    b[-2:] = (torch.randn(2, N, R, generator=g, device="cuda") * 0.1).bfloat16()
    sc = torch.ones(L, device="cuda")
    local = (torch.arange(M, device="cuda") % 2).int() if M < 300 else \
        (torch.arange(M, device="cuda") >= 150).int()
    out = f.fp8_linear_lora(x, wq, ws, a, b, local + (L - 2), sc)
    check(out, *lora_ref(x, wq, ws, a[-2:], b[-2:], local, sc[-2:]))
