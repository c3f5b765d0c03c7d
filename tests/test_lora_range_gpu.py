"""fp8_linear_lora's intermediate h = scaling * x . A^T at the ends of its range, on the adapters
alone (the projection's codes are zero).

The bound of an element, besides the sums' own terms (tests/rowsel_helpers.py): h goes to the
second product as a high part in the type and a low part of 2^7 times the rest.

* bf16 (8 bits): |h| < 2^(e+1) leaves a rest below 2^(e-7), rounded to half a step, at most
  2^(e-16): 2^-16 of h.
* fp16 (11 bits): the row is scaled by a power of two to a largest value of at least 2^14. The
  rest is below 2^(e-10) and its half step at most 2^(e-22): 2^-22 of h. Where 2^7 times the rest
  is subnormal, it is off by less than a step, 2^-24 / 2^7 = 2^-31: 2^-45 of the row's largest value.
"""
from __future__ import annotations

import pytest
import torch

import fp8linear_b200 as f
from tests.helpers import require_sm100
from tests.rowsel_helpers import check

pytestmark = pytest.mark.gpu

N = 136


@pytest.fixture(scope="module", autouse=True)
def _dev():
    require_sm100()


@pytest.fixture(autouse=True)
def _no_timeouts(capi):
    yield
    assert capi.device_status(clear=True) == 0


def adapters_alone(x, a, b, ids, scaling):
    K = x.shape[1]
    wq = torch.zeros(N, K, device="cuda").to(torch.float8_e4m3fn)
    return f.fp8_linear_lora(x, wq, torch.ones(N, device="cuda"), a, b, ids, scaling, None)


def ref(x, a, b, ids, scaling):
    """(value, bound) in fp64."""
    M, K = x.shape
    R = a.shape[1]
    out = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().flatten()
        A, B, s = a[i].double(), b[i].double(), scaling[i].double()
        h = (x[rows].double() @ A.T) * s
        mag = (x[rows].double().abs() @ A.abs().T) * s.abs()
        herr = mag * ((K / 16 + 24) * 2.0**-23 + 2.0**-24)
        if x.dtype == torch.float16:
            top = h.abs().where(h.isfinite(), 0.0).amax(1, keepdim=True)
            herr += h.abs() * 2.0**-22 + top * 2.0**-45
        else:
            herr += h.abs() * 2.0**-16
        out[rows] = h @ B.T
        err[rows] = herr @ B.abs().T + (h.abs() @ B.abs().T) * (R + 24) * 2.0**-23
    return out, err


# few tokens (x . A^T in the GEMM's own CTAs), the warps' MMAs, tiles of one adapter, of several
ROWS = [(3, "any"), (40, "any"), (200, "runs"), (200, "any")]


def make_ids(M, rows, L=3):
    i = torch.arange(M, device="cuda", dtype=torch.int32)
    return i * L // M if rows == "runs" else i % (L + 1) - 1


@pytest.mark.parametrize("M,rows", ROWS)
@pytest.mark.parametrize("R", [16, 40, 72, 128])
@pytest.mark.parametrize("up,down", [(10, -10), (14, -13)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ranks_far_apart(M, rows, R, up, down, dtype):
    """One rank's h is 2^20 or 2^27 times the others', and B leaves it out of half the columns,
    whose sums are the small ranks' alone."""
    g = torch.Generator(device="cuda").manual_seed(M + R)
    K = 96
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    a = torch.randn(3, R, K, generator=g, device="cuda") / 10
    a[:, 1:] *= 2.0**down
    a[:, 0] *= 2.0**up
    b = torch.randn(3, N, R, generator=g, device="cuda") * 100
    b[:, :, 0] *= 2.0**-15
    b[:, ::2, 0] = 0
    sc = torch.rand(3, generator=g, device="cuda") + 0.5
    args = x, a.to(dtype), b.to(dtype), make_ids(M, rows), sc
    check(adapters_alone(*args), *ref(*args))


@pytest.mark.parametrize("M,rows", [(3, "any"), (200, "runs"), (200, "any")])
@pytest.mark.parametrize("R", [16, 72])
@pytest.mark.parametrize("h", [-20, -30, -140])
def test_fp16_rows_far_below_one(M, rows, R, h):
    """Rows whose largest h is about 2^h: 2^-140 is below fp32's normal numbers too, and every
    fifth row of x is zero."""
    g = torch.Generator(device="cuda").manual_seed(M + R)
    K = 96
    x = torch.randn(M, K, generator=g, device="cuda").half()
    x[::5] = 0
    a = (torch.randn(3, R, K, generator=g, device="cuda") * 2.0**-10 / K**0.5).half()
    b = (torch.randn(3, N, R, generator=g, device="cuda") * 2.0**12).half()
    sc = torch.full((3,), 2.0 ** (h + 10), device="cuda")
    args = x, a, b, make_ids(M, rows), sc
    out = adapters_alone(*args)
    check(out, *ref(*args))
    assert torch.count_nonzero(out[::5]) == 0


@pytest.mark.parametrize("M,rows", ROWS)
def test_bf16_largest_values(M, rows):
    """h between bf16's largest value and fp32's."""
    x = torch.ones(M, 16, device="cuda").bfloat16()
    a = torch.ones(3, 8, 16, device="cuda").bfloat16()
    a[:, 1:] = 0
    b = torch.full((3, N, 8), 2.0**-120, device="cuda").bfloat16()
    sc = torch.full((3,), 3.4e38 / 16, device="cuda")
    args = x, a, b, make_ids(M, rows), sc
    check(adapters_alone(*args), *ref(*args))


def check_with_infinities(got, value, err):
    for of in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(of(got), of(value)), of.__name__
    ok = value.isfinite()
    check(got.where(ok, 0.0), value.where(ok, 0.0), err.where(ok, 0.0))


def with_infinities_in_b(M, rows, K, R, exact, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + R + K)

    def values(*shape):
        v = torch.randn(*shape, generator=g, device="cuda")
        return (v * (0.3 if K > 96 else 0.7)).round() if exact else v / 2

    x, a = values(M, K), values(3, R, K)
    b = torch.randn(3, N, R, generator=g, device="cuda")
    b[:, 1:60:3, 3] = float("inf")
    b[:, 60:100:3, R - 1] = -float("inf")
    b[:, 100:130, 3] = float("inf")
    b[:, 100:130:2, 5] = float("inf")
    return x.to(dtype), a.to(dtype), b.to(dtype), make_ids(M, rows), torch.ones(3, device="cuda")


@pytest.mark.parametrize("M,rows,K", [(*r, 96) for r in ROWS] + [(*r, 4096) for r in ROWS[1:]])
@pytest.mark.parametrize("R", [8, 40, 128])
@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_b(M, rows, K, R, exact, dtype):
    """The formula's infinities, by sign, and its NaN (an infinity times a zero h, two of
    opposite signs), whether h has a rest beside its high part or not (exact: whole numbers
    below 128, zeros among them)."""
    args = with_infinities_in_b(M, rows, K, R, exact, dtype)
    check_with_infinities(adapters_alone(*args), *ref(*args))


@pytest.mark.parametrize("M,rows", ROWS)
@pytest.mark.parametrize("R", [8, 72])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_h(M, rows, R, dtype):
    """An infinity in A: infinite h, against finite, zero and infinite values of B."""
    g = torch.Generator(device="cuda").manual_seed(M + R)
    K = 96
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    a = (torch.randn(3, R, K, generator=g, device="cuda") / 4).to(dtype)
    b = torch.randn(3, N, R, generator=g, device="cuda").to(dtype)
    a[1, 2, 7] = float("inf")
    x[:, 7] = torch.where(torch.arange(M, device="cuda") % 2 == 0, 1.0, -2.0).to(dtype)
    b[1, ::4, 2] = 0
    b[1, 1::4, 2] = float("inf")
    args = x, a, b, make_ids(M, rows), torch.ones(3, device="cuda")
    check_with_infinities(adapters_alone(*args), *ref(*args))


@pytest.mark.parametrize("M", [1, 2, 3, 8])
@pytest.mark.parametrize("K", [528, 4096])
@pytest.mark.parametrize("R", [8, 16, 40])
@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_b_of_few_tokens(M, K, R, exact, dtype):
    """The same where the CTAs of a tile have parts of K each, whose sums may differ in sign."""
    args = with_infinities_in_b(M, "runs" if M == 1 else "any", K, R, exact, dtype)
    check_with_infinities(adapters_alone(*args), *ref(*args))
