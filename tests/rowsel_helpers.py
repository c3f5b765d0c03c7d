"""Plain fp64 forms of the linears whose weights depend on the row, with error bounds.

Bounds, per output element (u = half a step of the output type, torch.finfo(t).eps / 2):

* the one rounding of the result: u * |ref|, and its error terms once more through it;
* the fp32 accumulation of the e4m3 products: a 32-element tensor-core step may lose
  2^-23 of the largest magnitude seen per term and per addition onto the accumulator, so at
  most (K / 32 + 32) * 2^-23 of the sum of the terms' magnitudes (split-K adds at most 8
  more additions); the three multiplications and additions of the epilogue 4 * 2^-24;
* adapters: h = x . A^T the same way with steps of 16 (fp32 FMAs on CUDA cores, for few
  rows, run at most K / 2048 + 16 deep: smaller), scaling 2^-24, its two 16-bit parts 2^-16,
  and the sum over the rank (R + 16) * 2^-23, each of the magnitudes' sum.
"""
from __future__ import annotations

import torch

from tests.helpers import torch_quant_ref


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def base_rows(xq, xs, wq, ws, bias):
    """(value, bound of the fp32 accumulation) of rows against one weight, in fp64."""
    K = xq.shape[1]
    d = xq.double() * xs.double()[:, None]
    w = wq.double() * ws.double()[:, None]
    ref = d @ w.T
    mag = d.abs() @ w.abs().T
    if bias is not None:
        ref = ref + bias.double()
        mag = mag + bias.double().abs()
    return ref, mag * ((K / 32 + 32 + 8) * 2.0**-23 + 4 * 2.0**-24)


def grouped_ref(xq, xs, wq, ws, offsets, bias=None):
    """offsets: the list the caller meant, already clamped. Rows of no expert: zero."""
    M, N = xq.shape[0], wq.shape[1]
    ref = torch.zeros(M, N, dtype=torch.float64, device=xq.device)
    err = torch.zeros_like(ref)
    for e in range(wq.shape[0]):
        i, j = offsets[e], offsets[e + 1]
        if i < j:
            ref[i:j], err[i:j] = base_rows(xq[i:j], xs[i:j], wq[e], ws[e],
                                           None if bias is None else bias[e])
    return ref, err


def lora_ref(x, wq, ws, a, b, ids, scaling, bias=None):
    xq, xs = torch_quant_ref(x)
    K, R = x.shape[1], a.shape[1]
    ref, err = base_rows(xq, xs, wq, ws, bias)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().flatten()
        if rows.numel() == 0:
            continue
        A, B, s = a[i].double(), b[i].double(), scaling[i].double()
        h = (x[rows].double() @ A.T) * s
        hmag = (x[rows].double().abs() @ A.abs().T) * s.abs()
        herr = hmag * ((K / 16 + 16 + 8) * 2.0**-23 + 2.0**-24) + h.abs() * 2.0**-16
        ref[rows] += h @ B.T
        err[rows] += herr @ B.abs().T + (h.abs() @ B.abs().T) * (R + 16) * 2.0**-23
    return ref, err


def check(got, ref, err, dtype=None):
    """Every element of `got` within its bound of `ref`."""
    u = half_step(dtype or got.dtype)
    assert got.shape == ref.shape
    d = (got.double() - ref).abs()
    tiny = torch.finfo(got.dtype).tiny * u * 2  # half a step of the subnormals
    limit = err * (1 + u) + ref.abs() * u + tiny
    bad = ~(d <= limit)
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
        f"worst {float((d / limit).nan_to_num(posinf=1e30).max()):.3g} of the bound")


def quantized_weight(g, *shape):
    """e4m3 codes and per-channel scales of N(0, 0.02) weights, [.., N, K]."""
    w = torch.randn(*shape, generator=g, device="cuda") * 0.02
    q, s = torch_quant_ref(w.reshape(-1, shape[-1]))
    return q.reshape(shape), s.reshape(shape[:-1])
