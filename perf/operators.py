"""Performance cases of the linears whose weights depend on the row.

Two operators, both built on the per-token x per-channel e4m3 linear:

* ``grouped``: rows sorted by expert, each expert with weights of its own
  (``fp8_grouped_linear``, and ``fp8_grouped_gemm`` on rows that are quantized already);
* ``lora``: one shared projection plus a low-rank adapter chosen per row
  (``fp8_linear_lora``).

``run`` has each in its plain form (elementary torch operations in 32 bits, rounded once)
and, with ``own`` set, as the package's call on the same tensors. The e4m3 rounding of the
activations belongs to both operators' definition: scale = max(amax / 448, 1e-12) per row,
code = e4m3(clamp(x * (1 / scale), -448, 448)), each step in fp32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # one token of a top-2 mixture of experts: nothing but launch and weight latency
        dict(name="experts, one token", op="grouped", E=16, M=2, K=2048, N=1024, dtype="bf16",
             bias=False, skew=0.0, codes=False),
        # a decode batch of 32 tokens, top-6 of 64 experts: nearly all weights, a few rows each
        dict(name="experts, decode batch", op="grouped", E=64, M=192, K=2048, N=2816,
             dtype="bf16", bias=False, skew=0.5, codes=False),
        # the second product of an expert whose rows an activation kernel has quantized;
        # K and N swapped, twice the rows
        dict(name="experts, quantized rows", op="grouped", E=64, M=384, K=1408, N=2048,
             dtype="bf16", bias=False, skew=0.5, codes=True),
        # ragged everything: K past a multiple of 128, an odd N, biases, empty experts, fp16
        dict(name="experts, odd sizes", op="grouped", E=12, M=1111, K=1552, N=1001,
             dtype="fp16", bias=True, skew=1.5, codes=False),
        # a chunk of prefill over many small experts
        dict(name="experts, short prefill", op="grouped", E=64, M=4096, K=2048, N=1408,
             dtype="bf16", bias=False, skew=0.7, codes=False),
        # prefill through the first product of few large experts
        dict(name="experts, prefill", op="grouped", E=8, M=8192, K=4096, N=14336, dtype="bf16",
             bias=False, skew=0.3, codes=False),
        # one token of one request
        dict(name="adapters, one token", op="lora", M=1, K=4096, N=4096, L=8, R=16,
             dtype="bf16", bias=False, rows="each"),
        # 64 requests decode one token each, with adapters of their own or none
        dict(name="adapters, decode batch", op="lora", M=64, K=4096, N=6144, L=32, R=32,
             dtype="bf16", bias=True, rows="each"),
        # a continuous batch: some prompts and many single tokens
        dict(name="adapters, prompts and decodes", op="lora", M=2000, K=4096, N=4096, L=32,
             R=64, dtype="bf16", bias=False, rows="mixed"),
        # ragged everything, fp16
        dict(name="adapters, odd sizes", op="lora", M=777, K=1552, N=1001, L=5, R=8,
             dtype="fp16", bias=True, rows="requests"),
        # images of 4608 tokens in one batch, an adapter for each
        dict(name="adapters, images", op="lora", M=9216, K=2560, N=7680, L=4, R=32,
             dtype="bf16", bias=True, rows="images"),
        # prefill of long prompts, wide adapters
        dict(name="adapters, prefill", op="lora", M=16384, K=4096, N=4096, L=16, R=128,
             dtype="bf16", bias=False, rows="requests"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    K = 16 * rng.randint(16, 400)
    N = rng.randint(200, 7000)
    if rng.random() < 0.5:
        N -= N % 64
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    bias = rng.random() < 0.5
    if rng.random() < 0.5:
        E = _log(rng, 2, 128)
        N = min(N, 400_000_000 // (E * K))  # the weights of all experts together
        return dict(op="grouped", E=E, M=_log(rng, 1, 8192), K=K, N=N, dtype=dtype, bias=bias,
                    skew=round(rng.uniform(0.0, 1.5), 2), codes=rng.random() < 0.3)
    M = _log(rng, 1, 12000)
    return dict(op="lora", M=M, K=K, N=N, L=rng.randint(1, 32), R=8 * rng.randint(1, 16),
                dtype=dtype, bias=bias,
                rows="each" if M <= 128 and rng.random() < 0.6 else
                rng.choice(["requests", "mixed"]))


# ---------------------------------------------------------------------------- inputs

def _expert_rows(c, rng: random.Random):
    """Rows of each expert: popularity ~ rank^-skew in random order; the largest cases leave
    some experts empty by themselves, skew > 1 nearly always does."""
    w = [(i + 1.0) ** -c["skew"] for i in range(c["E"])]
    rng.shuffle(w)
    n = [0] * c["E"]
    for e in rng.choices(range(c["E"]), weights=w, k=c["M"]):
        n[e] += 1
    return n


def _adapter_rows(c, rng: random.Random):
    """Adapter of each row (-1: none)."""
    M, L = c["M"], c["L"]
    if c["rows"] == "each":
        return [rng.randrange(L) if M == 1 or rng.random() < 0.9 else -1 for _ in range(M)]
    if c["rows"] == "images":
        return [i * L // M for i in range(M)]
    out = []
    decodes = M // 20 if c["rows"] == "mixed" else 0
    while len(out) < M - decodes:
        n = min(M - decodes - len(out), max(1, int(rng.lognormvariate(math.log(max(2, M // 10)), 0.7))))
        out += [rng.randrange(L) if rng.random() < 0.9 else -1] * n
    return out + [rng.randrange(L) for _ in range(decodes)]


def _codes(t):
    """Rows of a matrix in e4m3 with one fp32 scale each, by the definition above."""
    f = t.float()
    amax = f.abs().amax(dim=-1)
    scale = torch.clamp_min(amax / torch.full_like(amax, 448.0), 1e-12)
    inv = torch.ones_like(scale) / scale
    return (f * inv[..., None]).clamp(-448.0, 448.0).to(E4M3), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dt = TYPES[case["dtype"]]
    M, K, N = case["M"], case["K"], case["N"]
    # activations as the quantizer meets them: a few channels far above the others
    x = torch.randn(M, K, generator=g, device="cuda")
    x *= torch.where(torch.rand(K, generator=g, device="cuda") < 0.005, 50.0, 1.0)
    x = x.to(dt)
    s = dict(op=case["op"], x=x)
    if case["op"] == "grouped":
        E = case["E"]
        wq = torch.empty(E, N, K, dtype=E4M3, device="cuda")
        ws = torch.empty(E, N, dtype=torch.float32, device="cuda")
        for e in range(E):
            wq[e], ws[e] = _codes(torch.randn(N, K, generator=g, device="cuda") * 0.02)
        ends = torch.tensor([0] + _expert_rows(case, rng)).cumsum(0)
        s.update(wq=wq, ws=ws, offsets=ends.to(torch.int32).cuda(), counts=ends.tolist(),
                 bias=(torch.randn(E, N, generator=g, device="cuda") * 0.02).to(dt)
                 if case["bias"] else None)
        if case["codes"]:
            s["xq"], s["xs"] = _codes(x)
        return s
    L, R = case["L"], case["R"]
    s["wq"], s["ws"] = _codes(torch.randn(N, K, generator=g, device="cuda") * 0.02)
    s["a"] = (torch.randn(L, R, K, generator=g, device="cuda") / math.sqrt(K)).to(dt)
    s["b"] = (torch.randn(L, N, R, generator=g, device="cuda") * 0.05).to(dt)
    s["scaling"] = torch.rand(L, generator=g, device="cuda") + 0.5
    ids = _adapter_rows(case, rng)
    s["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
    s["rows_of"] = [(a, torch.tensor([i for i, v in enumerate(ids) if v == a], device="cuda"))
                    for a in sorted(set(ids)) if a >= 0]
    s["bias"] = (torch.randn(N, generator=g, device="cuda") * 0.02).to(dt) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------- the operators

def run(s):
    if own:
        import fp8linear_b200 as f

        if s["op"] == "lora":
            return f.fp8_linear_lora(s["x"], s["wq"], s["ws"], s["a"], s["b"], s["ids"],
                                     s["scaling"], s["bias"])
        if "xq" in s:
            return f.fp8_grouped_gemm(s["xq"], s["xs"], s["wq"], s["ws"], s["offsets"], s["bias"])
        return f.fp8_grouped_linear(s["x"], s["wq"], s["ws"], s["offsets"], s["bias"])
    x, wq, ws = s["x"], s["wq"], s["ws"]
    xq, xs = (s["xq"], s["xs"]) if "xq" in s else _codes(x)
    if s["op"] == "grouped":
        out = torch.zeros(x.shape[0], wq.shape[1], dtype=torch.bfloat16 if "xq" in s else x.dtype,
                          device=x.device)
        for e, (i, j) in enumerate(zip(s["counts"], s["counts"][1:])):
            if i < j:
                y = (xq[i:j].float() @ wq[e].float().T) * xs[i:j, None] * ws[e]
                out[i:j] = y if s["bias"] is None else y + s["bias"][e].float()
        return out
    y = (xq.float() @ wq.float().T) * xs[:, None] * ws
    if s["bias"] is not None:
        y = y + s["bias"].float()
    for a, rows in s["rows_of"]:
        h = (x[rows].float() @ s["a"][a].float().T) * s["scaling"][a]
        y[rows] += h @ s["b"][a].float().T
    return y.to(x.dtype)


def work(case):
    """Each input read once and each output written once; of the experts' and adapters'
    weights those that some row uses (their expected number)."""
    M, K, N = case["M"], case["K"], case["N"]
    if case["op"] == "grouped":
        w = [(i + 1.0) ** -case["skew"] for i in range(case["E"])]
        used = sum(1.0 - (1.0 - v / sum(w)) ** M for v in w)
        x = M * (K + 4) if case["codes"] else 2 * M * K
        b = x + 2 * M * N + used * N * (K + 4 + (2 if case["bias"] else 0)) + 4 * (case["E"] + 1)
        return {"bytes": int(b), "flops": 2 * M * N * K}
    L, R = case["L"], case["R"]
    runs = {"each": M, "images": L, "requests": 10, "mixed": 10 + M // 20}[case["rows"]]
    used = L if case["rows"] == "images" else L * (1.0 - (1.0 - 1.0 / L) ** min(runs, M))
    b = 2 * M * (K + N) + N * (K + 4) + used * 2 * R * (K + N) + 4 * M
    return {"bytes": int(b), "flops": 2 * M * N * K + 2 * M * R * (K + N)}


# ---------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions in fp64, row by row of the expert or adapter; the activations' codes
    are part of the definition and take its fp32 steps."""
    s = prepare(case, seed)
    x = s["x"]
    M, N = case["M"], case["N"]
    f = x.to(torch.float32)
    top = torch.maximum(f.max(dim=1, keepdim=True).values, -f.min(dim=1, keepdim=True).values)
    scale = torch.maximum(torch.div(top, torch.tensor(448.0, device=x.device).expand_as(top)),
                          torch.tensor(1e-12, device=x.device))
    step = torch.reciprocal(scale.double()).float()  # 1 / scale, rounded to fp32 once
    deq = torch.clamp(f * step, -448.0, 448.0).to(E4M3).double() * scale.double()
    out = torch.zeros(M, N, dtype=torch.float64, device=x.device)
    if case["op"] == "grouped":
        for e in range(case["E"]):
            i, j = int(s["offsets"][e]), int(s["offsets"][e + 1])
            if i == j:
                continue
            w = s["wq"][e].double() * s["ws"][e].double()[:, None]
            torch.matmul(deq[i:j], w.t(), out=out[i:j])
            if s["bias"] is not None:
                out[i:j] += s["bias"][e].double()
        return out
    torch.matmul(deq, (s["wq"].double() * s["ws"].double()[:, None]).t(), out=out)
    if s["bias"] is not None:
        out += s["bias"].double()
    ids = s["ids"].long()
    for a in range(case["L"]):
        mine = (ids == a).nonzero().flatten()
        if mine.numel():
            # (scaling * A) first, then B: another order than the plain form's
            down = s["a"][a].double() * s["scaling"][a].double()
            out[mine] += torch.einsum("mk,rk,nr->mn", x[mine].double(), down, s["b"][a].double())
    return out
