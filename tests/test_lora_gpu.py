"""fp8_linear_lora against a plain fp64 form on the GPU, and a served block of both operators."""
from __future__ import annotations

import pytest
import torch

import fp8linear_b200 as f
from tests.helpers import require_sm100
from tests.rowsel_helpers import check, grouped_ref, lora_ref, quantized_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    require_sm100()


@pytest.fixture(autouse=True)
def _no_timeouts(capi):
    yield
    assert capi.device_status(clear=True) == 0


def make(seed, M, K, N, L, R, dtype=torch.bfloat16, bias=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, ::97] *= 50
    wq, ws = quantized_weight(g, N, K)
    a = (torch.randn(L, R, K, generator=g, device="cuda") / K**0.5).to(dtype)
    b = (torch.randn(L, N, R, generator=g, device="cuda") * 0.1).to(dtype)
    sc = torch.rand(L, generator=g, device="cuda") + 0.5
    bb = None if bias is None else torch.randn(N, generator=g, device="cuda").to(bias)
    return x.to(dtype), wq, ws, a, b, sc, bb


def runs(*pairs):
    """(adapter, rows) pairs as the int32 ids on the GPU."""
    return torch.tensor([a for a, n in pairs for _ in range(n)], dtype=torch.int32, device="cuda")


CASES = [
    # M x K x N, L, R, runs of (adapter, rows)
    (16, 16, 1, 8, [(0, 1)]),
    (256, 128, 3, 16, [(2, 1)]),
    (512, 300, 4, 8, [(0, 1), (-1, 1), (3, 1), (1, 5)]),
    (1040, 257, 2, 24, [(1, 17)]),
    (4096, 1000, 8, 64, [(i % 8, 1) for i in range(64)]),
    (272, 2048, 5, 128, [(4, 100), (-1, 3), (0, 25)]),
    (128, 64, 1, 40, [(-1, 30)]),
    (1040, 384, 33, 32, [(i % 33, 1) for i in range(63)]),
    (1040, 384, 33, 32, [(i % 33, 1) for i in range(65)]),
    # more than 64 rows: tiles from the plan
    (16, 1, 1, 8, [(0, 129)]),
    (256, 320, 2, 16, [(0, 160), (1, 160)]),
    (1040, 257, 3, 8, [(0, 200), (-1, 31), (2, 1), (1, 400), (-1, 170)]),
    (528, 600, 4, 72, [(3, 320), (1, 65), (0, 255), (2, 7)]),
    (2048, 512, 7, 128, [(6, 500), (2, 12), (-1, 700), (3, 333)]),
    (640, 1001, 40, 32, [(0, 700)] + [(i, 1) for i in range(40)]),
    (320, 264, 140, 48, [(i, 1) for i in range(140)]),     # 128 adapters in one tile of rows
    (64, 96, 2, 56, [(-1, 300), (1, 2), (-1, 300)]),
    (400, 160, 3, 104, [(0, 320), (1, 320), (2, 320), (-1, 320)]),
]


@pytest.mark.parametrize("K,N,L,R,pairs", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora(K, N, L, R, pairs, dtype):
    ids = runs(*pairs)
    x, wq, ws, a, b, sc, bias = make(K + N + R, ids.numel(), K, N, L, R, dtype, bias=dtype)
    out = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias)
    assert out.dtype == dtype
    check(out, *lora_ref(x, wq, ws, a, b, ids, sc, bias))


@pytest.mark.parametrize("M,K,R", [(1, 16, 128), (1, 4112, 128), (2, 2064, 64), (7, 144, 16),
                                   (8, 1040, 16), (8, 1040, 24), (9, 1040, 8), (1, 272, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_tokens(M, K, R, dtype):
    """Both sides of the border below which the GEMM computes x . A^T itself."""
    x, wq, ws, a, b, sc, bias = make(M + K + R, M, K, 392, 5, R, dtype, bias=torch.float32)
    ids = (torch.arange(M, device="cuda", dtype=torch.int32) * 2) % 6 - 1
    ids[0] = 4
    check(f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias),
          *lora_ref(x, wq, ws, a, b, ids, sc, bias))


@pytest.mark.parametrize("M", [5, 128, 129, 1000])
def test_rows_in_any_order(M):
    g = torch.Generator(device="cuda").manual_seed(M)
    x, wq, ws, a, b, sc, bias = make(M, M, 336, 200, 6, 16, bias=torch.float32)
    ids = torch.randint(-1, 6, (M,), generator=g, device="cuda", dtype=torch.int32)
    check(f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias),
          *lora_ref(x, wq, ws, a, b, ids, sc, bias))


@pytest.mark.parametrize("M", [65, 511, 512, 513, 1025, 5000])
@pytest.mark.parametrize("longest", [2, 40, 700])
def test_runs_of_any_lengths(M, longest):
    """Long runs, short ones and none in turn, across every border of the token plan."""
    g = torch.Generator().manual_seed(M + longest)
    ids = []
    while len(ids) < M:
        n = int(torch.randint(1, longest + 1, (1,), generator=g))
        if torch.rand(1, generator=g) < 0.3:
            n = min(n, 3)
        ids += [int(torch.randint(-1, 5, (1,), generator=g))] * n
    ids = torch.tensor(ids[:M], dtype=torch.int32, device="cuda")
    x, wq, ws, a, b, sc, bias = make(M, M, 48, 72, 5, 8, bias=torch.float32)
    check(f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias),
          *lora_ref(x, wq, ws, a, b, ids, sc, bias))


@pytest.mark.parametrize("M", [7, 300])
def test_ids_outside_the_adapters_mean_none(M):
    x, wq, ws, a, b, sc, bias = make(M, M, 96, 136, 2, 8)
    ref = f.fp8_linear_lora(x, wq, ws, a, b, runs((-1, M)), sc, None)
    ids = torch.tensor([-1, 2, 2**31 - 1, -2**31, 77] * M, dtype=torch.int32, device="cuda")[:M]
    assert torch.equal(f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, None), ref)
    check(ref, *lora_ref(x, wq, ws, a, b, runs((-1, M)), sc))
    assert torch.equal(f.fp8_linear_lora(x, wq, ws, a[:0], b[:0], ids, sc[:0], None),
                       f.fp8_linear(x, wq, ws, None))


@pytest.mark.parametrize("M", [3, 128, 160, 700])
def test_one_request_does_not_reach_anothers_rows(M):
    """Infinities and NaN in an adapter or a row stay with that adapter's rows or that row."""
    x, wq, ws, a, b, sc, bias = make(M, M, 160, 264, 3, 16, bias=torch.bfloat16)
    ids = torch.arange(M, device="cuda", dtype=torch.int32) * 3 // M
    good = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias)
    check(good, *lora_ref(x, wq, ws, a, b, ids, sc, bias))
    for where in ("a", "b", "scaling"):
        a2, b2, s2 = a.clone(), b.clone(), sc.clone()
        if where == "a":
            a2[1] = float("nan")
        elif where == "b":
            b2[1, :, 3] = float("inf")
        else:
            s2[1] = float("nan")
        got = f.fp8_linear_lora(x, wq, ws, a2, b2, ids, s2, bias)
        hit = ids == 1
        assert not torch.isfinite(got[hit]).any()
        assert torch.equal(got[~hit], good[~hit])
    x2 = x.clone()
    x2[0, 5] = float("nan")  # ignored by the quantizer's maximum, not by the adapter
    got = f.fp8_linear_lora(x2, wq, ws, a, b, ids, sc, bias)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], good[1:])


@pytest.mark.parametrize("M", [4, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_intermediate_beyond_fp16(M, dtype):
    """h above fp16's largest value and far below its smallest: it is kept to fp32's accuracy."""
    x, wq, ws, a, b, sc, _ = make(M, M, 512, 64, 2, 16, dtype)
    ids = torch.arange(M, device="cuda", dtype=torch.int32) % 2
    big = (x * 100).to(dtype), (a * 600).to(dtype), (b * 1e-4).to(dtype)
    check(f.fp8_linear_lora(big[0], wq, ws, big[1], big[2], ids, sc, None),
          *lora_ref(big[0], wq, ws, big[1], big[2], ids, sc))
    small = x, (a * 2.0**-10).to(dtype), b, sc * 2.0**-20
    wz = torch.zeros_like(wq.view(torch.uint8)).view(wq.dtype)  # the adapters alone
    if dtype == torch.bfloat16:
        check(f.fp8_linear_lora(small[0], wz, ws, small[1], small[2], ids, small[3], None),
              *lora_ref(small[0], wz, ws, small[1], small[2], ids, small[3]))
    # one huge and many small values of h in a row
    wide = a.clone()
    wide[:, 0] *= 1000
    bw = b.clone()
    bw[:, :, 0] *= 1e-3
    check(f.fp8_linear_lora(x, wz, ws, wide, bw, ids, sc, None),
          *lora_ref(x, wz, ws, wide, bw, ids, sc))


def test_shapes_strides_and_alignment():
    x, wq, ws, a, b, sc, bias = make(3, 6 * 35, 128, 80, 3, 16, bias=torch.bfloat16)
    ids = (torch.arange(210, device="cuda", dtype=torch.int32) // 35) % 4 - 1
    ref = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias)
    out = f.fp8_linear_lora(x.view(2, 3, 35, 128), wq, ws, a, b, ids.view(2, 3, 35), sc, bias)
    assert out.shape == (2, 3, 35, 80) and torch.equal(out.view(210, 80), ref)
    wide = torch.zeros(210, 200, dtype=x.dtype, device="cuda")
    wide[:, 3:131] = x
    at = a.transpose(1, 2).contiguous().transpose(1, 2)
    bt = b.transpose(0, 1).contiguous().transpose(0, 1)
    i2 = torch.stack([ids, ids], 1)[:, 1]
    assert torch.equal(f.fp8_linear_lora(wide[:, 3:131], wq, ws, at, bt, i2, sc, bias), ref)
    one = f.fp8_linear_lora(x[0], wq, ws, a, b, ids[:1], sc, bias)
    assert one.shape == (80,)
    check(one[None], *lora_ref(x[:1], wq, ws, a, b, ids[:1], sc, bias))
    assert f.fp8_linear_lora(x[:0], wq, ws, a, b, ids[:0], sc, bias).shape == (0, 80)


@pytest.mark.parametrize("M", [1, 64, 500])
def test_repeatable_and_written_just_before(M):
    """Every input rewritten on the stream right before the call is seen."""
    one = make(1, M, 512, 384, 4, 32)
    two = make(2, M, 512, 384, 4, 32)
    ids = torch.arange(M, device="cuda", dtype=torch.int32) % 4
    ids2 = ids.flip(0).contiguous()
    ref = [f.fp8_linear_lora(*v[:5], i, v[5], None) for v, i in ((one, ids), (two, ids2))]
    torch.cuda.synchronize()
    buf = [t.clone() for t in one[:6]]
    ib = ids.clone()
    for _ in range(3):
        got = []
        for v, i in ((one, ids), (two, ids2)):
            for d, s in zip(buf, v[:6]):
                d.copy_(s)
            ib.copy_(i)
            got.append(f.fp8_linear_lora(*buf[:5], ib, buf[5], None))
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("M", [16, 300])
def test_captured_graphs(M):
    """Two captured graphs replayed in turn with new ids."""
    x, wq, ws, a, b, sc, bias = make(M, M, 256, 200, 3, 16, bias=torch.float32)
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for v in (x, x.flip(0).contiguous()):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((f.fp8_linear_lora(v, wq, ws, a, b, ids, sc, bias), v))
        graphs.append(g)
    for new in (ids + 1, torch.arange(M, device="cuda", dtype=torch.int32) % 4 - 1, ids - 1):
        ids.copy_(new.to(torch.int32))
        for g in graphs:
            g.replay()
        for o, v in outs:
            check(o, *lora_ref(v, wq, ws, a, b, ids, sc, bias))


def test_two_streams_at_once():
    sets = []
    for seed, M in ((1, 40), (2, 900)):
        x, wq, ws, a, b, sc, _ = make(seed, M, 512, 640, 3, 16)
        ids = torch.arange(M, device="cuda", dtype=torch.int32) * 3 // M
        sets.append((x, wq, ws, a, b, ids, sc, None))
    ref = [f.fp8_linear_lora(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(4):
        for st, s, r in zip(streams, sets, ref):
            with torch.cuda.stream(st):
                got.append((f.fp8_linear_lora(*s), r))
    torch.cuda.synchronize()
    for o, r in got:
        assert torch.equal(o, r)


def test_capi_matches_op(capi):
    for M in (9, 333):
        x, wq, ws, a, b, sc, bias = make(M, M, 176, 90, 3, 24, torch.float16, bias=torch.float32)
        ids = torch.arange(M, device="cuda", dtype=torch.int32) % 4
        assert torch.equal(capi.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias),
                           f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, bias))


def test_bad_calls_are_refused_on_the_gpu():
    x, wq, ws, a, b, sc, bias = make(5, 6, 64, 32, 2, 16, bias=torch.bfloat16)
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    for args in [
        (x.float(), wq, ws, a, b, ids, sc, bias), (x[:, :48], wq, ws, a, b, ids, sc, bias),
        (x, wq, ws[:3], a, b, ids, sc, bias), (x, wq, ws, a.half(), b, ids, sc, bias),
        (x, wq, ws, a, b[:, :, :8], ids, sc, bias), (x, wq, ws, a, b, ids.long(), sc, bias),
        (x, wq, ws, a, b, ids[:5], sc, bias), (x, wq, ws, a, b, ids, sc[:1], bias),
        (x, wq, ws, a, b, ids, sc.half(), bias), (x, wq, ws, a.cpu(), b, ids, sc, bias),
        (x, wq, ws, a, b, ids.cpu(), sc, bias), (x, wq, ws, a, b, ids, sc, bias.cpu()),
        (x, wq, ws, a[:, :12], b[:, :, :12], ids, sc, bias),
        (x, wq, ws, a[:, :0], b[:, :, :0], ids, sc, bias),
        (x, wq, ws, a.repeat(1, 9, 1), b.repeat(1, 1, 9), ids, sc, bias),
    ]:
        with pytest.raises(RuntimeError, match="fp8_linear_lora"):
            f.fp8_linear_lora(*args)


@pytest.mark.parametrize("tokens", [4, 700])
def test_served_block(tokens):
    """Both operators as a model runs them: a projection with adapters, then a top-2 mixture
    of experts, everything captured in one graph, against fp64 step by step."""
    K, N, E, H = 256, 512, 6, 384
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, wq, ws, a, b, sc, _ = make(tokens, tokens, K, N, 3, 16)
    ids = torch.arange(tokens, device="cuda", dtype=torch.int32) % 4 - 1
    w1 = torch.randn(E, H, N, generator=g, device="cuda").bfloat16() * 0.05
    w2 = torch.randn(E, K, H, generator=g, device="cuda").bfloat16() * 0.05
    q1, s1 = f.quantize_expert_weights(w1)
    q2, s2 = f.quantize_expert_weights(w2)
    gate = torch.randn(N, E, generator=g, device="cuda")

    def block():
        y = f.fp8_linear_lora(x, wq, ws, a, b, ids, sc, None)
        p, e = (y.float() @ gate).softmax(-1).topk(2)
        e = e.flatten()
        order = e.argsort(stable=True)
        offsets = torch.searchsorted(e[order], torch.arange(E + 1, device="cuda")).to(torch.int32)
        rows = order // 2
        h = torch.relu(f.fp8_grouped_linear(y[rows], q1, s1, offsets))
        z = f.fp8_grouped_linear(h, q2, s2, offsets)
        out = torch.zeros(tokens, K, device="cuda").index_add_(
            0, rows, z.float() * p.flatten()[order][:, None])
        return y, offsets, rows, h, z, out

    block()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        block()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, offsets, rows, h, z, out = block()
    for _ in range(2):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        check(y, *lora_ref(x, wq, ws, a, b, ids, sc))
        o = offsets.tolist()
        assert o[0] == 0 and o[-1] == 2 * tokens
        xq, xs = f.quantize_fp8(y[rows])
        r, e = grouped_ref(xq, xs, q1, s1, o)
        check(h, r.clamp_min(0), e)  # relu does not enlarge a difference
        xq, xs = f.quantize_fp8(h)
        check(z, *grouped_ref(xq, xs, q2, s2, o))
        assert torch.isfinite(out).all()
