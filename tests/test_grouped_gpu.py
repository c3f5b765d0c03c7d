"""fp8_grouped_gemm / fp8_grouped_linear against plain fp64 forms on the GPU."""
from __future__ import annotations

import pytest
import torch

import fp8linear_b200 as f
from tests.helpers import require_sm100, torch_quant_ref
from tests.rowsel_helpers import check, grouped_ref, quantized_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    require_sm100()


@pytest.fixture(autouse=True)
def _no_timeouts(capi):
    yield
    assert capi.device_status(clear=True) == 0


def make(seed, counts, K, N, dtype=torch.bfloat16, bias=None, lead=0, tail=0):
    """lead / tail: rows before the first and behind the last expert's."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    E = len(counts)
    offs = [lead]
    for c in counts:
        offs.append(offs[-1] + c)
    M = offs[-1] + tail
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, ::97] *= 50
    wq, ws = quantized_weight(g, E, N, K)
    b = None if bias is None else (torch.randn(E, N, generator=g, device="cuda")).to(bias)
    return x.to(dtype), wq, ws, torch.tensor(offs, dtype=torch.int32, device="cuda"), offs, b


CASES = [
    # counts, K, N: one row, one expert, ..
    ([1], 16, 1),
    ([1], 256, 128),
    ([0, 1, 0], 512, 300),
    ([3, 0, 5, 1], 144, 257),
    ([16, 17], 1024, 64),
    ([127, 128, 129], 272, 512),
    ([130], 4096, 1000),
    # many experts of few rows (persistent, single CTAs)
    ([1] * 40, 384, 1024),
    ([0, 1, 2, 3, 4, 5, 6, 7] * 8, 640, 1408),
    ([300] + [1] * 60, 256, 1001),
    ([0] * 30 + [2] + [0] * 33, 2048, 130),
    # larger groups (persistent, CTA pairs)
    ([257, 0, 511, 64], 1040, 1537),
    ([1000, 24, 256, 3, 0, 33], 528, 2048),
    ([2500], 2064, 777),
    ([700, 900], 128, 96),   # more rows than columns: the other tile order
]


@pytest.mark.parametrize("counts,K,N", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_linear(counts, K, N, dtype):
    x, wq, ws, off, offs, b = make(len(counts) + K, counts, K, N, dtype, bias=dtype)
    out = f.fp8_grouped_linear(x, wq, ws, off, b)
    assert out.dtype == dtype
    xq, xs = torch_quant_ref(x)
    check(out, *grouped_ref(xq, xs, wq, ws, offs, b))


@pytest.mark.parametrize("counts,K,N", CASES[2:13:3])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.float16])
def test_grouped_gemm_on_codes(counts, K, N, bias):
    x, wq, ws, off, offs, b = make(7 + K, counts, K, N, bias=bias)
    xq, xs = f.quantize_fp8(x)
    out = f.fp8_grouped_gemm(xq, xs, wq, ws, off, b)
    assert out.dtype == torch.bfloat16
    check(out, *grouped_ref(xq, xs, wq, ws, offs, b))
    assert torch.equal(out, f.fp8_grouped_linear(x, wq, ws, off, b))


@pytest.mark.parametrize("counts", [[2, 0, 3], [40] * 40, [300, 200]])
@pytest.mark.parametrize("lead,tail", [(0, 5), (7, 0), (130, 261)])
def test_rows_of_no_expert_are_zero(counts, lead, tail):
    x, wq, ws, off, offs, b = make(3, counts, 320, 200, bias=torch.bfloat16, lead=lead, tail=tail)
    out = f.fp8_grouped_linear(x, wq, ws, off, b)
    assert torch.count_nonzero(out[:lead]) == 0 and torch.count_nonzero(out[offs[-1]:]) == 0
    xq, xs = torch_quant_ref(x)
    check(out, *grouped_ref(xq, xs, wq, ws, offs, b))


@pytest.mark.parametrize("M,E", [(4, 3), (600, 2), (900, 60)])
def test_no_rows_at_all(M, E):
    x, wq, ws, _, _, b = make(5, [M] + [0] * (E - 1), 64, 72, bias=torch.bfloat16)
    for o in ([0] * (E + 1), [M] * (E + 1)):
        out = f.fp8_grouped_linear(x, wq, ws, torch.tensor(o, dtype=torch.int32, device="cuda"), b)
        assert torch.count_nonzero(out) == 0
    assert f.fp8_grouped_linear(x[:0], wq, ws, torch.zeros(E + 1, dtype=torch.int32,
                                                           device="cuda")).shape == (0, 72)


def clamped(raw, M):
    out, top = [], 0
    for o in raw:
        top = max(top, min(max(o, 0), M))
        out.append(top)
    return out


@pytest.mark.parametrize("raw", [
    [0, 10, 5, 20, 24],            # runs backwards: the group is empty, the next starts at 10
    [-3, 4, 9, 2**31 - 1, 7],      # outside [0, M]
    [24, 0, 0, 0, 0],
    [-5, -4, -3, -2, -1],
])
@pytest.mark.parametrize("rows", [24, 1200])
def test_offsets_are_clamped(raw, rows):
    """The documented reading of offsets that are not sorted or lie outside the rows."""
    x, wq, ws, _, _, _ = make(9, [rows, 0, 0, 0], 96, 160)
    scale = rows // 24
    raw = [o if abs(o) > 10**6 else o * scale for o in raw]
    off = torch.tensor(raw, dtype=torch.int32, device="cuda")
    xq, xs = torch_quant_ref(x)
    check(f.fp8_grouped_linear(x, wq, ws, off), *grouped_ref(xq, xs, wq, ws, clamped(raw, rows)))


@pytest.mark.parametrize("counts", [[3, 2, 4], [20] * 30, [300, 100, 270]])
def test_one_expert_does_not_reach_anothers_rows(counts):
    """NaN weights, scales and biases of one expert, and NaN rows, stay where they belong."""
    x, wq, ws, off, offs, b = make(11, counts, 208, 300, bias=torch.float32)
    good = f.fp8_grouped_linear(x, wq, ws, off, b)
    wq, ws, b = wq.clone(), ws.clone(), b.clone()
    wq.view(torch.uint8)[1] = 0x7F  # e4m3 NaN
    ws[1] = float("inf")
    b[1] = float("nan")
    bad = f.fp8_grouped_linear(x, wq, ws, off, b)
    i, j = offs[1], offs[2]
    assert torch.isnan(bad[i:j]).all()
    assert torch.equal(bad[:i], good[:i]) and torch.equal(bad[j:], good[j:])
    xs_ = x.clone()
    xs_[0] = float("inf")
    got = f.fp8_grouped_linear(xs_, *make(11, counts, 208, 300, bias=torch.float32)[1:4],
                               make(11, counts, 208, 300, bias=torch.float32)[5])
    assert torch.equal(got[1:], good[1:])


def test_one_expert_is_the_linear():
    """E = 1 over all rows: the sums of fp8_linear, up to their order."""
    for M in (1, 40, 700):
        x, wq, ws, off, offs, _ = make(M, [M], 1024, 640)
        ref = f.fp8_linear(x, wq[0], ws[0], None)
        out = f.fp8_grouped_linear(x, wq, ws, off)
        xq, xs = torch_quant_ref(x)
        r, e = grouped_ref(xq, xs, wq, ws, offs)
        check(out, r, e)
        check(ref, r, e)


@pytest.mark.parametrize("E", [33, 257, 1024])
def test_many_experts(E):
    g = torch.Generator().manual_seed(E)
    counts = torch.randint(0, 4, (E,), generator=g).tolist()
    x, wq, ws, off, offs, _ = make(E, counts, 64, 48)
    xq, xs = torch_quant_ref(x)
    check(f.fp8_grouped_linear(x, wq, ws, off), *grouped_ref(xq, xs, wq, ws, offs))


def test_strided_and_misaligned_inputs():
    x, wq, ws, off, offs, b = make(13, [5, 0, 70], 256, 96, bias=torch.bfloat16)
    ref = f.fp8_grouped_linear(x, wq, ws, off, b)
    wide = torch.zeros(x.shape[0], 300, dtype=x.dtype, device="cuda")
    wide[:, 7:263] = x
    two = torch.stack([wq.view(torch.uint8)] * 2, dim=1).view(torch.float8_e4m3fn)
    off2 = torch.stack([off, off], dim=1)[:, 0]
    wst = ws.t().contiguous().t()
    out = f.fp8_grouped_linear(wide[:, 7:263], two[:, 1], wst, off2, b.t().contiguous().t())
    assert torch.equal(out, ref)


def test_repeatable_and_back_to_back():
    """Equal bits from call to call; calls in a row on one stream do not disturb each other."""
    args = [make(s, c, K, N)[:4] for s, (c, K, N) in enumerate(
        [([1, 2], 2048, 512), ([4] * 50, 512, 640), ([400, 300], 512, 768)])]
    ref = []
    for a in args:
        ref.append(f.fp8_grouped_linear(*a))
        torch.cuda.synchronize()
    for _ in range(3):
        got = [f.fp8_grouped_linear(*a) for a in args + args]
        for r, o in zip(ref + ref, got):
            assert torch.equal(r, o)


def test_weights_and_offsets_written_just_before():
    """The kernel may read weights and offsets before its dependency wait; a writer of both
    right before the call on the stream must still be seen."""
    for counts, K, N in (([2, 3], 4096, 256), ([4] * 64, 512, 768), ([500, 400], 512, 512)):
        x, wq, ws, off, offs, _ = make(17, counts, K, N)
        buf_w, buf_o = torch.zeros_like(wq), torch.zeros_like(off)
        ref = f.fp8_grouped_linear(x, wq, ws, off)
        rev = torch.tensor([0] + [offs[-1]] * (len(offs) - 1), dtype=torch.int32, device="cuda")
        back = wq.view(torch.uint8).flip(0).contiguous().view(wq.dtype)
        ref2 = f.fp8_grouped_linear(x, back, ws, rev)
        torch.cuda.synchronize()
        for _ in range(3):
            buf_w.copy_(wq)
            buf_o.copy_(off)
            a = f.fp8_grouped_linear(x, buf_w, ws, buf_o)
            buf_w.copy_(back)
            buf_o.copy_(rev)
            b = f.fp8_grouped_linear(x, buf_w, ws, buf_o)
            assert torch.equal(a, ref) and torch.equal(b, ref2)


@pytest.mark.parametrize("counts,other", [([2, 3, 1], [0, 6, 0]), ([9] * 70, [630] + [0] * 69),
                                          ([500, 10, 90], [0, 0, 600])])
def test_captured_graph_reads_new_offsets(counts, other):
    x, wq, ws, off, offs, b = make(19, counts, 272, 520, bias=torch.bfloat16)
    f.fp8_grouped_linear(x, wq, ws, off, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f.fp8_grouped_linear(x, wq, ws, off, b)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f.fp8_grouped_linear(x, wq, ws, off, b)
    xq, xs = torch_quant_ref(x)
    for c in (counts, other, counts):
        o = [0]
        for v in c:
            o.append(o[-1] + v)
        off.copy_(torch.tensor(o, dtype=torch.int32))
        graph.replay()
        check(out, *grouped_ref(xq, xs, wq, ws, o, b))


def test_two_streams_at_once():
    a = make(21, [200, 300], 1024, 1024)[:4]
    b = make(22, [3, 1], 1024, 512)[:4]
    ra, rb = f.fp8_grouped_linear(*a), f.fp8_grouped_linear(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            got.append((f.fp8_grouped_linear(*a), ra))
        with torch.cuda.stream(s2):
            got.append((f.fp8_grouped_linear(*b), rb))
    torch.cuda.synchronize()
    for o, r in got:
        assert torch.equal(o, r)


def test_quantize_expert_weights():
    g = torch.Generator(device="cuda").manual_seed(1)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        w = (torch.randn(5, 70, 48, generator=g, device="cuda") * 0.02).to(dt)
        wq, ws = f.quantize_expert_weights(w)
        assert wq.shape == w.shape and ws.shape == (5, 70)
        for e in range(5):
            q, s = f.quantize_weight(w[e])
            assert torch.equal(wq[e].view(torch.uint8), q.view(torch.uint8))
            assert torch.equal(ws[e], s)


def test_capi_matches_op(capi):
    x, wq, ws, off, offs, b = make(23, [3, 0, 90, 7], 400, 333, torch.float16, bias=torch.float32)
    ref = f.fp8_grouped_linear(x, wq, ws, off, b)
    assert torch.equal(capi.fp8_grouped_linear(x, wq, ws, off, b), ref)
    xq, xs = f.quantize_fp8(x)
    assert torch.equal(capi.fp8_grouped_gemm(xq, xs, wq, ws, off, b, out_dtype=torch.float16), ref)


def test_bad_calls_are_refused_on_the_gpu():
    x, wq, ws, off, offs, b = make(25, [3, 4], 64, 32, bias=torch.bfloat16)
    for args in [
        (x.float(), wq, ws, off, b), (x[0], wq, ws, off, b), (x[:, :48], wq, ws, off, b),
        (x, wq[0], ws, off, b), (x, wq, ws.half(), off, b), (x, wq, ws[:1], off, b),
        (x, wq, ws, off.long(), b), (x, wq, ws, off[:2], b), (x, wq, ws, off, b[:1]),
        (x, wq, ws, off.cpu(), b), (x, wq.cpu(), ws, off, b), (x, wq, ws, off, b.cpu()),
        (x, wq[:0], ws[:0], off[:1], None),
        (x[:, :24].contiguous(), wq[:, :, :24].contiguous(), ws, off, b),
    ]:
        with pytest.raises(RuntimeError, match="fp8_grouped_linear"):
            f.fp8_grouped_linear(*args)
