"""GPU parity of the 8-bit linear operator (stof.quant) against the definition in float64.

Quantised values and scales are compared exactly: the scale is one fp32 division, a value the exact quotient
rounded to even.  Outputs: the integer sum is exact; turning it into fp32, the product of the two scales, its
use and the bias are one rounding each (4 x 2^-24 of |sum sx sw| + |bias|), the GELU polynomial is within 2.6e-5
(erf form; tanh form: 2^-20 of its argument), the store half a step of the format."""
import math

import pytest
import torch

from stof.ops import StofError
from stof.quant import gemm_i8, linear_i8, quantize_rows_i8

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _quant64(x):
    """Exact steps (float64 holds the quotient of two 16-bit numbers times 127 far beyond what a tie needs) and fp32 scales."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * x / torch.where(a == 0, 1.0, a))
    return q, (a[..., 0].float() / torch.tensor(127.0))


def _act64(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y.clamp_min(0) if act == "relu" else y


def _want(q, sx, wq, ws, bias, act, dtype):
    raw = (q @ wq.double().t()) * sx.double()[..., None] * ws.double()
    y = raw + (bias.double() if bias is not None else 0.0)
    v = _act64(y, act)
    slack = 4 * 2.0 ** -24 * (raw.abs() + (bias.double().abs() if bias is not None else 0.0))
    if act.startswith("gelu"):
        slack = 1.13 * slack + (2.6e-5 if act == "gelu" else 0.0) + 2.0 ** -20 * y.abs()     # |GELU'| <= 1.13
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return v, slack + u * (v.abs() + slack) + tiny


def _close(got, want, what=""):
    v, bound = want
    err = (got.double().cpu() - v).abs()
    assert got.shape == v.shape and not bool((err > bound).any()) and not bool(torch.isnan(got).any()), \
        f"{what}: {int((err > bound).sum())} beyond the bound, worst {float((err / bound.clamp_min(1e-300)).max()):.2f} of it"


def _weights(N, K, dtype, seed):
    w = (torch.randn(N, K, generator=_gen(seed)) * 0.05).to(dtype)
    q, s = _quant64(w)
    return q.to(torch.int8), s, (torch.randn(N, generator=_gen(seed + 1)) * 0.1).to(dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 16), (5, 48), (64, 512), (3, 1040), (130, 4096), (3, 5008), (9, 8192), (2, 8208), (2, 16384), (3, 16400)])
def test_quantised_rows_exactly(dtype, M, K):
    x = torch.randn(M, K, generator=_gen(K)).to(DT[dtype])
    x[0, 0] = 100.0
    q, s = quantize_rows_i8(x.cuda())
    wq, ws = _quant64(x)
    assert torch.equal(q.cpu().double(), wq) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_value_of_the_format_against_several_maxima(dtype):
    """Ties (x = max / 2 gives 63.5) and everything beside them: all finite patterns of the format below each maximum."""
    pat = torch.arange(0, 65536, dtype=torch.int32).to(torch.int16).view(DT[dtype])
    pat = pat[torch.isfinite(pat)]
    rows = []
    tops = [1.0, 127.0, 254.0, 0.3333, 1.999, 65504.0, 2.0 ** -14, 6e-8] if dtype == "fp16" else [1.0, 127.0, 254.0, 0.3333, 3e38, 1e-30, 2.0 ** -126, 1e-40]
    for t in tops:
        t = torch.tensor(t).to(DT[dtype])
        row = torch.where(pat.double().abs() <= t.double(), pat, t)
        rows.append(torch.cat([row, t.expand(-row.numel() % 16 + 16)]))
    x = torch.stack(rows)
    q, s = quantize_rows_i8(x.cuda())
    wq, ws = _quant64(x)
    assert torch.equal(q.cpu().double(), wq)
    assert torch.equal(s.cpu(), ws)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x = torch.randn(6, 64, generator=_gen(1)).half()
    x[1] = 0
    x[2, 5] = math.inf
    x[3, 63] = math.nan
    x[4] = -0.0
    q, s = quantize_rows_i8(x.cuda())
    assert s.cpu()[[1, 4]].tolist() == [0, 0] and not bool(q[[1, 4]].any())
    assert bool(torch.isnan(s[[2, 3]]).all()) and bool(torch.isfinite(s[[0, 5]]).all())
    w, ws, b = _weights(16, 64, torch.float16, 3)
    for act in ("none", "relu", "gelu"):
        for rows in (x, x.repeat(10, 1)):                    # token form and tile form
            y = linear_i8(rows.cuda(), w.cuda(), ws.cuda(), b.cuda(), act=act).cpu()
            assert bool(torch.isnan(y[[2, 3]]).all()) and bool(torch.isfinite(y[[0, 1, 4, 5]]).all())
            want, bound = _want(*_quant64(x[[0, 1, 4, 5]]), w, ws, b, act, torch.float16)
            assert bool(((y[[0, 1, 4, 5]].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("M", [1, 3, 16, 17, 64, 65, 300])
@pytest.mark.parametrize("N,K", [(8, 16), (40, 144), (136, 1040), (256, 512)])
@pytest.mark.parametrize("dtype,act,bias", [("fp16", "gelu", True), ("bf16", "none", False), ("bf16", "relu", True), ("fp16", "gelu_tanh", False)])
def test_linear_and_product(M, N, K, dtype, act, bias):
    dt = DT[dtype]
    x = torch.randn(M, K, generator=_gen(M + K)).to(dt)
    w, ws, b = _weights(N, K, dt, N)
    b = b if bias else None
    cu = lambda t: None if t is None else t.cuda()
    want = _want(*_quant64(x), w, ws, b, act, dt)
    _close(linear_i8(x.cuda(), w.cuda(), ws.cuda(), cu(b), act=act), want, "linear_i8")
    q, s = quantize_rows_i8(x.cuda())
    _close(gemm_i8(q, s, w.cuda(), ws.cuda(), cu(b), act=act, dtype=dt), want, "gemm_i8")


@pytest.mark.parametrize("M,N,K", [(2048, 2056, 272), (2300, 4104, 144), (200, 264, 2064), (4096, 4104, 2064), (40, 8, 4096)])
def test_every_tile_form_at_its_edges(M, N, K):
    """128 x 128 tiles with two buffers and with one, 64 x 64 with groups along K, 256 x 256: sizes that end inside a tile."""
    x = torch.randn(M, K, generator=_gen(1)).half()
    w, ws, b = _weights(N, K, torch.float16, 2)
    _close(linear_i8(x.cuda(), w.cuda(), ws.cuda(), b.cuda()), _want(*_quant64(x), w, ws, b, "none", torch.float16))


def test_sums_at_the_largest_k():
    """Every product 127 x 127 at the largest K, and -128 x -128, whose sum 2147221504 is the largest there is below 2^31."""
    K = 131056
    x = torch.full((20, K), 3.0).bfloat16()
    w = torch.full((8, K), 127, dtype=torch.int8)
    w[1] = -127
    ws = torch.full((8,), 1e-9)
    for rows in (x, x[:1]):
        y = linear_i8(rows.cuda(), w.cuda(), ws.cuda()).cpu().double()
        want = 3.0 * 127 * K * 1e-9
        assert bool(((y[:, 0] - want).abs() <= 2.0 ** -7 * want).all()) and bool((y[:, 1] == -y[:, 0]).all())
    low = torch.full((20, K), -128, dtype=torch.int8)
    y = gemm_i8(low.cuda(), torch.ones(20).cuda(), low[:8].cuda(), ws.cuda(), dtype=torch.bfloat16).cpu().double()
    assert bool(((y - 2147221504e-9).abs() <= 2.0 ** -8 * 2.15).all())


@pytest.mark.parametrize("M,K", [(16, 4048), (1, 65520), (16, 4096), (2, 32752), (2, 32768), (3, 4640), (15, 2064), (1, 65536)])
def test_token_form_at_the_limit_of_its_lds(M, K):
    """64 KB of quantised rows in LDS, and the first sizes beyond, which take the other form."""
    x = torch.randn(M, K, generator=_gen(M)).bfloat16()
    w, ws, b = _weights(24, K, torch.bfloat16, 3)
    _close(linear_i8(x.cuda(), w.cuda(), ws.cuda(), b.cuda()), _want(*_quant64(x), w, ws, b, "none", torch.bfloat16))


def test_batch_dims_strides_and_guard_rows():
    x = torch.randn(2, 30, 3 * 64, generator=_gen(5)).half()
    w, ws, b = _weights(24, 64, torch.float16, 6)
    part = x.cuda()[..., 64:128]
    want = _want(*_quant64(x[..., 64:128]), w, ws, b, "none", torch.float16)
    _close(linear_i8(part, w.cuda(), ws.cuda(), b.cuda()), want)
    wide = torch.full((24, 96), 55, dtype=torch.int8)
    wide[:, :64] = w
    _close(linear_i8(part, wide.cuda()[:, :64], ws.cuda(), b.cuda()), want, "strided weights")
    q, s = quantize_rows_i8(part)
    assert q.shape == (2, 30, 64) and s.shape == (2, 30)
    qw = torch.full((60, 128), 77, dtype=torch.int8, device="cuda")
    qw[:, :64] = q.view(60, 64)
    _close(gemm_i8(qw[:, :64], s.view(60), w.cuda(), ws.cuda(), b.cuda()).view(2, 30, 24), want, "strided rows")
    for M in (7, 60):
        buf = torch.full((M + 8, 24), 9.0, dtype=torch.float16, device="cuda")
        rows = x.view(60, 192)[:M, :64].contiguous()
        linear_i8(rows.cuda(), w.cuda(), ws.cuda(), b.cuda(), out=buf[4:4 + M])
        _close(buf[4:4 + M], _want(*_quant64(rows), w, ws, b, "none", torch.float16))
        assert bool((buf[:4] == 9).all()) and bool((buf[4 + M:] == 9).all())
    assert linear_i8(x.cuda()[:0, :, :64], w.cuda(), ws.cuda()).shape == (0, 30, 24)
    odd = torch.randn(4, 65, generator=_gen(7)).half().cuda()[:, 1:]      # rows that cannot be read as they lie: a copy
    _close(linear_i8(odd, w.cuda(), ws.cuda(), b.cuda()), _want(*_quant64(odd.cpu()), w, ws, b, "none", torch.float16))


@pytest.mark.parametrize("M,K,N", [(1, 96, 8200), (2, 1040, 8208), (5, 64, 20000), (16, 512, 16392)])
def test_token_form_with_several_feature_blocks_per_workgroup(M, K, N):
    x = torch.randn(M, K, generator=_gen(M)).half()
    w, ws, b = _weights(N, K, torch.float16, 4)
    _close(linear_i8(x.cuda(), w.cuda(), ws.cuda(), b.cuda(), act="gelu"), _want(*_quant64(x), w, ws, b, "gelu", torch.float16))


def test_two_streams_at_once():
    w, ws, b = (t.cuda() for t in _weights(520, 272, torch.float16, 18))
    xs = [torch.randn(m, 272, generator=_gen(m)).half().cuda() for m in (300, 333)]
    want = [linear_i8(x, w, ws, b) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(linear_i8(xs[n], w, ws, b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[n]) for n in range(2) for g in got[n])


def test_captured_graphs_replayed_together():
    w, ws, b = (t.cuda() for t in _weights(512, 256, torch.float16, 8))
    for M in (1, 100):
        x = torch.randn(M, 256, generator=_gen(9)).half().cuda()
        call = lambda: linear_i8(x, w, ws, b, act="gelu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                y = call()
            graphs.append((gr, y))
        for seed in (1, 2, 3):
            x.copy_(torch.randn(x.shape, generator=_gen(seed)))
            want = call()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graphs[0][0].replay()
            graphs[1][0].replay()
            torch.cuda.synchronize()
            assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_refusals():
    h = lambda *s, d=torch.float16: torch.zeros(*s, dtype=d, device="cuda")
    x, w, s, b = h(4, 64), h(16, 64, d=torch.int8), h(16, d=torch.float32), h(16)
    bad = [
        lambda: linear_i8(x.cpu(), w, s),
        lambda: linear_i8(x.float(), w, s),
        lambda: linear_i8(x.clone().requires_grad_(), w, s),
        lambda: linear_i8(x, w.half(), s),
        lambda: linear_i8(x, w[:, :48], s),
        lambda: linear_i8(x, h(12, 64, d=torch.int8), s[:12]),
        lambda: linear_i8(x, w, s.half()),
        lambda: linear_i8(x, w, s[:8]),
        lambda: linear_i8(x, w, s, b.bfloat16()),
        lambda: linear_i8(x, w, s, b[:8]),
        lambda: linear_i8(x, w, s, b, act="silu"),
        lambda: linear_i8(x, w, s, out=h(4, 24)),
        lambda: linear_i8(x, w, s, out=h(4, 16, d=torch.bfloat16)),
        lambda: linear_i8(h(4, 40), h(16, 40, d=torch.int8), s),
        lambda: linear_i8(x, h(16, 72, d=torch.int8)[:, :64], s),       # rows 72 bytes apart
        lambda: linear_i8(x, w.cpu(), s),
        lambda: quantize_rows_i8(h(4, 40)),
        lambda: quantize_rows_i8(h(4, 0)),
        lambda: quantize_rows_i8(x.float()),
        lambda: gemm_i8(x, s[:4], w, s),
        lambda: gemm_i8(w[:4], s[:3], w, s),
        lambda: gemm_i8(w[:4], s[:4], w, s, dtype=torch.float32),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(StofError):
            call()
            pytest.fail(f"refusal {n} was accepted")


def test_parameters_that_ask_for_a_gradient():
    h = lambda *s, d=torch.float16: torch.zeros(*s, dtype=d, device="cuda")
    x, w, s, b = h(4, 64), h(16, 64, d=torch.int8), h(16, d=torch.float32), h(16)
    ask = lambda t: t.clone().requires_grad_()
    calls = [lambda: linear_i8(x, w, s, ask(b)), lambda: linear_i8(x, w, ask(s), b), lambda: gemm_i8(w[:4], s[:4], w, s, ask(b)),
             lambda: gemm_i8(w[:4], s[:4], w, ask(s), b), lambda: gemm_i8(w[:4], ask(s[:4]), w, s)]
    for n, call in enumerate(calls):
        with pytest.raises(StofError, match="gradient"):
            call()
            pytest.fail(f"call {n} was accepted")
        with torch.no_grad():
            call()


def test_contiguous_rows_at_an_odd_address():
    """A view at an odd offset of a flat buffer is contiguous and cannot be read as it lies: a copy, as for odd strides."""
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    w, ws = quantize_rows_i8(torch.randn(16, 64, generator=torch.Generator().manual_seed(4)).half().cuda())
    flat = torch.empty(4 * 64 + 1, dtype=torch.float16, device="cuda")
    odd = flat[1:].view(4, 64)
    odd.copy_(x)
    q, s = quantize_rows_i8(x)
    q2, s2 = quantize_rows_i8(odd)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    assert torch.equal(linear_i8(odd, w, ws), linear_i8(x, w, ws)) and torch.equal(linear_i8(odd[:1], w, ws), linear_i8(x[:1], w, ws))
    flat8 = torch.empty(4 * 64 + 8, dtype=torch.int8, device="cuda")
    odd8 = flat8[8:].view(4, 64)
    odd8.copy_(q)
    assert torch.equal(gemm_i8(odd8, s, w, ws), gemm_i8(q, s, w, ws))
