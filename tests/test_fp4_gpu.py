"""The microscaled 4-bit operators against their definitions in 64 bits (oracle/fp4.py).

Tolerances.  Quantisation is exact: every rounding decision is taken on exact quotients, so
codes and scales have to match in value.  A product of 4-bit operands has exact terms; the
tensor core adds 64 of them to an fp32 accumulator per step and each step is off by at most
2^-21 of the sum of magnitudes S = |a| |w|^T (fp32 truncation of the running sum and of the
aligned terms), so the accumulator is within ceil(K / 64) 2^-21 S; the bf16 result adds half an
ulp, 2^-8 of its magnitude at most.  Where a value computed in fp32 is then quantised, a value
within its error e of a midpoint may take the other code: the allowed difference is that
between the codes of |h| - e and |h| + e.
"""
import math

import pytest
import torch

from oracle import fp4 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
FMTS = ["nv", "mx"]
BF16 = 2.0 ** -8


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def acts(g, M, K):
    x = randn(g, M, K)
    return x * torch.where(torch.rand(K, generator=g, device=DEV) < 0.05, 8.0, 1.0)


def steps(K):
    return -(-K // 64) * 2.0 ** -21


def check(out, ref, tol):
    assert out.shape == ref.shape
    d = (out.double() - ref).abs()
    assert bool((d <= tol).all()), (d / tol.clamp(min=1e-300)).max().item()


def same(a, b):
    """Equal values, NaN where the other is NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ----------------------------------------------------------------------------- quantisation
def check_quant(x, fmt):
    from flashvsr_sm89_ops_b200 import dequantize_fp4, quantize_fp4
    q = quantize_fp4(x, fmt)
    v, _, row = R.quantize(x.cpu(), fmt)
    assert same(R.values(q), v)
    assert not R.padding(q).any()
    if fmt == "nv":
        assert torch.equal(q.row_scale.cpu().double(), row)
    else:
        assert q.row_scale is None
    for dt in (torch.bfloat16, torch.float32):
        # a block scale rounded up at the very top of the range can stand for more than fp32 holds
        assert same(dequantize_fp4(q, dt).cpu().double(), v.float().to(dt).double())
    return q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (1, 1536), (3, 33), (129, 63), (7, 65), (200, 512),
                                 (5, 1000), (33, 1536), (2, 2049), (130, 4608), (9, 8960), (2, 10241),
                                 (3, 16385)])
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_exact(M, K, dtype, fmt):
    check_quant(acts(gen(M * 7 + K), M, K).to(dtype), fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_every_bf16_value(fmt):
    """Every finite bf16 value, alone in its block and next to each larger power of two."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[torch.isfinite(x.float())]
    rows = []
    for up in (0, 1, 3):
        b = torch.zeros(x.numel(), 32, dtype=torch.bfloat16)
        b[:, 0] = x
        # a neighbour that sets the block's scale (3.4e38 stays finite)
        b[:, 7] = (x.float().abs() * 2.0 ** up * 1.25).clamp(max=3.3e38).to(torch.bfloat16) if up else 0
        rows.append(b)
    check_quant(torch.cat(rows).to(DEV), fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties(fmt):
    """Exact midpoints of codes (against every E4M3 mantissa for nv) and of E4M3 scales."""
    rows = []
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for m in range(8):
        for e in (-3, 0, 5):
            s = (1 + m / 8) * 2.0 ** e
            r = torch.zeros(64)
            r[0:8], r[8:16] = mids * s, -mids * s
            r[16:24] = mids * s * (1 + 2.0 ** -20)
            r[31] = 6 * s
            r[24] = 5 * s * (1 - 2.0 ** -20)
            r[48] = 6 * s * (1 + 1 / 16)  # amax / 6 half way between two E4M3 values
            r[32 + 5] = 6 * s * (1 + 3 / 16)
            rows.append(r)
    check_quant(torch.stack(rows).to(DEV), fmt)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_extremes(fmt, dtype):
    """Zero rows and blocks, the largest and smallest magnitudes, infinities and NaN."""
    g = gen(5)
    x = randn(g, 12, 96).to(dtype)
    big = torch.finfo(dtype).max
    x[0] = 0
    x[1, 16:48] = 0
    x[2] = big
    x[3, 0] = -big
    x[4] = x[4].float().mul(1e-38).to(dtype)
    x[5, 3] = math.inf
    x[6, 40] = math.nan
    x[6, 41] = -math.inf
    x[7] = math.nan
    x[8] = -0.0
    x[9, :] = torch.finfo(dtype).tiny
    x[10, 0:16] = 1e-30
    x[11, 95] = -math.inf
    q = check_quant(x, fmt)
    v = R.values(q)
    assert v[7].isnan().all() and v[0].abs().max() == 0
    n = R.BLOCK[fmt]
    assert v[5, :n].isnan().all() and not v[5, n:].isnan().any()


@pytest.mark.parametrize("dtype,bits,low", [(torch.bfloat16, 8, -126), (torch.float16, 11, -14),
                                            (torch.float32, 24, -126)])
def test_dequantize_rounds_once(dtype, bits, low):
    """Any fp32 row scale, chosen so that a code times its scales lies within an fp32 rounding of
    the middle of two neighbours of the output type; and row scales at the ends of fp32's range."""
    from flashvsr_sm89_ops_b200 import FP4Tensor, dequantize_fp4
    g = torch.Generator().manual_seed(bits)
    p = torch.tensor([c * (1 + j / 8) for c in (1.0, 1.5) for j in range(8)], dtype=torch.float64)
    i = torch.randint(2 ** min(bits - 1, 20), (400,), generator=g).double()
    mid = (2.0 ** (bits - 1) + i + 0.5) / 2.0 ** (bits - 1)
    row = (mid[:, None] / p).float().reshape(-1)
    row = torch.cat((row, -row[:64], torch.tensor([2.0 ** -149, 2.0 ** -126, 1.7e-38, 2.0 ** 119, 2.0 ** 127, 0.0])))
    M = row.numel()
    codes = torch.full((M, 16), 0x20, dtype=torch.uint8)  # codes 0 (value 0) and 2 (value 1)
    codes[:, 1::2] = 0xB2  # 2 (1) and 11 (-1.5)
    tiles = torch.zeros(-(-M // 128) * 512, dtype=torch.uint8)
    m = torch.arange(M)
    for j in (0, 1):  # E4M3 1 .. 1.875
        tiles[m // 128 * 512 + m % 32 * 16 + m % 128 // 32 * 4 + j] = (0x38 + m % 8).to(torch.uint8)
    q = FP4Tensor(codes.to(DEV), tiles.to(DEV), row.to(DEV), (M, 32), "nv")
    v = R.values(q)
    e = (torch.frexp(v)[1] - 1).clamp(min=low).double()
    step = torch.pow(torch.full_like(v, 2.0), e - bits + 1)
    want = torch.round(v / step) * step
    want = torch.where(want.abs() > torch.finfo(dtype).max, want * math.inf, want)
    assert torch.equal(dequantize_fp4(q, dtype).cpu().double(), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_strides(fmt):
    """Row pitches, unaligned starts, a transposed view: all as their contiguous copy."""
    from flashvsr_sm89_ops_b200 import dequantize_fp4, quantize_fp4
    base = acts(gen(8), 70, 400).to(torch.bfloat16)
    for x in (base[:, :200], base[:, 8:208], base[:, 3:203], base[::2, 5:], base.t(), base[:1, 7:],
              base[:, 9:10], base[:1].expand(6, 400)):
        a = dequantize_fp4(quantize_fp4(x, fmt))
        assert torch.equal(a, dequantize_fp4(quantize_fp4(x.contiguous(), fmt)))
        assert torch.equal(a.cpu().double(), R.quantize(x.cpu(), fmt)[0])


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_empty(fmt):
    from flashvsr_sm89_ops_b200 import dequantize_fp4, quantize_fp4
    for shape in ((0, 64), (4, 0), (0, 0)):
        q = quantize_fp4(torch.empty(shape, dtype=torch.bfloat16, device=DEV), fmt)
        assert dequantize_fp4(q).shape == shape


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_offsets_past_32_bits(fmt):
    """More than 2^31 elements: the last rows are where 32-bit offsets would have wrapped."""
    from flashvsr_sm89_ops_b200 import dequantize_fp4, quantize_fp4
    K = 16384
    M = 2 ** 31 // K + 130
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = acts(gen(3), 3, K).to(torch.bfloat16)
    q = quantize_fp4(x, fmt)
    ref = R.quantize(x[-3:].cpu(), fmt)[0]
    v = dequantize_fp4(q)
    assert torch.equal(v[-3:].cpu().double(), ref)
    assert not v[:64].any() and not v[M // 2:M // 2 + 64].any()


# ----------------------------------------------------------------------------- product
def mm_case(M, N, K, fmt, seed=0):
    from flashvsr_sm89_ops_b200 import quantize_fp4
    g = gen(seed + M + 3 * N + 5 * K)
    a = quantize_fp4(acts(g, M, K).to(torch.bfloat16), fmt)
    w = quantize_fp4(randn(g, N, K) * K ** -0.5, fmt)
    bias = (randn(g, N) * 0.1).to(torch.bfloat16)
    res = randn(g, M, N).to(torch.bfloat16)
    gate = randn(g, N).to(torch.bfloat16)
    return a, w, bias, res, gate


def mm_ref(a, w):
    """(a w^T, |a| |w|^T) in 64 bits."""
    va, vw = R.values(a).to(DEV), R.values(w).to(DEV)
    return va @ vw.t(), va.abs() @ vw.abs().t()


SIZES = [(1, 1, 1), (1, 8, 64), (1, 1536, 1536), (2, 257, 100), (5, 64, 8960), (16, 136, 1000),
         (17, 1544, 257), (33, 40, 2048), (64, 512, 512), (100, 136, 1000), (128, 128, 256),
         (127, 129, 4600), (129, 256, 320), (130, 264, 96), (257, 72, 1536), (300, 333, 1000),
         (256, 512, 65), (517, 1544, 1000), (1000, 1536, 1536), (700, 2000, 8960)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("fmt", FMTS)
def test_product(M, N, K, fmt):
    from flashvsr_sm89_ops_b200 import _lib, fp4_mm
    a, w, bias, res, gate = mm_case(M, N, K, fmt)
    y, S = mm_ref(a, w)
    acc = steps(K) * S
    check(fp4_mm(a, w), y, BF16 * y.abs() + acc)
    yb = y + bias.double()
    check(fp4_mm(a, w, bias), yb, BF16 * yb.abs() + acc + 2.0 ** -22 * yb.abs())
    # two more fp32 roundings at most, each 2^-24 of the magnitudes it adds
    o = res.double() + gate.double() * yb
    mag = res.double().abs() + gate.double().abs() * (yb.abs() + S)
    check(fp4_mm(a, w, bias, residual=res, gate=gate), o,
          BF16 * o.abs() + gate.double().abs() * acc + 2.0 ** -22 * mag)
    o = res.double() + y
    check(fp4_mm(a, w, residual=res), o, BF16 * o.abs() + acc + 2.0 ** -22 * (res.double().abs() + S))
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_product_many_tiles(fmt):
    """More tiles than the grid holds, so both accumulators are used again and again."""
    from flashvsr_sm89_ops_b200 import fp4_mm
    for M, N, K in ((5000, 4608, 192), (4000, 120, 640), (120, 40000, 128)):
        a, w, bias, res, gate = mm_case(M, N, K, fmt)
        y, S = mm_ref(a, w)
        y = y + bias.double()
        check(fp4_mm(a, w, bias), y, BF16 * y.abs() + (steps(K) + 2.0 ** -22) * S + 2.0 ** -22 * y.abs())


@pytest.mark.parametrize("M,N,K", [(2500, 2056, 300), (2305, 2001, 1000), (4000, 1544, 64), (3000, 1536, 1600),
                                   (2049, 2600, 2300), (4100, 4000, 520)])
@pytest.mark.parametrize("fmt", FMTS)
def test_product_pair_tiles(M, N, K, fmt):
    """Sizes that run on CTA pairs: rows and columns that end inside a tile or leave a pair's
    second CTA without rows, K that ends inside a block, odd N (no TMA for the output)."""
    from flashvsr_sm89_ops_b200 import _lib, fp4_mm
    a, w, bias, res, gate = mm_case(M, N, K, fmt)
    y, S = mm_ref(a, w)
    acc = steps(K) * S
    check(fp4_mm(a, w), y, BF16 * y.abs() + acc)
    yb = y + bias.double()
    o = res.double() + gate.double() * yb
    mag = res.double().abs() + gate.double().abs() * (yb.abs() + S)
    tol = BF16 * o.abs() + gate.double().abs() * acc + 2.0 ** -22 * mag
    check(fp4_mm(a, w, bias, residual=res, gate=gate), o, tol)
    wide = torch.zeros(M, N + 3, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:N + 1] = res
    check(fp4_mm(a, w, bias, residual=wide[:, 1:N + 1], gate=gate), o, tol)
    out = res.clone()
    fp4_mm(a, w, bias, residual=out, gate=gate, out=out)
    check(out, o, tol)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("M,N,K", [(1, 128, 512), (3, 300, 2048), (128, 1536, 4096), (129, 1536, 8960),
                                   (40, 130, 9000), (200, 520, 2100), (256, 256, 20000)])
@pytest.mark.parametrize("fmt", FMTS)
def test_product_parts_of_k(M, N, K, fmt):
    """Sizes whose K is divided among the CTAs of a cluster: the same bits every time."""
    from flashvsr_sm89_ops_b200 import _lib, fp4_mm
    a, w, bias, res, gate = mm_case(M, N, K, fmt)
    y, S = mm_ref(a, w)
    yb = y + bias.double()
    out = fp4_mm(a, w, bias)
    check(out, yb, BF16 * yb.abs() + steps(K) * S + 2.0 ** -21 * (yb.abs() + S))
    for _ in range(3):
        assert torch.equal(fp4_mm(a, w, bias), out)
    o = res.double() + gate.double() * yb
    mag = res.double().abs() + gate.double().abs() * (yb.abs() + S)
    check(fp4_mm(a, w, bias, residual=res, gate=gate), o,
          BF16 * o.abs() + gate.double().abs() * steps(K) * S + 2.0 ** -21 * mag)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("M", [1, 3, 200])
def test_product_row_scale_forms(M):
    """nv operands whose second scale is one number or missing, as checkpoints ship them."""
    from flashvsr_sm89_ops_b200 import FP4Tensor, fp4_mm
    a, w, *_ = mm_case(M, 96, 160, "nv")
    for rs_a, rs_w in ((torch.tensor([0.37], device=DEV), torch.tensor([1.7], device=DEV)),
                       (None, None), (torch.tensor([0.37], device=DEV), w.row_scale)):
        a2 = FP4Tensor(a.codes, a.scales, rs_a, a.shape, "nv")
        w2 = FP4Tensor(w.codes, w.scales, rs_w, w.shape, "nv")
        y, S = mm_ref(a2, w2)
        # the row scales multiply the finished sum: two more fp32 roundings
        check(fp4_mm(a2, w2), y, BF16 * y.abs() + (steps(160) + 2.0 ** -22) * S)


@pytest.mark.parametrize("M", [3, 200])
@pytest.mark.parametrize("fmt", FMTS)
def test_product_nan_scale_stays_in_its_row(fmt, M):
    """A NaN scale makes its own row (of A) or column (of W) NaN and nothing else; scales
    beyond the matrix are never read into a result."""
    from flashvsr_sm89_ops_b200 import fp4_mm, quantize_fp4
    g = gen(9)
    x = randn(g, M, 200).to(torch.bfloat16)
    wt = randn(g, 70, 200)
    x[1, 130] = math.nan
    wt[33, 5] = math.inf
    a, w = quantize_fp4(x, fmt), quantize_fp4(wt, fmt)
    y = fp4_mm(a, w)
    n = y.isnan()
    assert n[1].all() and n[:, 33].all()
    n[1], n[:, 33] = False, False
    assert not n.any()


@pytest.mark.parametrize("fmt", FMTS)
def test_product_in_place_strided_and_unaligned(fmt):
    from flashvsr_sm89_ops_b200 import fp4_mm
    for M, N in ((3, 64), (200, 264), (140, 77)):
        a, w, bias, res, gate = mm_case(M, N, 128, fmt)
        want = fp4_mm(a, w, bias, residual=res, gate=gate)
        wide = torch.randn(M, N + 5, device=DEV).to(torch.bfloat16)
        wide[:, 3:3 + N] = res
        assert torch.equal(fp4_mm(a, w, bias, residual=wide[:, 3:3 + N], gate=gate), want)
        shifted = torch.empty(N + 1, dtype=torch.bfloat16, device=DEV)
        shifted[1:] = bias
        assert torch.equal(fp4_mm(a, w, shifted[1:], residual=res, gate=gate), want)
        out = res.clone()
        assert fp4_mm(a, w, bias, residual=out, gate=gate, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want)
        odd = torch.empty(M * N + 1, dtype=torch.bfloat16, device=DEV)[1:].view(M, N)
        assert torch.equal(fp4_mm(a, w, bias, residual=res, gate=gate, out=odd), want)


def test_product_is_repeatable_and_graph_safe():
    """The same bits on every call, on a side stream and from a CUDA graph."""
    from flashvsr_sm89_ops_b200 import dequantize_fp4, fp4_mm, quantize_fp4
    for M in (1, 40, 700):
        g = gen(M)
        x = acts(g, M, 1536).to(torch.bfloat16)
        w = quantize_fp4(randn(g, 1544, 1536) / 40, "nv")
        want = fp4_mm(quantize_fp4(x, "nv"), w)
        for _ in range(3):
            assert torch.equal(fp4_mm(quantize_fp4(x, "nv"), w), want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            side = fp4_mm(quantize_fp4(x, "nv"), w)
            back = dequantize_fp4(quantize_fp4(x, "nv"))
        s.synchronize()
        assert torch.equal(side, want)
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp4_mm(quantize_fp4(static, "nv"), w)
        static.copy_(x.flip(1))
        graph.replay()
        assert torch.equal(y, fp4_mm(quantize_fp4(x.flip(1), "nv"), w))
        static.copy_(x)
        graph.replay()
        assert torch.equal(y, want)
        assert torch.equal(back, dequantize_fp4(quantize_fp4(x, "nv")))


@pytest.mark.parametrize("N", [8192, 8191])
def test_product_offsets_past_32_bits(N):
    """An output and a residual of more than 2^31 elements, with and without TMA for them."""
    from flashvsr_sm89_ops_b200 import FP4Tensor, fp4_mm
    M = 2 ** 31 // N + 300
    a, w, bias, res, gate = mm_case(300, N, 64, "mx")
    # the same 300 rows first and last, zero codes between
    codes = torch.zeros(M, 32, dtype=torch.uint8, device=DEV)
    codes[:300], codes[-300:] = a.codes, a.codes
    last = torch.arange(M - 300, M, device=DEV)
    scales = torch.zeros(-(-M // 128) * 512, dtype=torch.uint8, device=DEV)
    for rows in (torch.arange(300, device=DEV), last):
        for j in range(2):
            at = rows // 128 * 512 + rows % 32 * 16 + rows % 128 // 32 * 4 + j
            own = torch.arange(300, device=DEV)
            scales[at] = a.scales[own // 128 * 512 + own % 32 * 16 + own % 128 // 32 * 4 + j]
    big = FP4Tensor(codes, scales, None, (M, 64), "mx")
    residual = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    residual[:300], residual[-300:] = res, res
    out = fp4_mm(big, w, bias, residual=residual, gate=gate, out=residual)
    y, S = mm_ref(a, w)
    yb = y + bias.double()
    o = res.double() + gate.double() * yb
    mag = res.double().abs() + gate.double().abs() * (yb.abs() + S)
    tol = BF16 * o.abs() + gate.double().abs() * steps(64) * S + 2.0 ** -22 * mag
    check(out[:300], o, tol)
    check(out[-300:], o, tol)


# ----------------------------------------------------------------------------- FFN
def spread(h, e, fmt):
    """How far apart the quantised values of |h| - e and |h| + e are, elementwise: what an
    error of e before the quantisation can change, block scales included."""
    a = h.abs()
    lo, hi = (a - e).clamp(min=0), a + e
    vs = [R.quantize(t, fmt)[0] for t in (lo, a, hi)]
    d = torch.stack(vs)
    out = d.amax(0) - d.amin(0)
    # a scale that moves moves every code of its block (nv: of its row) by up to half a step
    # of the larger scale on top
    s = [R.quantize(t, fmt)[1] for t in (lo, a, hi)]
    moved = ((s[0] != s[1]) | (s[1] != s[2]))
    top = torch.stack(s).amax(0)
    n = R.BLOCK[fmt]
    return out + (moved * top).repeat_interleave(n, 1)[:, :h.shape[1]] * 2


@pytest.mark.parametrize("M,D,F,N", [(1, 64, 32, 64), (3, 256, 500, 96), (13, 1000, 1000, 136),
                                     (100, 136, 1544, 137), (128, 256, 256, 256), (129, 264, 4096, 264),
                                     (300, 1536, 8960, 1536), (700, 72, 2056, 512),
                                     (2500, 264, 2056, 1500), (2309, 200, 2001, 2003), (5000, 100, 1040, 72)])
@pytest.mark.parametrize("fmt", FMTS)
def test_ffn(M, D, F, N, fmt):
    from flashvsr_sm89_ops_b200 import _lib, ffn_fp4, quantize_fp4
    g = gen(M + D + F)
    a = quantize_fp4(acts(g, M, D).to(torch.bfloat16), fmt)
    w0 = quantize_fp4(randn(g, F, D) * D ** -0.5, fmt)
    w2 = quantize_fp4(randn(g, N, F) * F ** -0.5, "mx")
    b0, b2 = (randn(g, F) * 0.1).to(torch.bfloat16), (randn(g, N) * 0.1).to(torch.bfloat16)
    res, gate = randn(g, M, N).to(torch.bfloat16), randn(g, N).to(torch.bfloat16)
    u, S0 = mm_ref(a, w0)
    u = u + b0.double()
    h = R.gelu_tanh(u)
    # GELU's slope is below 1.13; its own fp32 evaluation is within 2^-20 of |u| (a sum, an
    # exponential and a reciprocal of a few ulp each)
    e = 1.13 * (steps(D) * S0 + 2.0 ** -22 * (S0 + u.abs())) + 2.0 ** -20 * u.abs()
    hq = R.quantize(h, "mx")[0]
    vw = R.values(w2).to(DEV)
    y = hq @ vw.t() + b2.double()
    S2 = hq.abs() @ vw.abs().t()
    err = steps(F) * S2 + spread(h, e, "mx") @ vw.abs().t() * (1 + 2.0 ** -10) + 2.0 ** -22 * (y.abs() + S2)
    check(ffn_fp4(a, w0, b0, w2, b2), y, BF16 * (y.abs() + err) + err)
    o = res.double() + gate.double() * y
    eo = gate.double().abs() * err + 2.0 ** -22 * (res.double().abs() + o.abs())
    check(ffn_fp4(a, w0, b0, w2, b2, residual=res, gate=gate), o, BF16 * (o.abs() + eo) + eo)
    ws = torch.empty(_lib.load().fvb_fp4_ffn_workspace_bytes(M, F), dtype=torch.uint8, device=DEV)
    ws.fill_(255)  # a NaN in every scale: nothing may be read that was not written
    assert torch.equal(ffn_fp4(a, w0, b0, w2, b2, workspace=ws), ffn_fp4(a, w0, b0, w2, b2))
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def test_ffn_hidden_extremes():
    """Hidden values from exactly 0 to far past GELU's tails stay finite and right."""
    from flashvsr_sm89_ops_b200 import ffn_fp4, quantize_fp4
    M, D, F = 40, 64, 96
    x = torch.zeros(M, D, device=DEV)
    x[:, 0] = torch.linspace(-3000, 3000, M, device=DEV)
    w0 = torch.zeros(F, D, device=DEV)
    w0[:, 0] = torch.logspace(-6, 1, F, device=DEV)
    w2 = torch.eye(F, device=DEV)[:64].contiguous()
    a, q0, q2 = quantize_fp4(x.to(torch.bfloat16), "nv"), quantize_fp4(w0, "nv"), quantize_fp4(w2, "mx")
    y = ffn_fp4(a, q0, None, q2, None)
    u, S = mm_ref(a, q0)
    h = R.gelu_tanh(u)
    e = 2.0 ** -19 * u.abs()
    ref = R.quantize(h, "mx")[0][:, :64]
    check(y, ref, spread(h, e, "mx")[:, :64] + BF16 * ref.abs())


@pytest.mark.parametrize("M,F", [(98, 64), (2500, 2080)])
@pytest.mark.parametrize("fmt", FMTS)
def test_ffn_hidden_deep_negative(fmt, M, F):
    """Blocks of nothing but large negative hidden values, to -2^100, are exactly 0 (GELU of
    -7.5 is -4e-18), on few tiles and on pairs; -inf makes its row NaN as the formula does."""
    from flashvsr_sm89_ops_b200 import ffn_fp4, quantize_fp4
    x = torch.zeros(M, 64, device=DEV)
    x[:, 0] = -torch.pow(2.0, torch.arange(M, device=DEV) % 98 + 3)
    w0 = torch.zeros(F, 64, device=DEV)
    w0[:, 0] = 1.0
    w2 = torch.zeros(40, F, device=DEV)
    w2[torch.arange(40), torch.arange(40)] = 1.0
    a, q0, q2 = quantize_fp4(x.to(torch.bfloat16), fmt), quantize_fp4(w0, fmt), quantize_fp4(w2, "mx")
    assert mm_ref(a, q0)[0].max() < -7.5  # nv's scale of a lone 8 is within 1/16 of 8 / 6
    assert not ffn_fp4(a, q0, None, q2, None).any()
    b0 = torch.zeros(F, dtype=torch.bfloat16, device=DEV)
    b0[35] = -math.inf
    assert ffn_fp4(a, q0, b0, q2, None).isnan().all()


def test_ffn_hidden_negative_tail():
    """Hidden values -4, -4.25, ... -9, each a block of its own, so that its scale is theirs."""
    from flashvsr_sm89_ops_b200 import ffn_fp4, quantize_fp4
    n = 21
    u = -(4 + torch.arange(n, device=DEV) / 4)
    F = 32 * n
    a = quantize_fp4(torch.zeros(5, 64, device=DEV), "nv")
    q0 = quantize_fp4(torch.ones(F, 64, device=DEV), "nv")
    w2 = torch.zeros(n, F, device=DEV)
    w2[torch.arange(n), 32 * torch.arange(n)] = 1.0
    y = ffn_fp4(a, q0, u.repeat_interleave(32).to(torch.bfloat16), quantize_fp4(w2, "mx"), None)
    # in 64 bits 1 + tanh cancels: x / (1 + exp(-2 u)) is the same formula
    x = u.double().repeat_interleave(32)
    h = (x / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))).expand(5, F)
    # v (61 at most) carries 6 roundings of 2^-24, so 2^v is within 2^-15; below -7.5 the value is 0
    e = 2.0 ** -15 * h.abs() + 4.2e-18
    ref = R.quantize(h, "mx")[0]
    check(y, ref[:, ::32], (spread(h, e, "mx") + BF16 * ref.abs())[:, ::32])


# ----------------------------------------------------------------------------- residual norm
def rn_case(B, L, D, seed=0):
    g = gen(seed + B + L + D)
    bf = torch.bfloat16
    return {"x": (randn(g, B, L, D) * 2).to(bf), "y": (acts(g, B * L, D).view(B, L, D) + 0.25).to(bf),
            "gate": randn(g, B, 1, D).to(bf), "rows": randn(g, B, L, D).to(bf),
            "pw": (1 + 0.1 * randn(g, D)).to(bf), "pb": (0.1 * randn(g, D)).to(bf),
            "w": (1 + 0.1 * randn(g, D)).to(bf), "b": (0.1 * randn(g, D)).to(bf),
            "scale": (0.2 * randn(g, B, 1, D)).to(bf), "shift": (0.2 * randn(g, B, 1, D)).to(bf)}


FULL = dict(gate="gate", post_weight="pw", post_bias="pb", weight="w", bias="b", scale="scale",
            shift="shift")


def rn_check(c, names, emit=None, **kw):
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    t = {k: c[v] for k, v in names.items()}
    r = fused_residual_norm(c["x"], c["y"], **t, **kw, emit_fp4=emit)
    ok = {k: v for k, v in kw.items() if k != "want_out"}
    ok["norm_kind"] = ok.pop("norm", "layer")
    xn, h = R.residual_norm(c["x"], c["y"], **t, **ok)
    # fp32 sums of D terms, tree-added: 2^-20 of what is added bounds each chain of roundings
    g = t["gate"].double() if "gate" in t else torch.ones(1, device=DEV, dtype=torch.float64)
    y = c["y"].double()
    post = kw.get("post_norm")
    pr = 1.0
    if post is not None:
        v = y - y.mean(-1, keepdim=True) if post == "layer" else y
        pr = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + kw.get("post_eps", 1e-6))
    rms = torch.sqrt((y * y).mean(-1, keepdim=True)) if post else 0.0
    pw = t["post_weight"].double().abs() if "post_weight" in t else 1.0
    pb = t["post_bias"].double().abs() if "post_bias" in t else 0.0
    mag = abs(kw.get("residual_scale", 1.0)) * c["x"].double().abs() + g.abs() * ((y.abs() + rms) * pr * pw + pb)
    ex = 2.0 ** -20 * mag
    check(r[0], xn, BF16 * xn.abs() + ex * 1.01)
    v = xn - xn.mean(-1, keepdim=True) if kw.get("norm", "layer") == "layer" else xn
    nr = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + kw.get("eps", 1e-6))
    m2 = (mag + torch.sqrt((mag * mag).mean(-1, keepdim=True))) * nr
    # the normed value's error: its own and the statistics', which are as exact relative to the
    # row's magnitudes
    m2 = m2 + (v * nr).abs() * torch.sqrt((mag * mag).mean(-1, keepdim=True)) * nr
    w = t["weight"].double().abs() if "weight" in t else 1.0
    b = t["bias"].double().abs() if "bias" in t else 0.0
    s = (1 + t["scale"].double()).abs() if "scale" in t else 1.0
    sh = t["shift"].double().abs() if "shift" in t else 0.0
    eh = 2.0 ** -19 * ((m2 * w + b) * s + sh)
    if r[1] is not None:
        check(r[1], h, BF16 * h.abs() + eh * 1.01)
    if emit:
        D = h.shape[-1]
        q = r[2]
        ref = R.quantize(h.reshape(-1, D), emit)[0]
        d = (R.values(q).to(DEV) - ref).abs()
        assert bool((d <= spread(h.reshape(-1, D), eh.expand_as(h).reshape(-1, D), emit)).all())
        assert not R.padding(q).any()
    return r


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("B,L,D", [(1, 1, 8), (2, 3, 64), (3, 7, 1000), (1, 9, 1536), (2, 5, 2048),
                                   (1, 3, 4608), (1, 2, 8960), (1, 1, 16384)])
def test_residual_norm(B, L, D, post, norm):
    c = rn_case(B, L, D)
    names = {k: v for k, v in FULL.items() if post or not k.startswith("post")}
    rn_check(c, names, post_norm=post, norm=norm, residual_scale=0.75, eps=1e-5, post_eps=1e-6)
    rn_check(c, {}, post_norm=post, norm=norm)


@pytest.mark.parametrize("emit", FMTS)
@pytest.mark.parametrize("B,L,D", [(1, 1, 8), (2, 3, 40), (1, 130, 64), (2, 67, 264), (3, 43, 1000),
                                   (1, 9, 1536), (2, 5, 2040), (1, 3, 4608), (1, 2, 16384)])
def test_residual_norm_emits_codes(B, L, D, emit):
    c = rn_case(B, L, D)
    rn_check(c, FULL, emit=emit, post_norm="rms", norm="layer")
    r = rn_check(c, dict(scale="scale", shift="shift"), emit=emit, norm="layer", want_out=False)
    assert r[1] is None


@pytest.mark.parametrize("emit", FMTS)
def test_residual_norm_codes_on_midpoints(emit):
    """An h that is exact in fp32 (scale -1 leaves the shift) gets the codes of its definition:
    every midpoint of two codes under every E4M3 mantissa, on its even side."""
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    exact = torch.cat([torch.cat((mids, -mids)) * (1 + j / 8) * 2.0 ** e for e in (-3, 0, 5) for j in range(8)])
    h = exact.to(torch.bfloat16)
    assert torch.equal(h.float(), exact)
    D = h.numel()
    z = torch.zeros(1, 3, D, dtype=torch.bfloat16, device=DEV)
    minus = torch.full((1, 1, D), -1.0, dtype=torch.bfloat16, device=DEV)
    _, out, q = fused_residual_norm(z, z, scale=minus, shift=h.view(1, 1, D).to(DEV), emit_fp4=emit)
    assert torch.equal(out[0].cpu(), h.expand(3, D))
    assert torch.equal(R.values(q), R.quantize(h.expand(3, D), emit)[0])


@pytest.mark.parametrize("emit", FMTS)
@pytest.mark.parametrize("B,L,D", [(1, 1200, 1536), (3, 401, 1040), (2, 600, 1032)])
def test_residual_norm_emits_codes_for_many_rows(B, L, D, emit):
    """Rows enough for one warp each."""
    c = rn_case(B, L, D)
    rn_check(c, {k: v for k, v in FULL.items() if k != "post_bias"}, emit=emit, post_norm="rms", norm="layer")
    rn_check(c, dict(FULL, gate="rows"), emit=emit, post_norm="layer", norm="rms")


@pytest.mark.parametrize("emit", [None] + FMTS)
@pytest.mark.parametrize("D", [256, 512, 1024, 2048, 4096, 8192])
def test_residual_norm_widest_rows(D, emit):
    """The widest row of each layout, whose column operands fill the layout's shared memory."""
    c = rn_case(2, 5, D)
    rn_check(c, {k: v for k, v in FULL.items() if k != "post_bias"}, emit=emit, post_norm="rms", norm="layer")
    rn_check(c, FULL, emit=emit, post_norm="layer", norm="rms")


@pytest.mark.parametrize("emit", FMTS)
def test_residual_norm_offsets_past_32_bits(emit):
    """More than 2^31 elements: the last rows get what they get alone."""
    from flashvsr_sm89_ops_b200 import dequantize_fp4, fused_residual_norm
    D = 8192
    L = 2 ** 31 // D + 130
    c = rn_case(1, 5, D)
    x = torch.zeros(1, L, D, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros_like(x)
    x[:, -5:], y[:, -5:] = c["x"], c["y"]
    kw = dict(gate=c["gate"], scale=c["scale"], shift=c["shift"], post_norm="rms", emit_fp4=emit)
    xn, h, q = fused_residual_norm(x, y, **kw)
    xs, hs, qs = fused_residual_norm(c["x"], c["y"], **kw)
    assert torch.equal(xn[:, -5:], xs) and torch.equal(h[:, -5:], hs)
    assert not xn[:, :64].any() and torch.equal(h[:, L // 2], c["shift"][:, 0])
    v = dequantize_fp4(q)
    assert torch.equal(v[-5:], dequantize_fp4(qs))
    assert torch.equal(v[:1], v[L // 2:L // 2 + 1]) and v[:1].any()


def test_residual_norm_gate_forms():
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    c = rn_case(2, 6, 264)
    rn_check(c, dict(FULL, gate="rows"), post_norm="rms", norm="rms")
    full = c["gate"].expand(2, 6, 264)
    a = fused_residual_norm(c["x"], c["y"], gate=full, post_norm="rms")
    b = fused_residual_norm(c["x"], c["y"], gate=c["gate"], post_norm="rms")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    nc = c["x"].transpose(0, 1)
    a = fused_residual_norm(nc, c["y"].transpose(0, 1))
    b = fused_residual_norm(nc.contiguous(), c["y"].transpose(0, 1).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_residual_norm_unaligned_views():
    """Operands that start off a 16-byte boundary: as their aligned copies."""
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    c = rn_case(2, 6, 264)

    def off(t):
        wide = torch.empty(t.numel() + 3, dtype=t.dtype, device=DEV)[3:].view(t.shape)
        return wide.copy_(t)

    for gate in ("gate", "rows"):
        t = {k: c[v] for k, v in dict(FULL, gate=gate).items()}
        a = fused_residual_norm(c["x"], c["y"], post_norm="layer", emit_fp4="nv", **t)
        b = fused_residual_norm(off(c["x"]), off(c["y"]), post_norm="layer", emit_fp4="nv",
                                **{k: off(v) for k, v in t.items()})
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(R.values(a[2]), R.values(b[2]))


def test_residual_norm_refuses_operands_of_another_shape():
    """As many entries in another order: [1, L, D] with L = B is not a row for each batch item."""
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    for B, L, D in ((2, 2, 64), (3, 2, 64)):
        x = randn(gen(4), B, L, D).to(torch.bfloat16)
        for name in ("gate", "scale", "shift"):
            t = randn(gen(5), B, 1, D).to(torch.bfloat16)
            a = fused_residual_norm(x, x, **{name: t})
            b = fused_residual_norm(x, x, **{name: t.view(B, D)})
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            for shape in ((1, B, D), (B, D, 1), (1, 1, B * D)):
                with pytest.raises(ValueError, match=name):
                    fused_residual_norm(x, x, **{name: t.reshape(shape)})
        rows = randn(gen(6), B, L, D).to(torch.bfloat16)
        for shape in ((1, B * L, D), (B, D, L)) + (((L, B, D),) if L != B else ()):
            with pytest.raises(ValueError, match="gate"):
                fused_residual_norm(x, x, gate=rows.reshape(shape))


def test_residual_norm_extremes():
    """Constant and zero rows (a variance of 0), and a NaN that stays in its row."""
    from flashvsr_sm89_ops_b200 import dequantize_fp4, fused_residual_norm
    x = torch.zeros(1, 5, 96, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros_like(x)
    x[0, 1] = 3.0
    x[0, 2] = randn(gen(1), 96).to(torch.bfloat16)
    x[0, 3, 7] = math.nan
    x[0, 4] = randn(gen(2), 96).to(torch.bfloat16)
    for norm in ("rms", "layer"):
        for post in (None, "rms", "layer"):
            xn, h, q = fused_residual_norm(x, y, norm=norm, post_norm=post, emit_fp4="nv")
            v = dequantize_fp4(q)
            bad = torch.tensor([False, False, False, True, False], device=DEV)
            assert torch.equal(h[0].isnan().any(-1), bad) and torch.equal(v.isnan().any(-1), bad)
            assert not h[0, 0].any() and torch.equal(xn[0, 4], x[0, 4])
            want = torch.zeros(96, device=DEV) if norm == "layer" else torch.ones(96, device=DEV)
            assert torch.equal(h[0, 1].float(), want)


FIRST_CALLS = """
import threading
import torch
from flashvsr_sm89_ops_b200 import _lib
lib, bad = _lib.load(), []

def go(d, p, rows, fmt, bar):
    bar.wait()
    for _ in range(3):
        q = p[5:] if fmt else [None] * 3
        rc = lib.fvb_residual_norm(p[0], p[1], p[2] if rows else None, rows, 1.0, 0, None, None, 1e-6, 2, None,
                                   None, None, None, 1e-6, 1, 2, d, p[3], p[4], fmt, *q, None)
        if rc:
            bar.bad.append((d, rc, lib.fvb_last_error()))

for fmt in (0, 1, 2):
    for rows in (0, 1):
        for dims in ((4104, 8184, 6000, 8184), (8200, 16376, 12000, 16376)):
            bar = threading.Barrier(len(dims))
            bar.bad = bad
            bufs = [[torch.zeros(128 * d, dtype=torch.uint8, device="cuda") for _ in range(8)] for d in dims]
            torch.cuda.synchronize()
            ts = [threading.Thread(target=go, args=(d, [t.data_ptr() for t in b], rows, fmt, bar))
                  for d, b in zip(dims, bufs)]
            [t.start() for t in ts]
            [t.join() for t in ts]
            torch.cuda.synchronize()
assert not bad, bad
"""


def test_residual_norm_first_calls_from_threads():
    """Rows of different widths from several threads at once, in a process that has not launched
    these kernels before: every call gets the shared memory of its own width."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("emit", FMTS)
@pytest.mark.parametrize("L,D", [(3, 40), (5, 256), (3, 1000), (2, 1536), (1200, 1536), (2, 4104)])
def test_residual_norm_nonfinite_columns(L, D, emit):
    """An infinity or NaN in one column of h makes that column's block NaN and no other; the
    block's finite values still count in the row's maximum."""
    from flashvsr_sm89_ops_b200 import fused_residual_norm
    c = rn_case(1, L, D)
    n = R.BLOCK[emit]
    shift = c["shift"].clone()
    hot = (D // 3) // n * n
    shift[0, 0, hot] = 300.0  # the row's maximum, in the block that is then spoilt
    _, _, ref = fused_residual_norm(c["x"], c["y"], scale=c["scale"], shift=shift, emit_fp4=emit)
    for bad in (math.inf, -math.inf, math.nan):
        spoilt = shift.clone()
        spoilt[0, 0, hot + 5] = spoilt[0, 0, D - 1] = bad
        _, h, q = fused_residual_norm(c["x"], c["y"], scale=c["scale"], shift=spoilt, emit_fp4=emit)
        v, want = R.values(q), R.values(ref)
        nan = torch.zeros(D, dtype=torch.bool)
        nan[hot:hot + n] = nan[(D - 1) // n * n:] = True
        assert torch.equal(v.isnan(), nan.expand(L, D))
        assert torch.equal(v[:, ~nan], want[:, ~nan])
        assert not R.padding(q).any()


def test_empty_batches():
    from flashvsr_sm89_ops_b200 import ffn_fp4, fp4_mm, fused_residual_norm, quantize_fp4
    x = torch.empty(2, 0, 64, dtype=torch.bfloat16, device=DEV)
    xn, h, q = fused_residual_norm(x, x, emit_fp4="mx")
    assert xn.shape == h.shape == x.shape and q.shape == (0, 64)
    w = quantize_fp4(torch.randn(32, 64, device=DEV), "mx")
    w2 = quantize_fp4(torch.randn(16, 32, device=DEV), "mx")
    assert fp4_mm(q, w).shape == (0, 32)
    assert ffn_fp4(q, w, None, w2, None).shape == (0, 16)


# ----------------------------------------------------------------------------- modules, refusals
def test_linear_and_ffn_modules():
    """The modules equal the operators they chain, for any leading shape."""
    import torch.nn as nn
    from flashvsr_sm89_ops_b200 import FP4FFN, FP4Linear, ffn_fp4, fp4_mm, quantize_fp4
    torch.manual_seed(0)
    x = torch.randn(2, 5, 136, device=DEV, dtype=torch.bfloat16)
    l0, l2 = nn.Linear(136, 200).to(DEV), nn.Linear(200, 136, bias=False).to(DEV)
    for fmt in FMTS:
        m = FP4Linear(l0, fmt)
        y = m(x)
        assert y.shape == (2, 5, 200)
        a = quantize_fp4(x.view(10, 136), fmt)
        assert torch.equal(y.view(10, 200), fp4_mm(a, quantize_fp4(l0.weight, fmt), l0.bias))
        f = FP4FFN(m, FP4Linear(l2, "mx"))
        want = ffn_fp4(a, m.weight_fp4(), l0.bias, quantize_fp4(l2.weight, "mx"), None)
        assert torch.equal(f(x).view(10, 136), want)
        # a cast of the whole model leaves its results alone: row scales are powers of two
        assert torch.equal(FP4Linear(l0, fmt).to(torch.bfloat16)(x), y)
    with pytest.raises(ValueError, match="mx"):
        FP4FFN(FP4Linear(l0, "nv"), FP4Linear(l2, "nv"))


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_survives_a_cast_of_the_model(fmt):
    """Row scales far outside fp16 (weights near 1e-9 and 1e9) after .to(fp16 / fp64)."""
    import torch.nn as nn
    from flashvsr_sm89_ops_b200 import FP4Linear
    lin = nn.Linear(64, 48, bias=False).to(DEV)
    with torch.no_grad():
        lin.weight[:16] *= 1e-9
        lin.weight[16:32] *= 1e9
    x = randn(gen(1), 5, 64).to(torch.bfloat16)
    y = FP4Linear(lin, fmt)(x)
    assert y[:, :16].any() and torch.isfinite(y).all()
    for dt in (torch.float16, torch.float64, torch.bfloat16):
        assert torch.equal(FP4Linear(lin, fmt).to(dt)(x), y)


def test_refusals():
    from flashvsr_sm89_ops_b200 import (FP4Tensor, dequantize_fp4, ffn_fp4, fp4_mm,
                                        fused_residual_norm, quantize_fp4)
    x = torch.randn(4, 64, device=DEV, dtype=torch.bfloat16)
    a, w = quantize_fp4(x, "nv"), quantize_fp4(torch.randn(8, 64, device=DEV), "nv")
    m = quantize_fp4(x, "mx")
    bad = [
        lambda: quantize_fp4(x, "fp4"),
        lambda: quantize_fp4(x[0]),
        lambda: quantize_fp4(x.int()),
        lambda: quantize_fp4(x.cpu()),
        lambda: dequantize_fp4(a, torch.int8),
        lambda: fp4_mm(a, m),
        lambda: fp4_mm(a, quantize_fp4(torch.randn(8, 32, device=DEV), "nv")),
        lambda: fp4_mm(a, w, torch.zeros(7, device=DEV)),
        lambda: fp4_mm(a, w, torch.zeros(8)),
        lambda: fp4_mm(a, w, gate=torch.zeros(8, device=DEV)),
        lambda: fp4_mm(a, w, residual=torch.zeros(4, 9, device=DEV, dtype=torch.bfloat16)),
        lambda: fp4_mm(a, w, residual=torch.zeros(4, 8, device=DEV)),
        lambda: fp4_mm(a, w, out=torch.zeros(4, 8, device=DEV)),
        lambda: ffn_fp4(a, w, None, w, None),
        lambda: ffn_fp4(a, w, None, quantize_fp4(torch.randn(4, 9, device=DEV), "mx"), None),
        lambda: ffn_fp4(a, w, None, quantize_fp4(torch.randn(4, 8, device=DEV), "mx"), None,
                        workspace=torch.empty(8, dtype=torch.uint8, device=DEV)),
        lambda: FP4Tensor(a.codes, a.scales[:-1], a.row_scale, a.shape, "nv"),
        lambda: FP4Tensor(a.codes, a.scales, a.row_scale[:3], a.shape, "nv"),
        lambda: FP4Tensor(a.codes[:, :16], a.scales, a.row_scale, a.shape, "nv"),
        lambda: FP4Tensor(m.codes, m.scales, a.row_scale, m.shape, "mx"),
        lambda: fused_residual_norm(x, x),
        lambda: fused_residual_norm(x[None], x[None, :3]),
        lambda: fused_residual_norm(x[None], x[None].float()),
        lambda: fused_residual_norm(x[None], x[None], norm="batch"),
        lambda: fused_residual_norm(x[None], x[None], post_weight=x[0]),
        lambda: fused_residual_norm(x[None], x[None], want_out=False),
        lambda: fused_residual_norm(x[None], x[None], emit_fp4="int4"),
        lambda: fused_residual_norm(x[None], x[None], gate=x[:2]),
        lambda: fused_residual_norm(x[None, :, :60], x[None, :, :60]),
        lambda: fused_residual_norm(x[None], x[None].cpu()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    torch.cuda.synchronize()


def test_ffn_refuses_a_workspace_with_less_memory_than_entries():
    from flashvsr_sm89_ops_b200 import _lib, ffn_fp4, quantize_fp4
    a = quantize_fp4(torch.randn(200, 64, device=DEV), "mx")
    w0, w2 = (quantize_fp4(torch.randn(s, device=DEV), "mx") for s in ((96, 64), (8, 96)))
    need = _lib.load().fvb_fp4_ffn_workspace_bytes(200, 96)
    wide = torch.empty(256, dtype=torch.uint8, device=DEV)[:1].expand(need)
    with pytest.raises(ValueError, match="contiguous"):
        ffn_fp4(a, w0, None, w2, None, workspace=wide)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert torch.equal(ffn_fp4(a, w0, None, w2, None, workspace=ws), ffn_fp4(a, w0, None, w2, None))


# ----------------------------------------------------------------------------- the model's path
def small_dit(device, dtype=torch.bfloat16):
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    dit = W.WanDiT(num_layers=1, dim=256, num_heads=2, ffn_dim=512).init_random(seed=3)
    return W, dit.to(dtype).to(device)


@pytest.mark.parametrize("fmt", FMTS)
def test_enable_on_a_host_model(fmt, monkeypatch):
    """enable() before the model is moved to the GPU gives the weights of enable() after it."""
    from flashvsr_sm89_ops_b200 import integrate
    monkeypatch.setenv("FS89_FP4_FMT", fmt)
    made = []
    for device in ("cpu", DEV):
        W, dit = small_dit(device)
        applied = integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False, fp4_parts=["ffn"])
        assert applied["fp4_linears"] == 2
        lin = dit.blocks[0].ffn.lin0
        assert all(t.device.type == torch.device(device).type for t in (lin.weight, lin.w_scales, lin.bias))
        made.append(dit.to(DEV).blocks[0].ffn)
    x = randn(gen(2), 3, 5, 256).to(torch.bfloat16)
    a, b = made
    for s, t in ((a.lin0, b.lin0), (a.lin2, b.lin2)):
        assert torch.equal(s.weight, t.weight)
        assert torch.equal(R.values(s.weight_fp4()), R.values(t.weight_fp4()))
    assert torch.equal(a(x), b(x))


def test_enable_again_with_other_parts(monkeypatch):
    """A second enable() without the 4-bit parts leaves them as they are and converts the rest;
    one with them again too; the other format is refused."""
    from flashvsr_sm89_ops_b200 import FP4FFN, FP8Linear, integrate
    W, dit = small_dit(DEV)
    monkeypatch.delenv("FS89_FP4", raising=False)
    pipe = W.DiTPipe(dit)
    assert integrate.enable(pipe, dit_module=W, parts=[], verbose=False, fp4_parts=["ffn"])["fp4_linears"] == 2
    ffn = dit.blocks[0].ffn
    for _ in range(2):
        applied = integrate.enable(pipe, dit_module=W, verbose=False)
        assert applied["fp8_ffn_blocks"] == 0 and dit.blocks[0].ffn is ffn and type(ffn) is FP4FFN
        assert type(dit.blocks[0].self_attn.q) is FP8Linear
    assert integrate.enable(pipe, dit_module=W, verbose=False, fp4_parts=["ffn"])["fp4_linears"] == 0
    monkeypatch.setenv("FS89_FP4_FMT", "mx")
    with pytest.raises(ValueError, match="already nv"):
        integrate.enable(pipe, dit_module=W, verbose=False, fp4_parts=["ffn"])
    assert dit.blocks[0].ffn is ffn


@pytest.mark.parametrize("fmt", FMTS)
def test_block_with_a_4bit_ffn(fmt, monkeypatch):
    """enable() with FS89_FP4=ffn: the block's FFN half equals its definition in 64 bits on the
    tensors that reached it, and the FP8 half before it is untouched."""
    from flashvsr_sm89_ops_b200 import FP4FFN, _lib, integrate
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    from oracle import wan as OW
    f, h, w = 2, 16, 24
    P, x, t_mod, ctx, cache = OW.block_case(seed=4, f=f, h=h, w=w)
    W.MASK_RULE = "causal"
    state = OW.standin_state_dict(P)

    def block(fp4):
        dit = W.WanDiT(num_layers=1).to(torch.bfloat16)
        dit.blocks[0].load_state_dict(state, strict=True)
        dit = dit.to(DEV)
        monkeypatch.setenv("FS89_FP4", "ffn" if fp4 else "")
        monkeypatch.setenv("FS89_FP4_FMT", fmt)
        applied = integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False)
        assert applied.get("fp4_linears") == (2 if fp4 else None)
        assert integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False).get("fp4_linears", 0) == 0
        dit.init_cross_kv(ctx.to(DEV))
        return dit

    def run(dit):
        fr = W.grid_freqs(dit.freqs, f, h, w, f0=6).to(DEV)
        with torch.no_grad():
            return dit.blocks[0](x.to(DEV), None, t_mod.to(DEV), fr, f, h, w, kv_len=3, is_stream=True,
                                 pre_cache_k=cache[0].to(DEV), pre_cache_v=cache[1].to(DEV))

    y8, k8, v8 = run(block(False))
    dit = block(True)
    ffn = dit.blocks[0].ffn
    assert isinstance(ffn, FP4FFN) and ffn.lin0.fmt == fmt and ffn.lin2.fmt == "mx"
    seen = {}
    seam = integrate.fused_residual_norm

    def spy(xx, yy, **kw):
        seen.update(x=xx.clone(), y=yy.clone(), kw=kw)
        return seam(xx, yy, **kw)

    monkeypatch.setattr(integrate, "fused_residual_norm", spy)
    y4, k4, v4 = run(dit)
    assert torch.equal(k4, k8) and torch.equal(v4, v8)
    kw = seen["kw"]
    D = x.shape[-1]
    xn, hn = R.residual_norm(seen["x"], seen["y"], norm_kind="layer", scale=kw["scale"], shift=kw["shift"],
                             eps=kw["eps"])
    a = R.quantize(hn.reshape(-1, D), fmt)[0]
    u = a @ R.quantize(state["ffn.0.weight"].to(DEV), fmt)[0].t() + state["ffn.0.bias"].to(DEV).double()
    hq = R.quantize(R.gelu_tanh(u), "mx")[0]
    o = hq @ R.quantize(state["ffn.2.weight"].to(DEV), "mx")[0].t() + state["ffn.2.bias"].to(DEV).double()
    mod = dit.blocks[0].modulation.double() + t_mod.to(DEV).double()
    want = xn.reshape(-1, D).to(torch.bfloat16).double() + mod[:, 5] * o
    err = ((y4.double().reshape(-1, D) - want).norm() / want.norm()).item()
    # bf16 modulation and result: a few 2^-9 relative
    assert err < 4 * 2.0 ** -9, err
    assert _lib.device_error() == 0


class Captured:
    """A 4-bit linear of the oracle's block: the output that the block's own linear gave.  Checks
    that output against the linear's definition in 64 bits on the input that the linear had, and
    that the oracle has come to the same input."""

    def __init__(self, w, b, fmt):
        self.w, self.s = R.quantize(w.to(DEV), fmt)[0], []
        self.b, self.fmt = b.to(DEV).double(), fmt

    def saw(self, x, y):
        x2, y2 = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
        a = R.quantize(x2, self.fmt)[0]
        ref, S = a @ self.w.t() + self.b, a.abs() @ self.w.abs().t()
        check(y2, ref, BF16 * ref.abs() + (steps(x2.shape[1]) + 2.0 ** -22) * S + 2.0 ** -22 * ref.abs())
        self.s.append((x.cpu(), y.cpu()))

    def __call__(self, x):
        from oracle import wan as OW
        xin, y = self.s.pop(0)
        assert OW.rel_l2(x.reshape(xin.shape), xin) < 2e-2
        return y


@pytest.mark.parametrize("fmt", FMTS)
def test_block_with_4bit_attention(fmt, monkeypatch):
    """enable() with FS89_FP4=self,cross: the block against the oracle's (2e-2 relative L2, the bar
    of the FP8 block's test) with the 4-bit linears' own outputs in it, each of them held against its
    definition; and all of it on the fused paths."""
    from flashvsr_sm89_ops_b200 import FP4Linear, _lib, integrate
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    from oracle import wan as OW
    f, h, w, heads = 2, 16, 24, 12
    P, x, t_mod, ctx, cache = OW.block_case(seed=6, f=f, h=h, w=w)
    W.MASK_RULE = "causal"
    monkeypatch.setenv("FS89_FP4", "self,cross")
    monkeypatch.setenv("FS89_FP4_FMT", fmt)
    monkeypatch.setenv("FS89_FP8_SCALE", "token")
    dit = W.WanDiT(num_layers=1).to(torch.bfloat16)
    dit.blocks[0].load_state_dict(OW.standin_state_dict(P), strict=True)
    dit = dit.to(DEV)
    applied = integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False)
    assert applied["fp4_linears"] == 8 and applied["fp8_linears"] == 2
    blk = dit.blocks[0]
    Q = OW.quantize_block(P, "token")
    sd = OW.to_bf16(P)
    for part, mod in (("self", blk.self_attn), ("cross", blk.cross_attn)):
        for n in ("q", "k", "v", "o"):
            lin = getattr(mod, n)
            assert type(lin) is FP4Linear and lin.fmt == fmt
            Q[part][n] = cap = Captured(*sd[part][n], fmt)
            lin.register_forward_hook(lambda m, i, o, cap=cap: cap.saw(i[0], o))
    quant, mm = integrate.quantize_fp4, integrate.fp4_mm
    fused = []

    def spy_quant(t, f):
        fused.append(t)
        return quant(t, f)

    def spy_mm(*a):
        y = mm(*a)
        for n, part in zip("qkv", y.chunk(3, 1)):
            Q["self"][n].saw(fused[0][None], part[None])
        return y

    monkeypatch.setattr(integrate, "quantize_fp4", spy_quant)
    monkeypatch.setattr(integrate, "fp4_mm", spy_mm)
    with torch.no_grad():
        dit.init_cross_kv(ctx.to(DEV))
        fr = W.grid_freqs(dit.freqs, f, h, w, f0=6).to(DEV)
        y, ck, cv = blk(x.to(DEV), None, t_mod.to(DEV), fr, f, h, w, kv_len=3, is_stream=True,
                        pre_cache_k=cache[0].to(DEV), pre_cache_v=cache[1].to(DEV))
    assert len(fused) == 1  # one product for q, k and v
    assert hasattr(ck, "_fvb_arena") and hasattr(ck, "_fvb_kpool")  # the fused self-attention's caches
    cos, sin = OW.O.freqs_cos_sin(OW.grid_freqs(f, h, w, f0=6))
    ref, (rk, rv) = OW.block_forward(Q, x, t_mod, cos, sin, (f, h, w), OW.cross_kv(Q, ctx),
                                     OW.causal_mask_fn(heads, 6, 0.25), heads, cache, 3)
    e, ek, ev = OW.rel_l2(y.cpu(), ref), OW.rel_l2(ck.cpu(), rk), OW.rel_l2(cv.cpu(), rv)
    assert e < 2e-2 and ek < 2e-2 and ev < 2e-2, (e, ek, ev)
    assert all(not Q[p][n].s for p in ("self", "cross") for n in "qkvo")
    assert _lib.device_error() == 0


@pytest.mark.parametrize("parts", ["ffn", "self", "ffn,self,cross"])
def test_streaming_step_in_4_bits_replays_from_a_graph(parts, monkeypatch):
    """The f = 6 start chunk and the streaming step with 4-bit parts, eagerly and from a CUDA graph."""
    from flashvsr_sm89_ops_b200 import _lib
    from flashvsr_sm89_ops_b200.runner import StreamingDiT
    monkeypatch.setenv("FS89_FP4", parts)
    r = StreamingDiT(num_layers=2, height=256, width=384, device=DEV)
    assert r.applied["fp4_linears"] == 2 * (2 * ("ffn" in parts) + 4 * ("self" in parts) + 4 * ("cross" in parts))
    r.prime()
    x = r.make_input(2)
    eager = r.step(x).clone()
    assert torch.isfinite(eager).all()
    g, y = r.capture(x)
    x.copy_(r.make_input(2, seed=9))
    g.replay()
    assert torch.equal(y, r.step(x)) and not torch.equal(y, eager)
    x.copy_(r.make_input(2))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, eager)
    assert _lib.device_error() == 0
