"""The 4-bit operators where no GPU is needed: host-side checks of the C entry points, sizes of
their buffers, and the oracle of tests/test_fp4_gpu.py against hand-written values."""
import math

import pytest
import torch

from oracle import fp4 as R


def test_entry_points_check_arguments_on_the_host():
    from flashvsr_sm89_ops_b200 import _lib
    lib = _lib.load()
    bad, ok = _lib.FVB_ERR_INVALID, _lib.FVB_OK
    p = 4096  # any aligned address: nothing is launched
    assert lib.fvb_quant_fp4(None, 0, 0, -1, 4, 1, None, None, None, None) == bad
    assert lib.fvb_quant_fp4(p, 0, 0, 4, 64, 3, p, p, p, None) == bad  # format
    assert lib.fvb_quant_fp4(p, 9, 0, 4, 64, 1, p, p, p, None) == bad  # dtype
    assert lib.fvb_quant_fp4(p, 0, 0, 4, 64, 1, p, p, None, None) == bad  # nv without row_scale
    assert lib.fvb_quant_fp4(p, 0, 63, 4, 64, 1, p, p, p, None) == bad  # row pitch
    assert lib.fvb_quant_fp4(p, 0, 0, 4, 64, 2, p + 8, p, None, None) == bad  # alignment
    assert lib.fvb_quant_fp4(p, 0, 0, 1 << 31, 64, 2, p, p, None, None) == bad
    assert lib.fvb_quant_fp4(None, 0, 0, 0, 64, 1, None, None, None, None) == ok
    assert lib.fvb_dequant_fp4(p, p, None, 5, 4, 64, 1, 0, p, None) == bad
    assert lib.fvb_dequant_fp4(None, p, None, 0, 4, 64, 1, 0, p, None) == bad

    def gemm(A=p, M=4, N=8, K=64, fmt=1, bias=None, res=None, ldr=0, gate=None, out=p):
        return lib.fvb_fp4_gemm(A, p, None, 0, p, p, None, 0, fmt, bias, res, ldr, gate, M, N, K,
                                out, None)
    assert gemm(A=None) == bad and gemm(A=p + 1) == bad and gemm(K=0) == bad and gemm(M=-1) == bad
    assert gemm(fmt=0) == bad and gemm(out=None) == bad and gemm(gate=p) == bad
    assert gemm(res=p, ldr=7) == bad and gemm(M=1 << 31) == bad
    assert gemm(M=0) == ok and gemm(N=0) == ok
    ffn = [p, p, None, 0, p, p, None, 0, 1, None, p, p, None, None, 0, None, 4, 64, 32, 8, p, p, None]
    assert lib.fvb_fp4_ffn(*ffn[:21], p + 16, None) == bad  # workspace alignment
    assert lib.fvb_fp4_ffn(*ffn[:21], None, None) == bad
    assert lib.fvb_fp4_ffn(*ffn[:18], 0, *ffn[19:]) == bad  # F = 0
    assert lib.fvb_fp4_ffn(*ffn[:16], 0, *ffn[17:]) == ok

    def norm(x=p, post=0, nrm=2, B=1, L=2, D=64, out=p, fmt=0, codes=None):
        return lib.fvb_residual_norm(x, p, None, 0, 1.0, post, None, None, 1e-6, nrm, None, None,
                                     None, None, 1e-6, B, L, D, p, out, fmt, codes, codes, codes, None)
    assert norm(x=None) == bad and norm(D=60) == bad and norm(D=16392) == bad and norm(post=3) == bad
    assert norm(nrm=0) == bad and norm(out=None) == bad and norm(fmt=1) == bad and norm(x=p + 2) == bad
    assert norm(fmt=7, codes=p) == bad and norm(B=0) == ok
    assert "fvb_residual_norm" in lib.fvb_last_error().decode()


def test_ffn_entry_point_refuses_before_it_launches():
    """What only the second product would refuse is refused at once."""
    from flashvsr_sm89_ops_b200 import _lib
    p = 4096
    good = dict(A=p, sfA=p, rsA=None, am=0, W0=p, sfW0=p, rsW0=None, wm=0, fmt=1, b0=None, W2=p, sfW2=p,
                b2=None, res=None, ldr=0, gate=None, M=4, D=64, F=32, N=8, out=p, ws=p, stream=None)
    for bad in (dict(W2=None), dict(sfW2=None), dict(out=None), dict(W2=p + 8), dict(sfW2=p + 1),
                dict(gate=p), dict(res=p, ldr=7)):
        assert _lib.load().fvb_fp4_ffn(*{**good, **bad}.values()) == _lib.FVB_ERR_INVALID, bad


def test_buffer_sizes():
    from flashvsr_sm89_ops_b200 import _lib
    lib = _lib.load()
    assert lib.fvb_fp4_codes_bytes(3, 33) == 3 * 32
    assert lib.fvb_fp4_scales_bytes(1, 64, 1) == 512 and lib.fvb_fp4_scales_bytes(1, 65, 1) == 1024
    assert lib.fvb_fp4_scales_bytes(129, 128, 2) == 1024 and lib.fvb_fp4_scales_bytes(128, 129, 2) == 1024
    assert lib.fvb_fp4_scales_bytes(4, 4, 3) == 0
    # held as [M, F] bf16 the hidden state would take 8448 * 8960 * 2
    assert lib.fvb_fp4_ffn_workspace_bytes(8448, 8960) < 8448 * 8960 * 2 / 3.7


def test_fp4_tensor_checks_and_cpu_refusal():
    from flashvsr_sm89_ops_b200 import FP4Tensor, dequantize_fp4, fused_residual_norm, quantize_fp4
    codes, scales = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    q = FP4Tensor(codes, scales, torch.ones(2), (2, 64), "nv")
    assert "nv" in repr(q) and q.row_mode() == 1
    assert FP4Tensor(codes, scales, torch.ones(1), (2, 64), "nv").row_mode() == 0
    for args in ((codes.int(), scales, None, (2, 64), "nv"), (codes, scales[1:], None, (2, 64), "nv"),
                 (codes, scales, torch.ones(3), (2, 64), "nv"), (codes, scales, None, (2, 65), "nv"),
                 (codes, scales, torch.ones(2).double(), (2, 64), "nv"),
                 (codes, scales, torch.ones(2), (2, 64), "mx"), (codes, scales, None, (2, 64), "e2m1")):
        with pytest.raises(ValueError):
            FP4Tensor(*args)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for f in (lambda: quantize_fp4(x), lambda: dequantize_fp4(q),
              lambda: fused_residual_norm(x[None], x[None])):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_oracle_rounds_as_written():
    x = torch.tensor([0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 9.0], dtype=torch.float64)
    assert R.e2m1(x).tolist() == [0, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6]
    y = torch.tensor([0, 2.0 ** -10, 1.5 * 2.0 ** -9, 1.0625, 1.1875, 447, 500], dtype=torch.float64)
    assert R.e4m3(y).tolist() == [0, 0, 2.0 ** -8, 1, 1.25, 448, 448]
    # mx: amax 7 -> scale 1, saturated at 6; amax 8 -> scale 2
    r = torch.zeros(1, 64)
    r[0, :3] = torch.tensor([7.0, -0.5, 0.2])
    r[0, 32:35] = torch.tensor([8.0, 1.0, 0.5])
    v, s, row = R.quantize(r, "mx")
    assert s.tolist() == [[1, 2]] and row is None
    assert v[0, :3].tolist() == [6, -0.5, 0] and v[0, 32:35].tolist() == [8, 1, 0]
    # nv: amax 2688 keeps the row scale at 1, just above it doubles it
    for top, k in ((2688.0, 1.0), (2689.0, 2.0), (1344.0, 0.5)):
        r = torch.zeros(1, 16)
        r[0, 0] = top
        v, s, row = R.quantize(r, "nv")
        assert row.item() == k and v[0, 0] == min(top, 6 * s.item())
    r[0, 3] = math.nan
    assert R.quantize(r, "nv")[0].isnan().all() and R.quantize(torch.zeros(2, 16), "nv")[2].tolist() == [1, 1]


def test_values_reads_the_documented_layout():
    from flashvsr_sm89_ops_b200 import FP4Tensor
    M, K = 130, 80  # two bands of rows, two tiles a band (5 blocks of 16)
    codes = torch.zeros(M, 48, dtype=torch.uint8)
    scales = torch.zeros(2 * 2 * 512, dtype=torch.uint8)
    codes[129, 39] = 0x9F  # elements 78 (low nibble: -6) and 79 (high: -0.5)
    # row 129 is row 1 of band 1; block 4 is block 0 of tile 1
    scales[(1 * 2 + 1) * 512 + 1 * 16 + 0 * 4 + 0] = 0x38  # E4M3 1.0
    codes[70, 0] = 0x02
    scales[(70 % 32) * 16 + (70 // 32) * 4] = 0x40  # E4M3 2.0
    v = R.values(FP4Tensor(codes, scales, None, (M, K), "nv"))
    assert v[129, 78] == -6 and v[129, 79] == -0.5 and v[70, 0] == 2.0
    assert v.abs().sum() == 8.5
    assert not R.padding(FP4Tensor(codes, scales, None, (M, K), "nv")).any()


def test_conversion_refuses_what_it_does_not_know():
    import torch.nn as nn
    from flashvsr_sm89_ops_b200 import convert_linears_fp4
    model = nn.Sequential(nn.Linear(8, 8))
    with pytest.raises(ValueError, match="unknown parts"):
        convert_linears_fp4(model, parts=("ffn", "mlp"))
    with pytest.raises(ValueError, match="format"):
        convert_linears_fp4(model, fmt="int4")
    assert convert_linears_fp4(model) == 0 and type(model[0]) is nn.Linear


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_conversion_without_a_gpu_says_so_and_converts_nothing():
    import torch.nn as nn
    from flashvsr_sm89_ops_b200 import FP4Linear, integrate
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    with pytest.raises(ValueError, match="CUDA device"):
        FP4Linear(nn.Linear(64, 64))
    dit = W.WanDiT(num_layers=1, dim=256, num_heads=2, ffn_dim=512)
    with pytest.raises(ValueError, match="CUDA device"):
        integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False, fp4_parts=["ffn", "self"])
    assert all(type(m) is nn.Linear for n, m in dit.named_modules() if n.endswith((".q", ".o", ".ffn.0")))


@pytest.mark.parametrize("fused", ["0", "1"])
@pytest.mark.parametrize("part", ["ffn", "self", "cross"])
def test_enable_refuses_4_bits_for_a_part_that_is_fp8(part, fused, monkeypatch):
    from flashvsr_sm89_ops_b200 import integrate
    from flashvsr_sm89_ops_b200 import wan_video_dit as W
    monkeypatch.setenv("FS89_FP8_FFNFUSED", fused)
    dit = W.WanDiT(num_layers=1, dim=256, num_heads=2, ffn_dim=512).to(torch.bfloat16)
    assert integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False)["fp8_linears"] == 10
    before = {n: type(m) for n, m in dit.named_modules()}
    with pytest.raises(ValueError, match="already FP8"):
        integrate.enable(W.DiTPipe(dit), dit_module=W, verbose=False, fp4_parts=[part])
    assert {n: type(m) for n, m in dit.named_modules()} == before
