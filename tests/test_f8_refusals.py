"""What the 8-bit and 16-bit operators refuse, on the host, before anything is launched."""
import pytest
import torch

from sfnx_amd import _abi, moe
from tests.f8_util import matrices, quantize

P = 4096   # a device pointer that is never dereferenced
BIG = 1 << 40


@pytest.mark.parametrize("call, msg", [
    (lambda L: L.sfnx_quantize_f8(2, P, 128, 1, 128, P, P, None), "x type must be"),
    (lambda L: L.sfnx_quantize_f8(0, P, 120, 1, 120, P, P, None), "cols must be"),
    (lambda L: L.sfnx_quantize_f8(0, P, 112, 1, 128, P, P, None), "ldx must be"),
    (lambda L: L.sfnx_quantize_f8(0, P, 136, 1, 128, P, P, None), "ldx must be"),
    (lambda L: L.sfnx_quantize_f8(0, P, 128, -1, 128, P, P, None), "rows out of range"),
    (lambda L: L.sfnx_quantize_f8(0, None, 128, 1, 128, P, P, None), "null pointer"),
    (lambda L: L.sfnx_quantize_f8(0, P + 4, 128, 1, 128, P, P, None), "16-byte aligned"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 120, P, P, 1, 0, P, 128, None), "multiple of 16"),
    (lambda L: L.sfnx_f8_gemm(P, 0, 128, P, P, 1, 0, P, 128, None), "n_out out of range"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P, P, 1, 0, P, 127, None), "ldo smaller"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P, P, 1, 2, P, 128, None), "out type"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P, P, -1, 0, P, 128, None), "C out of range"),
    (lambda L: L.sfnx_f8_gemm(None, 128, 128, P, P, 1, 0, P, 128, None), "null pointer"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P + 8, P, 1, 0, P, 128, None), "16-byte aligned"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P, P, 1, 0, P + 2, 128, None), "aligned to its type"),
    (lambda L: L.sfnx_f8_gemm(P, 1 << 20, 128, P, P, 1 << 24, 1, P, 1 << 20, None), "too many jobs"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, BIG, 128, 120, P, P, 1, P, P, P, None), "FF must be"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, 1024, 128, 128, P, P, 1, P, P, P, None), "stride smaller"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, BIG + 4, 128, 128, P, P, 1, P, P, P, None), "stride must be"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, BIG, 128, 128, None, P, 1, P, P, P, None), "null pointer"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, BIG, 128, 128, P, P, -1, P, P, P, None), "njobs out of range"),
    (lambda L: L.sfnx_moe_down_f8(P, BIG, 8208, 128, P, P, 1, P, 0, P, None), "at most 8192"),
    (lambda L: L.sfnx_moe_down_f8(P, BIG, 128, 128, P, P, 1, None, 0, P, None), "null pointer"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8_big(P, BIG, 128, 128, P, P, 1, P, P, None, P, None), "null pointer"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8_big(P, BIG, 128, 120, P, P, 1, P, P, P, P, None), "FF must be"),
    (lambda L: L.sfnx_moe_down_f8_big(P, BIG, 128, 128, P, P, 1, P, P, 5, P, None), "out type"),
    (lambda L: L.sfnx_moe_mm_16(P, BIG, 0, 128, 128, P, P, 1, P, 0, P, None), "expert type"),
    (lambda L: L.sfnx_moe_mm_16(P, BIG, 1, 132, 128, P, P, 1, P, 0, P, None), "multiple of 8"),
    (lambda L: L.sfnx_moe_mm_16(P, 1024, 1, 128, 128, P, P, 1, P, 0, P, None), "stride smaller"),
    (lambda L: L.sfnx_moe_mm_16_big(P, BIG + 8, 30, 128, 128, P, P, 1, P, 0, P, None), "stride must be"),
    (lambda L: L.sfnx_moe_mm_16_big(P, BIG, 30, 128, 128, P, P, 1, P + 2, 0, P, None), "16-byte aligned"),
])
def test_library_refuses(call, msg):
    L = _abi.lib()
    assert call(L) == -1
    assert msg in L.sfnx_last_error().decode()


@pytest.mark.parametrize("call, msg", [
    (lambda L: L.sfnx_quantize_f8(0, P, 128, 1 << 24, 128, P, P, None), "rows out of range"),
    (lambda L: L.sfnx_quantize_f8(0, P, 128, 1, 128, P, P + 2, None), "scales must be"),
    (lambda L: L.sfnx_f8_gemm(P, 128, 128, P, P + 2, 1, 0, P, 128, None), "scales must be"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8(P, BIG, 128, 128, P, P, 1, P, P + 1, P, None), "scales must be"),
    (lambda L: L.sfnx_moe_gate_up_swiglu_f8_big(P, BIG, 128, 128, P, P, 1, P, P, P, P + 2, None), "scales must be"),
    (lambda L: L.sfnx_moe_down_f8_big(P, BIG, 128, 128, P, P, 1, P, P + 2, 0, P, None), "scales must be"),
    (lambda L: L.sfnx_f8_gemm(P, 1 << 16, 1 << 16, P, P, 1, 0, P, 1 << 16, None), "smaller than 4 GiB"),
    (lambda L: L.sfnx_f8_gemm(P, 128, (1 << 20) + 16, P, P, 1, 0, P, 128, None), "at most 2^20"),
    (lambda L: L.sfnx_moe_down_f8_big(P, BIG, 1 << 16, 1 << 16, P, P, 1, P, P, 0, P, None), "smaller than 4 GiB"),
    (lambda L: L.sfnx_moe_mm_16(P, BIG, 1, 1 << 16, 1 << 15, P, P, 1, P, 0, P, None), "smaller than 4 GiB"),
    (lambda L: L.sfnx_moe_mm_16_big(P, BIG, 30, (1 << 20) + 8, 8, P, P, 1, P, 0, P, None), "at most 2^20"),
])
def test_library_refuses_sizes(call, msg):
    """sizes past what the kernels' 32-bit offsets and launches hold, and scales off their type's alignment"""
    L = _abi.lib()
    assert call(L) == -1
    assert msg in L.sfnx_last_error().decode()


def test_matrix_bytes():
    L = _abi.lib()
    assert L.sfnx_f8_matrix_bytes(1024, 2048) == 1024 * 2048 + 4 * 8 * 16
    assert L.sfnx_f8_matrix_bytes(129, 144) == 129 * 144 + 4 * 2 * 2
    assert L.sfnx_f8_matrix_bytes(1, 16) == 32      # 16 values and a scale, rounded up
    assert L.sfnx_f8_matrix_bytes(0, 16) == 0
    g = torch.Generator().manual_seed(1)
    assert matrices(g, 2, 130, 144)[0].shape[1] == L.sfnx_f8_matrix_bytes(130, 144)


def test_python_refuses():
    x, q, s = torch.zeros((2, 128)), torch.zeros((2, 128), dtype=torch.uint8), torch.zeros((2, 1))
    with pytest.raises(ValueError, match="x: type"):
        moe.quantize_f8(x.double(), q, s)
    with pytest.raises(ValueError, match="x: not on the current GPU"):
        moe.quantize_f8(x, q, s)
    with pytest.raises(ValueError, match="not contiguous"):
        moe.quantize_f8(x.t(), q, s)
    with pytest.raises(ValueError, match="W: type"):
        moe.f8_gemm(x, 2, 128, q, s, x)


def test_plain_quantizer_rounds_once():
    """the tests' own quantizer: within half a step everywhere, its scales the definition's"""
    x = torch.randn((50, 272), generator=torch.Generator().manual_seed(2))
    q, s = quantize(x)
    back = q.double() * s.double().repeat_interleave(128, 1)[:, :272]
    assert ((back - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * s.double().repeat_interleave(128, 1)[:, :272] * (1 + 1e-6)).all()
