"""What the Python calls of the 8-bit and 16-bit experts refuse before anything is launched: expert matrices of another size,
type or stride than the call's."""
import pytest
import torch

from sfnx_amd import _abi, moe

N_IN, N_OUT, ROWS = 256, 256, 5
MAT8 = N_OUT * N_IN + 4 * 2 * 2
U8, F16, BF16, I32, F32 = torch.uint8, torch.float16, torch.bfloat16, torch.int32, torch.float32


def grouped(name, A, sa):
    """one of the grouped calls, right but for its experts; on the CPU, where the right call is refused for its tensors' place"""
    big = name.endswith("big")
    jobs = torch.zeros(2 * (_abi.BIGJOB_INTS if big else _abi.JOB_INTS), dtype=I32), torch.zeros(2, dtype=I32), 2
    q, s = torch.zeros((ROWS, N_IN), dtype=U8), torch.zeros((ROWS, 2))
    out = torch.zeros((ROWS, N_OUT))
    ff = N_OUT // 2
    if name == "gate_up":
        moe.moe_gate_up_swiglu_f8(A, sa, N_IN, ff, *jobs, q, s, torch.zeros((ROWS, ff)))
    elif name == "gate_up_big":
        moe.moe_gate_up_swiglu_f8_big(A, sa, N_IN, ff, *jobs, q, s, torch.zeros((ROWS, ff), dtype=U8), torch.zeros((ROWS, 1)))
    elif name == "down":
        moe.moe_down_f8(A, sa, N_IN, N_OUT, *jobs, torch.zeros((ROWS, N_IN)), out)
    elif name == "down_big":
        moe.moe_down_f8_big(A, sa, N_IN, N_OUT, *jobs, q, s, out)
    else:
        (moe.moe_mm_16_big if big else moe.moe_mm_16)(A, sa, N_IN, N_OUT, *jobs, torch.zeros((ROWS, N_IN), dtype=F16), out)


F8_CALLS = ["gate_up", "gate_up_big", "down", "down_big"]
MM_CALLS = ["mm", "mm_big"]


@pytest.mark.parametrize("name", F8_CALLS + MM_CALLS)
def test_experts_of_another_size(name):
    """experts that do not hold one matrix of the call's, a negative stride, an empty table"""
    f8 = name in F8_CALLS
    t, size, n = (U8, 1, MAT8) if f8 else (F16, 2, N_OUT * N_IN)
    sa = (n * size + 15) // 16 * 16
    with pytest.raises(ValueError, match="A: smaller than a matrix"):
        grouped(name, torch.zeros(n - 1, dtype=t), sa)
    with pytest.raises(ValueError, match="A: stride"):
        grouped(name, torch.zeros(n, dtype=t), -16)
    with pytest.raises(ValueError, match="A: an empty table"):
        grouped(name, torch.zeros(0, dtype=torch.int64), 0)
    for A, stride in ((torch.zeros(n, dtype=t), sa), (torch.zeros(1, dtype=torch.int64), 0)):
        with pytest.raises(ValueError, match="A: not on the current GPU"):   # nothing else is wrong
            grouped(name, A, stride)


@pytest.mark.parametrize("name", F8_CALLS + MM_CALLS)
def test_experts_of_another_type(name):
    """matrices of another type than the call's; matrices where their pointers are meant, and the other way about"""
    f8 = name in F8_CALLS
    t, other = (U8, F16) if f8 else (F16, BF16)
    sa = 4 * N_OUT * N_IN
    for wrong in (other, F32, torch.int64):
        with pytest.raises(ValueError, match="A: type" if f8 else "A: another type than x"):
            grouped(name, torch.zeros(8 * N_OUT * N_IN, dtype=wrong), sa)
    for wrong in (t, I32, F32):
        with pytest.raises(ValueError, match="A: type .* pointers"):
            grouped(name, torch.zeros(8 * N_OUT * N_IN, dtype=wrong), 0)


SHAPE = dict(H=1024, E=64, K=6, ff=256, shared=True)


def layer_on_the_cpu(cls, shape):
    L = cls.__new__(cls)   # the constructor asks for tensors on the GPU
    L.s, L.W = shape, torch.zeros((shape.E + 1, shape.H))
    return L


@pytest.mark.parametrize("cls, call", [(moe.MoeLayerF8, moe.layer_f8), (moe.MoeLayer16, moe.layer_16)])
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("other", [dict(H=2048), dict(E=32), dict(E=128), dict(K=4), dict(K=8), dict(ff=128), dict(shared=False)])
def test_layer_with_buffers_of_another_shape(cls, call, T, other):
    """the routing writes E + 1 logits and K picks a token, so smaller buffers would be written past their ends"""
    s = moe.LayerShape(**SHAPE)
    b = moe.FloatBuffers(moe.LayerShape(**{**SHAPE, **other}), T, device="cpu")
    x, y = torch.zeros((T, s.H)), torch.zeros((T, s.H))
    with pytest.raises(ValueError, match="b: made for another shape"):
        call(layer_on_the_cpu(cls, s), x, y, b)
    with pytest.raises(ValueError, match="x: not on the current GPU"):   # the right buffers: nothing else is wrong
        call(layer_on_the_cpu(cls, s), x, y, moe.FloatBuffers(moe.LayerShape(**SHAPE, wtype=moe.Q8_0), T, device="cpu"))


def test_rows_and_strides_past_the_library_s_integers():
    """the library takes rows and an output's stride as 32-bit integers: what does not fit is refused, not cut"""
    far, rows = 1 << 32, (1 << 32) + 5
    meta = dict(device="meta")   # sizes without memory
    with pytest.raises(ValueError, match="x: .* rows"):
        moe.quantize_f8(torch.empty((rows, 16), **meta), torch.empty((rows, 16), dtype=U8, **meta), torch.empty((rows, 1), **meta))
    W = torch.empty(MAT8 + 16, dtype=U8, **meta)
    q, s = torch.empty((2, N_IN), dtype=U8, **meta), torch.empty((2, 2), **meta)
    with pytest.raises(ValueError, match="out: .* apart"):
        moe.f8_gemm(W, N_OUT, N_IN, q, s, torch.empty_strided((2, N_OUT), (far + N_OUT, 1), **meta))
    q, s = torch.empty((rows, N_IN), dtype=U8, **meta), torch.empty((rows, 2), **meta)
    with pytest.raises(ValueError, match="xq: .* rows"):
        moe.f8_gemm(W, N_OUT, N_IN, q, s, torch.empty((rows, N_OUT), **meta))
    q, s = torch.empty((2, far + 16), dtype=U8, **meta), torch.empty((2, (far + 16 + 127) // 128), **meta)
    with pytest.raises(ValueError, match="x: .* columns"):
        moe.quantize_f8(torch.empty((2, far + 16), **meta), q, s)
    with pytest.raises(ValueError, match="W: .* columns"):
        moe.f8_gemm(torch.empty(far + (1 << 30), dtype=U8, **meta), 1, far + 16, q, s, torch.empty((2, 1), **meta))
    jobs = torch.empty(2 * _abi.JOB_INTS, dtype=I32, **meta), torch.empty(2, dtype=I32, **meta), 2
    with pytest.raises(ValueError, match="A: .* columns"):
        moe.moe_mm_16(torch.empty(4 * far, dtype=F16, **meta), 4 * far, N_IN, far + 8, *jobs, torch.empty((2, N_IN), dtype=F16, **meta),
                      torch.empty((2, far + 8), dtype=F16, **meta))


NO_JOBS = [
    lambda L, *n: L.sfnx_moe_gate_up_swiglu_f8(4096, 1 << 40, 128, 128, *n, None, None, None, None),
    lambda L, *n: L.sfnx_moe_down_f8(4096, 1 << 40, 128, 128, *n, None, 0, None, None),
    lambda L, *n: L.sfnx_moe_gate_up_swiglu_f8_big(4096, 1 << 40, 128, 128, *n, None, None, None, None, None),
    lambda L, *n: L.sfnx_moe_down_f8_big(4096, 1 << 40, 128, 128, *n, None, None, 0, None, None),
    lambda L, *n: L.sfnx_moe_mm_16(4096, 1 << 40, 1, 128, 128, *n, None, 0, None, None),
    lambda L, *n: L.sfnx_moe_mm_16_big(4096, 1 << 40, 30, 128, 128, *n, None, 0, None, None)]


@pytest.mark.parametrize("call", NO_JOBS)
def test_room_for_no_jobs(call):
    """a list with room for no jobs has no address: nothing to do, as in the calls of the quantized experts; with room for one
    it must have"""
    L = _abi.lib()
    # (without a GPU a call that has launched nothing still ends with the runtime's word that there is none)
    assert call(L, None, None, 0) == 0 or b"no ROCm-capable device" in L.sfnx_last_error()
    assert call(L, None, None, 1) == -1 and b"null pointer" in L.sfnx_last_error()
    assert call(L, None, None, -1) == -1 and b"njobs out of range" in L.sfnx_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("call", NO_JOBS)
def test_room_for_no_jobs_on_a_gpu(call):
    assert call(_abi.lib(), None, None, 0) == 0
