"""The grouped 8-bit and 16-bit calls at their edges: no jobs, offsets past 32 bits in experts, activations and outputs."""
import numpy as np
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403
from tests.test_gpu_f8 import close, dev, gen, job_tensors

pytestmark = pytest.mark.gpu

CALLS = ["gate_up", "gate_up_big", "down", "down_big", "mm", "mm_big"]


def call(name, A, sa, n_in, n_out, jobs, x, out):
    """one of CALLS: n_out the rows of a matrix; x and out what its kind takes ((q, s) for 8-bit rows)"""
    if name == "gate_up":
        moe.moe_gate_up_swiglu_f8(A, sa, n_in, n_out // 2, *jobs, *x, out)
    elif name == "gate_up_big":
        moe.moe_gate_up_swiglu_f8_big(A, sa, n_in, n_out // 2, *jobs, *x, *out)
    elif name == "down":
        moe.moe_down_f8(A, sa, n_in, n_out, *jobs, x, out)
    elif name == "down_big":
        moe.moe_down_f8_big(A, sa, n_in, n_out, *jobs, *x, out)
    else:
        (moe.moe_mm_16_big if name == "mm_big" else moe.moe_mm_16)(A, sa, n_in, n_out, *jobs, x, out)


@pytest.mark.parametrize("name", CALLS)
def test_no_jobs(name):
    """a list without jobs, and room for none: nothing is written"""
    n_in, n_out, rows = 256, 256, 5
    g, size = gen(3), 64 if name.endswith("big") else 16
    if name.startswith("mm"):
        A = torch.randn((2, n_out, n_in), generator=g).half().cuda()
        sa, x = 2 * n_out * n_in, torch.randn((rows, n_in), generator=g).half().cuda()
    else:
        A = matrices(g, 2, n_out, n_in)[0].cuda()
        sa, x = A.stride(0), torch.randn((rows, n_in), generator=g)
        x = dev(x) if name == "down" else tuple(map(dev, quantize(x)))
    ff = n_out // 2
    if name == "gate_up_big":
        out = torch.full((rows, ff), 0x55, dtype=torch.uint8, device="cuda"), torch.full((rows, nb(ff)), 77.0, device="cuda")
    else:
        out = torch.full((rows, ff if name == "gate_up" else n_out), 77.0, device="cuda")
    a = np.full((4, 2 + 2 * size), 0x3FFFFFFF, np.int32)
    jt, nt, cap = job_tensors(a, 0)
    call(name, A, sa, n_in, n_out, (jt, nt, cap), x, out)
    call(name, A, sa, n_in, n_out, (jt, nt, 0), x, out)
    for o in out if isinstance(out, tuple) else (out,):
        assert (o == (0x55 if o.dtype == torch.uint8 else 77)).all()


@pytest.mark.parametrize("name", CALLS)
def test_offsets_past_32_bits(name):
    """experts 2.5 GiB apart, activation rows and output rows past 4 GiB: as the same rows close together"""
    big, f8 = name.endswith("big"), not name.startswith("mm")
    n_in, n_out, E = 2048, 1024, 3
    esz = 1 if f8 else 2
    rows = (1 << 32) // (n_in * esz) + 1000          # the last rows start past 4 GiB
    out_rows = (1 << 32) // (4 * n_out) + 1000
    g, size = gen(5), 64 if big else 16
    R = 23 if big else 11
    ids = torch.tensor([rows - 1 - 7 * i if i % 2 else 3 * i for i in range(R)])
    outs = torch.tensor([out_rows - 1 - 5 * i if i % 3 else 2 * i for i in range(R)])
    half = R // 2
    a = np.full((2, 2 + 2 * size), -12345678, np.int32)
    flat = []
    for j, (e, span) in enumerate([(0, range(half)), (2, range(half, R))]):
        a[j, 0], a[j, 1] = e, len(span)
        a[j, 2:2 + len(span)] = ids[list(span)]
        a[j, 2 + size:2 + size + len(span)] = outs[list(span)]
        flat += [(e, i, i) for i in span]
    jobs_ = job_tensors(a, 2)
    stride = 5 << 29
    A = torch.empty(E * stride, dtype=torch.uint8, device="cuda")
    if f8:
        blob, W = matrices(g, E, n_out, n_in)
        raw = blob
    else:
        W = (torch.randn((E, n_out, n_in), generator=g) * 0.05).half()
        raw = W.reshape(E, -1).view(torch.uint8)
    for e in (0, 2):
        A[e * stride: e * stride + raw.shape[1]] = raw[e].cuda()
    x = torch.randn((R, n_in), generator=g)
    where = ids.cuda()
    if not f8:
        xb = x.half()
        X = torch.empty((rows, n_in), dtype=torch.float16, device="cuda")
        X[where] = xb.cuda()
        plain, arg, A = xb.double(), X, A.view(torch.float16)
    elif name == "down":
        X = torch.empty((rows, n_in), dtype=torch.float32, device="cuda")
        X[where] = x.cuda()
        plain, arg = dequantize(*quantize(x)), X
    else:
        q, s = quantize(x)
        Q = torch.empty((rows, n_in), dtype=torch.uint8, device="cuda")
        S = torch.empty((rows, nb(n_in)), device="cuda")
        Q[where], S[where] = q.view(torch.uint8).cuda(), s.cuda()
        plain, arg = dequantize(q, s), (Q, S)
    r, b, _ = grouped(plain, W.double(), flat, f8)
    if not name.startswith("gate_up"):
        out = torch.empty((out_rows, n_out), device="cuda")
        call(name, A, stride, n_in, n_out, jobs_, arg, out)
        close(out[outs.cuda()], r, b, torch.float32)
        return
    ff = n_out // 2
    want, bound = swiglu(r, b, ff)
    if not big:
        out = torch.empty((2 * out_rows, ff), device="cuda")
        call(name, A, stride, n_in, n_out, jobs_, arg, out)
        close(out[outs.cuda()], want, bound, torch.float32)
        return
    hq = torch.empty((8 * out_rows, ff), dtype=torch.uint8, device="cuda")
    hs = torch.empty((8 * out_rows, nb(ff)), device="cuda")
    far = torch.where(outs > out_rows // 2, outs + 7 * out_rows, outs)
    a[:, 2 + size:] = np.where(a[:, 2 + size:] > out_rows // 2, a[:, 2 + size:] + 7 * out_rows, a[:, 2 + size:])
    call(name, A, stride, n_in, n_out, job_tensors(a, 2), arg, (hq, hs))
    sc, v = hs[far.cuda()].cpu().double(), hq[far.cuda()].cpu().view(F8).double()
    lim = bound + (E4M3_HALF + 2 * ULP) * (want.abs() + bound) + E4M3_SUB * spread(sc, ff)
    assert ((v * spread(sc, ff) - want).abs() <= lim).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("C, n_in, n_out", [(777, 2000, 1301), (600, 1024, 1600), (513, 144, 1937), (1000, 2032, 1185), (66, 1152, 16001), (128, 528, 8192), (300, 144, 20000)])
def test_gemm_few_or_wide(C, n_in, n_out, t):
    """dense sizes of few row tiles and many column tiles and between, with rows and columns past their last tiles"""
    g = gen(C + n_out)
    blob, W = matrices(g, 1, n_out, n_in)
    q, s = quantize(torch.randn((C, n_in), generator=g))
    out = torch.full((C, n_out), 77.0, dtype=OUT[t], device="cuda")
    moe.f8_gemm(blob[0].cuda(), n_out, n_in, dev(q), dev(s), out)
    want, bound = product(dequantize(q, s), W[0], True)
    close(out, want, bound, OUT[t], many=True)
