"""The 8-bit floating-point operators (quantize_f8, f8_gemm, the grouped gate|up + SwiGLU and down) against plain forms in
64 bits, within the bounds of fp32 sums (tests/f8_util.py)."""
import random

import numpy as np
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(t):
    return t.cuda()


def job_tensors(a, n, cap_extra=2):
    """the job array on the GPU, with room for more jobs than there are (the count decides)"""
    pad = np.full((cap_extra, a.shape[1]), 0x3FFFFFFF, np.int32)
    return torch.from_numpy(np.concatenate([a, pad])).cuda().view(-1), torch.tensor([n, 0], dtype=torch.int32).cuda(), len(a) + cap_extra


def close(got, want, bound, t, many=False):
    """many: an 8-bit product of many rows"""
    got = got.double().cpu()
    if many and t != torch.float32:
        assert (got - want).norm() <= (COARSE_NORM + torch.finfo(t).eps / 2) * want.norm() + bound.norm()
        bound = bound * (COARSE / (131 * ULP))   # the sum of the terms' sizes is at most bound / (131 2^-23)
    lim = bound + half_step(t, want.abs() + bound)
    bad = (got - want).abs() > lim
    assert torch.isfinite(got).all()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst {float(((got - want).abs() / lim).max()):.3g} of its bound"


# ------------------------------------------------------------------------------------------------ quantizer
@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("rows, cols", [(1, 16), (1, 2048), (3, 144), (7, 128), (16, 2560), (65, 2000), (513, 4096)])
def test_quantize_equals_its_definition(rows, cols, t):
    x = torch.randn((rows, cols), generator=gen(rows + cols)) * torch.exp(3 * torch.randn((rows, 1), generator=gen(1)))
    x = x.to(OUT[t])
    q, s = torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty((rows, nb(cols)), device="cuda")
    moe.quantize_f8(dev(x), q, s)
    wq, ws = quantize(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq.view(torch.uint8))


def test_quantize_edge_values():
    """zeros, the smallest and largest values, blocks of one sign, ties of the rounding, infinities and NaN"""
    x = torch.zeros((12, 272))
    x[1] = 1e-45
    x[2] = torch.finfo(torch.float32).max * torch.where(torch.arange(272) % 2 == 0, 1.0, -1.0)
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    x[5] = float("-inf")
    x[6] = torch.linspace(-448, 448, 272)
    x[7, :16] = torch.tensor([448.0, 17, 19, 21, 23, 25, 27, 29, 31, 2 ** -10, 3 * 2 ** -10, 2 ** -9, 464, 1.0625, -1.0625, 1.1875])
    x[7, 12] = 448
    x[8] = 2.0 ** -126
    x[9] = -3.0
    x[10, 271] = -5e-3
    x[11] = torch.randn(272, generator=gen(3)) * 1e-38
    q, s = torch.empty((12, 272), dtype=torch.uint8, device="cuda"), torch.empty((12, 3), device="cuda")
    moe.quantize_f8(dev(x), q, s)
    wq, ws = quantize(x)
    assert torch.equal(s.cpu(), ws)
    got, want = q.cpu(), wq.view(torch.uint8)
    nan = torch.isnan(wq.float())
    assert torch.equal(got[~nan], want[~nan])
    assert ((got[nan] & 0x7F) == 0x7F).all()


def test_quantize_strided_rows_and_nothing():
    x = torch.randn((9, 512), generator=gen(4))
    big = dev(torch.cat([x, 1e9 * torch.ones_like(x)], 1))
    q, s = torch.empty((9, 512), dtype=torch.uint8, device="cuda"), torch.empty((9, 4), device="cuda")
    moe.quantize_f8(big[:, :512], q, s)
    wq, ws = quantize(x)
    assert torch.equal(q.cpu(), wq.view(torch.uint8)) and torch.equal(s.cpu(), ws)
    moe.quantize_f8(big[:0, :512], q[:0], s[:0])


# ------------------------------------------------------------------------------------------------ dense
GEMM = [(1, 16, 1), (1, 2048, 1024), (2, 128, 17), (5, 144, 130), (16, 2000, 257), (17, 256, 33), (63, 640, 300), (64, 1024, 256),
        (65, 1040, 513), (130, 2048, 129), (200, 4096, 640), (300, 48, 1301), (2000, 272, 4357)]


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("C, n_in, n_out", GEMM)
def test_gemm(C, n_in, n_out, t):
    g = gen(C + n_in + n_out)
    blob, W = matrices(g, 1, n_out, n_in)
    q, s = quantize(torch.randn((C, n_in), generator=g))
    out = torch.full((C + 1, n_out), 77.0, dtype=OUT[t], device="cuda")
    moe.f8_gemm(dev(blob), n_out, n_in, dev(q), dev(s), out[:C])
    want, bound = product(dequantize(q, s), W[0], True)
    close(out[:C], want, bound, OUT[t], C > 16)
    assert (out[C] == 77).all()


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("C, n_in, n_out", [(700, 2064, 2050), (1290, 2064, 4101), (3001, 2064, 4101)])
def test_gemm_large(C, n_in, n_out, t):
    """sizes that take each of the forms for many rows, short last blocks in every direction (the 64-bit products on the GPU)"""
    g = gen(C)
    blob, W = matrices(g, 1, n_out, n_in)
    q, s = quantize(torch.randn((C, n_in), generator=g))
    out = torch.full((C, n_out + 3), 77.0, dtype=OUT[t], device="cuda")
    moe.f8_gemm(dev(blob), n_out, n_in, dev(q), dev(s), out[:, :n_out])
    want, bound = product(dev(dequantize(q, s)), dev(W[0]), True)
    close(out[:, :n_out], want.cpu(), bound.cpu(), OUT[t], True)
    assert (out[:, n_out:] == 77).all()


@pytest.mark.parametrize("C", [3, 100])
@pytest.mark.parametrize("pad", [4, 5])
def test_gemm_strided_output(C, pad):
    g = gen(C)
    blob, W = matrices(g, 1, 200, 512)
    q, s = quantize(torch.randn((C, 512), generator=g))
    out = torch.full((C, 200 + pad), 77.0, device="cuda")
    moe.f8_gemm(dev(blob), 200, 512, dev(q), dev(s), out[:, :200])
    want, bound = product(dequantize(q, s), W[0], True)
    close(out[:, :200], want, bound, torch.float32)
    assert (out[:, 200:] == 77).all()


@pytest.mark.parametrize("C", [4, 70])
def test_gemm_nan_reaches_its_outputs_alone(C):
    """a NaN in an activation row reaches that row's outputs, one in a weight row that column's; infinite scales likewise"""
    g = gen(9)
    blob, W = matrices(g, 1, 150, 272)
    q, s = quantize(torch.randn((C, 272), generator=g))
    q.view(torch.uint8)[2, 271] = 0x7F
    blob[0, 149 * 272] = 0x7F
    out = torch.zeros((C, 150), device="cuda")
    moe.f8_gemm(dev(blob), 150, 272, dev(q), dev(s), out)
    nan = torch.isnan(out.cpu())
    want = torch.zeros_like(nan)
    want[2] = True
    want[:, 149] = True
    assert torch.equal(nan, want)


# ------------------------------------------------------------------------------------------------ grouped
SHAPES = [(1, 8, 3, 256, 128), (3, 5, 2, 144, 48), (7, 16, 4, 512, 144), (16, 64, 6, 1024, 512), (11, 4, 4, 640, 272)]


def gate_up_case(T, E, K, H, ff, shared, none, seed):
    g, rng = gen(seed), np.random.default_rng(seed)
    blob, W = matrices(g, E + 1, 2 * ff, H)
    q, s = quantize(torch.randn((T, H), generator=g))
    topi = picks(rng, T, E, K, none, hot=1)
    return blob, W, q, s, topi, T * K + (T if shared else 0)


@pytest.mark.parametrize("T, E, K, H, ff", SHAPES)
@pytest.mark.parametrize("table", [False, True])
def test_gate_up_window(T, E, K, H, ff, table):
    blob, W, q, s, topi, P = gate_up_case(T, E, K, H, ff, True, 0.1, T + H)
    a, n, flat = jobs(topi, E, True, 16, True, random.Random(1))
    jt, nt, cap = job_tensors(a, n)
    d = dev(blob)
    A, sa = (torch.tensor([d.data_ptr() + e * d.stride(0) for e in range(E + 1)], dtype=torch.int64).cuda(), 0) if table else (d, d.stride(0))
    h = torch.full((P, ff), 77.0, device="cuda")
    moe.moe_gate_up_swiglu_f8(A, sa, H, ff, jt, nt, cap, dev(q), dev(s), h)
    r, b, where = grouped(dequantize(q, s), W, flat, True)
    want, bound = swiglu(r, b, ff)
    close(h[where.cuda()], want, bound, torch.float32)
    rest = torch.ones(P, dtype=torch.bool)
    rest[where] = False
    assert (h.cpu()[rest] == 77).all()


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("T, E, K, H, ff", SHAPES)
def test_down_window(T, E, K, H, ff, t):
    """h is quantized as the quantizer defines it; the products are within their bound"""
    g, rng = gen(T + ff), np.random.default_rng(T)
    blob, W = matrices(g, E + 1, H, ff)
    P = T * K + T
    h = torch.randn((P, ff), generator=g) * torch.randn((P, ff), generator=g)
    h[0] = 0
    a, n, flat = jobs(picks(rng, T, E, K, 0.1, hot=1), E, True, 16, False)
    jt, nt, cap = job_tensors(a, n)
    d = dev(blob)
    out = torch.full((P, H), 77.0, dtype=OUT[t], device="cuda")
    moe.moe_down_f8(d, d.stride(0), ff, H, jt, nt, cap, dev(h), out)
    want, bound, where = grouped(dequantize(*quantize(h)), W, flat, True)
    close(out[where.cuda()], want, bound, OUT[t])
    rest = torch.ones(P, dtype=torch.bool)
    rest[where] = False
    assert (out.cpu()[rest] == 77).all()


BIG = [(1, 8, 3, 256, 128), (17, 5, 2, 144, 48), (65, 16, 4, 512, 144), (200, 12, 6, 1024, 512), (300, 4, 3, 640, 272), (70, 64, 8, 384, 384)]


@pytest.mark.parametrize("T, E, K, H, ff", BIG)
@pytest.mark.parametrize("table", [False, True])
def test_gate_up_prompt(T, E, K, H, ff, table):
    blob, W, q, s, topi, P = gate_up_case(T, E, K, H, ff, True, 0.1, T + H)
    a, n, flat = jobs(topi, E, True, 64, True, random.Random(2) if table else None)
    jt, nt, cap = job_tensors(a, n)
    d = dev(blob)
    A, sa = (torch.tensor([d.data_ptr() + e * d.stride(0) for e in range(E + 1)], dtype=torch.int64).cuda(), 0) if table else (d, d.stride(0))
    hq = torch.full((P, ff), 0x55, dtype=torch.uint8, device="cuda")
    hs = torch.full((P, nb(ff)), 77.0, device="cuda")
    moe.moe_gate_up_swiglu_f8_big(A, sa, H, ff, jt, nt, cap, dev(q), dev(s), hq, hs)
    r, b, where = grouped(dequantize(q, s), W, flat, True)
    want, bound = swiglu(r, b, ff)
    sc, hqc = hs.cpu()[where].double(), hq.cpu()[where].view(F8).double()
    # the scale: the block's largest |h| / 448, that value known to its bound, half a step each for 1 / 448 and the product
    amax = torch.stack([v.amax(1) for v in want.abs().split(BLK, 1)], 1)
    off = torch.stack([v.amax(1) for v in bound.split(BLK, 1)], 1)
    assert ((sc - amax / F8_MAX).abs() <= off / F8_MAX + ULP * sc).all()
    # the values: half a step of e4m3 beside h's own bound (the quotient's rounding in fp32 is far below it)
    lim = bound + (E4M3_HALF + 2 * ULP) * (want.abs() + bound) + E4M3_SUB * spread(sc, ff)
    assert torch.isfinite(hqc).all()
    assert ((hqc * spread(sc, ff) - want).abs() <= lim).all()
    # and they are the quantizer's: a value is another code only where h lies within its bound of a border
    w8 = (want / spread(sc, ff)).clamp(-F8_MAX, F8_MAX).float().to(F8).double()
    e = (bound / spread(sc, ff)) + 4 * ULP * F8_MAX
    lo, hi = ((want / spread(sc, ff) + d * e).clamp(-F8_MAX, F8_MAX).float().to(F8).double() for d in (-1, 1))
    assert ((hqc >= lo) & (hqc <= hi)).all()
    assert (hqc == w8).double().mean() > 0.99
    rest = torch.ones(P, dtype=torch.bool)
    rest[where] = False
    assert (hq.cpu()[rest] == 0x55).all() and (hs.cpu()[rest] == 77).all()


def test_gate_up_prompt_with_values_that_are_not_finite():
    """a NaN weight row and an overflowing activation row: NaN where they reach, the block's scale from its finite values"""
    T, E, K, H, ff = 70, 4, 2, 256, 192
    blob, W, q, s, topi, P = gate_up_case(T, E, K, H, ff, True, 0.0, 8)
    blob[2, 5 * H] = 0x7F            # expert 2's gate row 5
    s[9] = 3e38                      # token 9's products overflow, all of them or their products
    a, n, flat = jobs(topi, E, True, 64, True)
    jt, nt, cap = job_tensors(a, n)
    d = dev(blob)
    hq, hs = torch.zeros((P, ff), dtype=torch.uint8, device="cuda"), torch.zeros((P, 2), device="cuda")
    moe.moe_gate_up_swiglu_f8_big(d, d.stride(0), H, ff, jt, nt, cap, dev(q), dev(s), hq, hs)
    r, b, where = grouped(dequantize(q, s), W, flat, True)
    want, bound = swiglu(r, b, ff)
    token = {o: y for _, y, o in flat}
    sick = torch.tensor([token[int(o)] == 9 for o in where])
    expert = {o: e for e, _, o in flat}
    nan = torch.zeros((len(where), ff), dtype=torch.bool)
    nan[torch.tensor([expert[int(o)] == 2 for o in where]), 5] = True
    got, sc = hq.cpu()[where], hs.cpu()[where].double()
    fine = ~sick
    assert ((got[nan] & 0x7F) == 0x7F).all()
    assert torch.isfinite(sc).all()
    want = torch.where(nan, torch.zeros((), dtype=torch.float64), want)
    bound = torch.where(nan, torch.zeros((), dtype=torch.float64), bound)
    amax = torch.stack([v.amax(1) for v in want.abs().split(BLK, 1)], 1)
    off = torch.stack([v.amax(1) for v in bound.split(BLK, 1)], 1)
    assert ((sc - amax / F8_MAX).abs() <= off / F8_MAX + ULP * sc)[fine].all()
    v = got.view(F8).double()
    ok = (v * spread(sc, ff) - want).abs() <= bound + (E4M3_HALF + 2 * ULP) * (want.abs() + bound) + E4M3_SUB * spread(sc, ff)
    assert (ok | nan)[fine].all()
    # the overflowing row: what is finite in it is at most 448 of its scale, the rest NaN
    assert (torch.isnan(v[sick]) | (v[sick].abs() <= F8_MAX)).all()


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("T, E, K, H, ff", BIG)
def test_down_prompt(T, E, K, H, ff, t):
    g, rng = gen(T + ff), np.random.default_rng(T)
    H += 3   # an odd number of outputs
    blob, W = matrices(g, E + 1, H, ff)
    P = T * K + T
    q, s = quantize(torch.randn((P, ff), generator=g))
    a, n, flat = jobs(picks(rng, T, E, K, 0.1, hot=1), E, True, 64, False)
    jt, nt, cap = job_tensors(a, n)
    d = dev(blob)
    out = torch.full((P, H), 77.0, dtype=OUT[t], device="cuda")
    moe.moe_down_f8_big(d, d.stride(0), ff, H, jt, nt, cap, dev(q), dev(s), out)
    want, bound, where = grouped(dequantize(q, s), W, flat, True)
    close(out[where.cuda()], want, bound, OUT[t], True)
    rest = torch.ones(P, dtype=torch.bool)
    rest[where] = False
    assert (out.cpu()[rest] == 77).all()


# ------------------------------------------------------------------------------------------------ graphs, streams, repeats
def test_results_repeat_in_graphs_and_on_other_streams():
    """every call again, captured and replayed between eager work, and on another stream: the same bits"""
    T, E, K, H, ff = 40, 8, 3, 512, 256
    blob, W, q, s, topi, P = gate_up_case(T, E, K, H, ff, True, 0.0, 5)
    blob2, _ = matrices(gen(6), E + 1, H, ff)
    d, d2, qd, sd = dev(blob), dev(blob2), dev(q), dev(s)
    ju = job_tensors(*jobs(topi, E, True, 64, True)[:2])
    jd = job_tensors(*jobs(topi, E, True, 64, False)[:2])
    x = torch.randn((T, H), generator=gen(7)).cuda()
    hq, hs = torch.zeros((P, ff), dtype=torch.uint8, device="cuda"), torch.zeros((P, 2), device="cuda")
    out, dense = torch.zeros((P, H), device="cuda"), torch.zeros((T, 2 * ff), device="cuda")

    def work():
        moe.quantize_f8(x, qd, sd)
        moe.moe_gate_up_swiglu_f8_big(d, d.stride(0), H, ff, *ju, qd, sd, hq, hs)
        moe.moe_down_f8_big(d2, d2.stride(0), ff, H, *jd, hq, hs, out)
        moe.f8_gemm(d, 2 * ff, H, qd, sd, dense)

    work()
    torch.cuda.synchronize()
    want = [t.clone() for t in (hq, hs, out, dense)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (hq, hs, out, dense):
            t.zero_()
        work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((hq, hs, out, dense), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for i in range(3):
        for t in (hq, hs, out, dense):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((hq, hs, out, dense), want)), i
        x.mul_(1.0)
        torch.cuda.synchronize()
