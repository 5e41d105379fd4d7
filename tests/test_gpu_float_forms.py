"""The 8- and 16-bit calls where they take another way through their kernels: each form of a dense product with short last
groups, the widest window's down, lists of more jobs than one pass holds, jobs without rows, matrices of gigabytes, values and
scales that are not finite."""
import numpy as np
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403
from tests.test_gpu_f8 import close, dev, gen, job_tensors
from tests.test_gpu_float_edges import CALLS, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("C, n_in, n_out", [(300, 528, 1301), (200, 1040, 1500), (600, 2064, 1600), (3073, 2064, 4101), (3137, 2064, 4101)])
def test_gemm_forms(C, n_in, n_out, t):
    """the widest form of some tens of rows with more than one step of K a block; last groups of one and of two jobs"""
    g = gen(C + n_in)
    blob, W = matrices(g, 1, n_out, n_in)
    q, s = quantize(torch.randn((C, n_in), generator=g))
    out = torch.full((C + 1, n_out), 77.0, dtype=OUT[t], device="cuda")
    moe.f8_gemm(dev(blob), n_out, n_in, dev(q), dev(s), out[:C])
    want, bound = product(dev(dequantize(q, s)), dev(W[0]), True)
    close(out[:C], want.cpu(), bound.cpu(), OUT[t], True)
    assert (out[C] == 77).all()


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("ff", [4096, 8176, 8192])
def test_down_window_wide(ff, t):
    """16 rows of h up to the widest the call takes (135 KB of LDS)"""
    T, E, K, H = 16, 3, 2, 200
    g, rng = gen(ff), np.random.default_rng(ff)
    blob, W = matrices(g, E + 1, H, ff)
    h = torch.randn((T * K + T, ff), generator=g)
    a, n, flat = jobs(picks(rng, T, E, K), E, True, 16, False)
    d, out = dev(blob), torch.full((T * K + T, H), 77.0, dtype=OUT[t], device="cuda")
    moe.moe_down_f8(d, d.stride(0), ff, H, *job_tensors(a, n), dev(h), out)
    want, bound, where = grouped(dequantize(*quantize(h)), W, flat, True)
    assert len(where) == T * K + T
    close(out[where.cuda()], want, bound, OUT[t])


def inputs(name, g, n, rows, cols, n_in):
    """(experts, their stride, their 64-bit values, activations as the call takes them, their 64-bit values)"""
    x = torch.randn((rows, n_in), generator=g)
    if name.startswith("mm"):
        W, x = (torch.randn((n, cols, n_in), generator=g) * 0.05).half(), x.half()
        return dev(W), 2 * cols * n_in, W.double(), dev(x), x.double()
    blob, W = matrices(g, n, cols, n_in)
    q, s = quantize(x)
    return dev(blob), blob.shape[1], W, dev(x) if name == "down" else (dev(q), dev(s)), dequantize(q, s)


def outputs(name, rows, n_out):
    ff = n_out // 2
    if name == "gate_up_big":
        return torch.full((rows, ff), 0x55, dtype=torch.uint8, device="cuda"), torch.full((rows, nb(ff)), 77.0, device="cuda")
    return torch.full((rows, ff if name == "gate_up" else n_out), 77.0, device="cuda")


def check_outputs(name, out, r, b, where, n_out):
    """rows `where` of out against the products r known to b; the others as outputs() made them"""
    ff = n_out // 2
    rest = torch.ones(len(out[0] if name == "gate_up_big" else out), dtype=torch.bool)
    rest[where] = False
    if name == "gate_up_big":
        want, bound = swiglu(r, b, ff)
        hq, hs = out[0].cpu(), out[1].cpu()
        sc = spread(hs[where].double(), ff)
        v = hq[where].view(F8).double() * sc
        assert ((v - want).abs() <= bound + (E4M3_HALF + 2 * ULP) * (want.abs() + bound) + E4M3_SUB * sc).all()
        assert (hq[rest] == 0x55).all() and (hs[rest] == 77).all()
        return
    close(out[where.cuda()], *(swiglu(r, b, ff) if name == "gate_up" else (r, b)), torch.float32)
    assert (out.cpu()[rest] == 77).all()


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("n_in, n_out", [(64, 96), (528, 10720)])
def test_jobs_without_rows(name, n_in, n_out):
    """jobs of no rows alone, first, last and inside the list and inside an expert's run of jobs: the others are as without them"""
    size = 64 if name.endswith("big") else 16
    g = gen(n_in)
    E, sizes = 4, [(0, 0), (0, 5), (1, 0), (1, size), (1, 0), (1, size), (1, 3), (2, 0), (2, 0), (2, 0), (2, 0), (2, 0), (3, 1), (3, 0)]
    rows = sum(n for _, n in sizes)
    A, sa, W, x, xv = inputs(name, g, E, rows, n_out, n_in)
    perm = torch.randperm(rows, generator=g).tolist()
    a, flat, at = np.full((len(sizes), 2 + 2 * size), -12345678, np.int32), [], 0
    for i, (e, n) in enumerate(sizes):
        a[i, 0], a[i, 1] = e, n
        a[i, 2:2 + n] = perm[at:at + n]
        a[i, 2 + size:2 + size + n] = range(at + 1, at + 1 + n)
        flat += [(e, perm[at + k], at + 1 + k) for k in range(n)]
        at += n
    out = outputs(name, rows + 2, n_out)
    call(name, A, sa, n_in, n_out, job_tensors(a, len(sizes)), x, out)
    check_outputs(name, out, *grouped(xv, W, flat, not name.startswith("mm")), n_out)
    empty = a[[0, 2, 4, 7, 8, 13]]
    out = outputs(name, rows + 2, n_out)
    call(name, A, sa, n_in, n_out, job_tensors(empty, len(empty)), x, out)
    for o in out if isinstance(out, tuple) else (out,):
        assert (o == (0x55 if o.dtype == torch.uint8 else 77)).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("per", [1, 5])
def test_more_jobs_than_a_list_holds(t, per):
    """over 2 * 8192 jobs of one or two rows, an expert's `per` of them together (5: taken as groups), runs that cross the lists'
    borders: each against its own product"""
    n_in, n_out, J = 64, 40, 2 * 8192 + 77
    g, rng = gen(per), np.random.default_rng(per)
    E = 600
    W = (torch.randn((E, n_out, n_in), generator=g) * 0.1).to(OUT[t])
    x = torch.randn((500, n_in), generator=g).to(OUT[t])
    n = rng.integers(1, 3, J)
    first = np.concatenate([[0], np.cumsum(n)[:-1]])
    e = np.arange(J) // per % E
    y = rng.integers(0, 500, (J, 2))
    a = np.full((J, 130), -12345678, np.int32)
    a[:, 0], a[:, 1] = e, n
    a[:, 2] = y[:, 0]
    a[:, 66] = first
    two = n == 2
    a[two, 3], a[two, 67] = y[two, 1], first[two] + 1
    P = int(n.sum())
    out = torch.full((P + 1, n_out), 77.0, device="cuda")
    moe.moe_mm_16_big(dev(W), 2 * n_out * n_in, n_in, n_out, *job_tensors(a, J), dev(x), out)
    er, yr = np.repeat(e, n), np.concatenate([y[i, :n[i]] for i in range(J)])
    xr, Wr = x.double()[yr], W.double()
    want, bound = torch.empty((P, n_out), dtype=torch.float64), torch.empty((P, n_out), dtype=torch.float64)
    for k in range(E):
        i = torch.from_numpy(np.flatnonzero(er == k))
        want[i], bound[i] = product(xr[i], Wr[k], False)
    close(out[:P], want, bound, torch.float32)
    assert (out[P] == 77).all()


def big_matrix(g, rows, cols, t):
    """a matrix whose rows repeat every 1024, times a power of two for each 128: (the 1024 rows in 64 bits, their factors)"""
    if t == "f8":
        v = (torch.randn((1024, cols), generator=g) * 100).clamp(-F8_MAX, F8_MAX).to(F8)
        s = 2.0 ** -torch.randint(6, 12, (nb(rows), 1), generator=g).float()
        m = torch.empty(rows * cols + 4 * nb(rows) * nb(cols), dtype=torch.uint8, device="cuda")
        m[: rows * cols].view(-1, 1024 * cols)[:] = dev(v.view(torch.uint8)).view(-1)
        m[rows * cols:] = dev(s.expand(-1, nb(cols)).contiguous()).view(-1).view(torch.uint8)
        return m, v.double(), s.double().repeat_interleave(128, 0)[:rows]
    v = (torch.randn((1024, cols), generator=g) * 0.05).to(OUT[t])
    m = dev(v).repeat(rows // 1024, 1)
    return m, v.double(), torch.ones((rows, 1), dtype=torch.float64)


def far_close(out, x, v, f, blocked, t):
    """the outputs of rows past 2 and 3 GiB and before, all of them"""
    want, bound = product(x, v, blocked)
    for r0 in range(0, len(f), 1 << 16):
        k = f[r0: r0 + (1 << 16), 0]
        n = len(k) // 1024
        close(out[:, r0: r0 + (1 << 16)], want.repeat(1, n) * k, bound.repeat(1, n) * k, t, True)


@pytest.mark.parametrize("C, t", [(3, "f32"), (20, "bf16"), (70, "f32"), (300, "bf16")])
def test_gemm_of_a_matrix_of_gigabytes(C, t):
    """3.2 GB of e4m3: a few rows, streamed, grouped"""
    rows, cols = 786432, 4096
    g = gen(C)
    m, v, f = big_matrix(g, rows, cols, "f8")
    q, s = quantize(torch.randn((C, cols), generator=g))
    out = torch.full((C, rows), 77.0, dtype=OUT[t], device="cuda")
    moe.f8_gemm(m, rows, cols, dev(q), dev(s), out)
    far_close(out, dequantize(q, s), v, f, True, OUT[t])


@pytest.mark.parametrize("name, n", [("mm", [5]), ("mm_big", [40]), ("mm_big", [64, 64, 64, 7])])
def test_expert_of_gigabytes(name, n):
    """a 16-bit expert of 3.2 GB: a window's job, one streamed, a group"""
    rows, cols = 393216, 4096
    g = gen(len(n))
    m, v, f = big_matrix(g, rows, cols, "f16")
    size, P = 64 if name == "mm_big" else 16, sum(n)
    x = torch.randn((P, cols), generator=g).half()
    a, at = np.zeros((len(n), 2 + 2 * size), np.int32), 0
    for i, k in enumerate(n):
        a[i, 1] = k
        a[i, 2:2 + k] = a[i, 2 + size:2 + size + k] = range(at, at + k)
        at += k
    out = torch.full((P, rows), 77.0, device="cuda")
    call(name, m, 2 * rows * cols, cols, rows, job_tensors(a, len(n)), dev(x), out)
    far_close(out, x.double(), v, f, False, torch.float32)


NOT_FINITE = [(4, 272, 150), (40, 272, 150), (70, 272, 150), (300, 528, 1301), (700, 1040, 2100), (1290, 2064, 4101), (3073, 2064, 4101)]


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("C, n_in, n_out", NOT_FINITE)
def test_gemm_not_finite(C, n_in, n_out, t):
    """a NaN activation, weight or scale reaches its row's or column's outputs, an infinite scale makes them infinite, and neither
    reaches others; in each form and type"""
    g = gen(C)
    blob, W = matrices(g, 1, n_out, n_in)
    q, s = quantize(torch.randn((C, n_in), generator=g))
    q.view(torch.uint8)[2, n_in - 1] = 0x7F
    blob[0, (n_out - 1) * n_in] = 0xFF                        # a NaN weight in the last row
    s[C - 1, 0] = float("nan")
    s[0, nb(n_in) - 1] = float("inf")
    out = torch.zeros((C, n_out), dtype=OUT[t], device="cuda")
    moe.f8_gemm(dev(blob), n_out, n_in, dev(q), dev(s), out)
    got = out.cpu()
    nan = torch.zeros((C, n_out), dtype=torch.bool)
    nan[2], nan[C - 1], nan[:, n_out - 1] = True, True, True
    s[0, nb(n_in) - 1] = 0
    s[C - 1, 0] = 0
    x = dequantize(q, s)
    last = q[:1, (nb(n_in) - 1) * BLK:].double() @ W[0][:, (nb(n_in) - 1) * BLK:].t()   # the sign of row 0's infinite block
    sure = last[0].abs() > 1e-3 * last[0].abs().mean()        # away from a sum of 0, whose product with infinity is NaN
    assert torch.equal(torch.isnan(got)[1:], nan[1:])
    inf = torch.where(last[0] > 0, float("inf"), float("-inf"))[: n_out - 1]
    assert (got[0, : n_out - 1].double() == inf)[sure[: n_out - 1]].all() and torch.isnan(got[0, n_out - 1])
    fine = [i for i in range(C) if i not in (0, 2, C - 1)]
    want, bound = product(dev(x[fine]), dev(W[0][: n_out - 1]), True)
    close(out[fine][:, : n_out - 1], want.cpu(), bound.cpu(), OUT[t], C > 16)


@pytest.mark.parametrize("where", ["first", "last"])
def test_gemm_infinite_weight_scale(where):
    """an infinite scale of a block of the matrix: its rows' outputs are infinite, the others finite"""
    n_in, n_out = 400, 300
    for C in (4, 70, 600):
        g = gen(C)
        blob, W = matrices(g, 1, n_out, n_in)
        b = 0 if where == "first" else nb(n_out) * nb(n_in) - 1
        blob[0, n_out * n_in + 4 * b: n_out * n_in + 4 * b + 4] = torch.tensor([float("inf")]).view(torch.uint8)
        q, s = quantize(torch.randn((C, n_in), generator=g))
        out = torch.zeros((C, n_out), device="cuda")
        moe.f8_gemm(dev(blob), n_out, n_in, dev(q), dev(s), out)
        rows, cols = (slice(0, 128), slice(0, 128)) if where == "first" else (slice(256, 300), slice(384, 400))
        v = blob[0, : n_out * n_in].view(F8).view(n_out, n_in).double()
        d = q[:, cols].double() @ v[rows, cols].t()
        got = out.cpu()
        sick = torch.zeros(n_out, dtype=torch.bool)
        sick[rows] = True
        assert torch.isfinite(got[:, ~sick]).all()
        sure = d.abs() > 1e-3 * d.abs().mean()
        assert (got[:, rows].double() == torch.where(d > 0, float("inf"), float("-inf")))[sure].all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_down_window_of_rows_not_finite(t):
    """h's rows of zeros, of small and large values, with infinities and NaN, quantized in the call: a value that is not finite
    makes its row's outputs NaN, and no other's"""
    T, E, K, H, ff = 10, 3, 2, 150, 272
    g, rng = gen(8), np.random.default_rng(8)
    blob, W = matrices(g, E + 1, H, ff)
    P = T * K + T
    h = torch.randn((P, ff), generator=g)
    h[0], h[1, ::2], h[2], h[3] = 0, -0.0, h[2] * 1e-20, h[3] * 1e30
    sick = {4: float("inf"), 9: float("nan"), 15: float("-inf"), 29: float("nan")}
    for r, v in sick.items():
        h[r, (37 * r) % ff] = v
    a, n, flat = jobs(picks(rng, T, E, K), E, True, 16, False)
    d, out = dev(blob), torch.full((P, H), 77.0, dtype=OUT[t], device="cuda")
    moe.moe_down_f8(d, d.stride(0), ff, H, *job_tensors(a, n), dev(h), out)
    bad = torch.zeros(P, dtype=torch.bool)
    bad[list(sick)] = True
    got = out.cpu()
    assert torch.isnan(got[bad]).all() and not torch.isnan(got[~bad]).any()
    h[bad] = 0
    want, bound, where = grouped(dequantize(*quantize(h)), W, flat, True)
    keep = ~bad[where]
    close(out[where[keep].cuda()], want[keep], bound[keep], OUT[t])
