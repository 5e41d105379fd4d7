"""adapter_mm on job lists that no grouping makes, and s = scale A x: that it keeps 24 bits in both forms, and the ends of its range."""
import pytest
import torch

from sfnx_amd import _abi, moe
from tests.rows_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu

KINDS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]   # of the adapters and of x


def listed(*jobs):
    """a job list of (adapter, [row or None for a row outside])"""
    a = torch.zeros((len(jobs), _abi.BIGJOB_INTS), dtype=torch.int32)
    outside = [-1, 2 ** 31 - 1, -2 ** 31, 5000]
    for j, (w, rows) in enumerate(jobs):
        num = torch.tensor([outside[i % 4] if r is None else r for i, r in enumerate(rows)], dtype=torch.int32)
        a[j, 0], a[j, 1] = w, len(rows)
        a[j, 2:2 + len(rows)] = num
        a[j, 2 + _abi.PF_JOB:2 + _abi.PF_JOB + len(rows)] = num
    return a.view(-1).cuda(), torch.tensor([len(jobs), 0], dtype=torch.int32).cuda(), len(jobs)


@pytest.mark.parametrize("t, x_t", KINDS)
@pytest.mark.parametrize("T, R", [(1, 8), (4, 16), (8, 32), (16, 24), (20, 16), (33, 8), (48, 32), (4, 40), (8, 64), (20, 128)])
def test_rows_behind_rows_outside(T, R, t, x_t):
    """a job may have more entries than x has rows: its last entries count, however many before them are outside"""
    n, n_in, n_out, t, x_t, g = 3, 264, 333, TYPES[t], TYPES[x_t], gen(T + R)
    A, B, x, base = rand(g, (n, R, n_in), t), rand(g, (n, n_out, R), t), rand(g, (T, n_in), x_t), rand(g, (T, n_out), torch.float32)
    for at in (16, 32, 47, 63):
        rows = list(range(T))
        first, second, rest = rows[:1], rows[1:3], rows[3:5]
        jobs = listed((1, [None] * at + first), (2, [None] * (at - len(second)) + second), (7, [None] * (at - 2) + rest))
        ids = torch.full((T,), -1, dtype=torch.int32)
        ids[first], ids[second] = 1, 2
        done = torch.zeros(T, dtype=torch.bool)
        done[first + second + rest] = True
        want, bound = adapted(x, A, B, None, ids, base)
        out = torch.full((T, n_out), 9.0).cuda()
        moe.adapter_mm(moe.Adapters(A.cuda(), B.cuda()), *jobs, x.cuda(), base.cuda(), out)
        within(out[done.cuda()], want[done], bound[done], torch.float32)
        assert torch.equal(out[rest].cpu(), base[rest]) and (out[~done.cuda()] == 9).all(), at
        there = base.cuda()
        moe.adapter_mm(moe.Adapters(A.cuda(), B.cuda()), *jobs, x.cuda(), there, there)
        assert torch.equal(there[done.cuda()], out[done.cuda()]) and torch.equal(there[~done.cuda()].cpu(), base[~done])


def in_order(T, n):
    ids = torch.arange(T, dtype=torch.int32) % n
    g = moe.RowGroups(T, n, in_place=True)
    moe.group_rows(ids.cuda(), g)
    return ids, g


def spread(T, R, n_in, bits, t, x_t):
    """x and A whose s = sum of 2^-b over bits, negative in odd ranks and times 2^(row % 3): every term comes from columns of its own, far apart, and is
    the product of two normal numbers.  All sums of terms are exact in 32 bits, in any order."""
    A, x = torch.zeros((2, R, n_in)), torch.zeros((T, n_in))
    for i, b in enumerate(bits):
        c = (i * (n_in - 1)) // max(1, len(bits) - 1)
        A[:, :, c] = 2.0 ** -(b // 2) * (1 - 2 * (torch.arange(R) % 2))
        x[:, c] = 2.0 ** -(b - b // 2) * 2.0 ** (torch.arange(T) % 3)
    s = sum(2.0 ** -b for b in bits)
    return x.to(x_t), A.to(t), s * 2.0 ** (torch.arange(T) % 3).double()[:, None] * (1 - 2 * (torch.arange(R) % 2)).double()


SHAPES = [(2, 8, 2048), (2, 32, 1024), (2, 40, 2048), (2, 64, 4096), (3, 128, 2048), (70, 64, 136), (1100, 8, 2048), (1100, 32, 256)]


@pytest.mark.parametrize("t, x_t", KINDS)
@pytest.mark.parametrize("T, R, n_in", SHAPES)
def test_s_keeps_24_bits(T, R, n_in, t, x_t):
    """s = 1 + 2^-9 + 2^-17 + 2^-23 needs all bits of 32, and comes out times a power of two; with s = 1 + 2^-9 + 2^-12 values of B of 11 bits
    give products of 23: everything is exact, in both forms"""
    n_out, t, x_t = 145, TYPES[t], TYPES[x_t]
    ids, g = in_order(T, 2)
    scale = torch.tensor([0.5, -4.0])
    k = torch.arange(n_out) % R
    for bits, b in (((0, 9, 17, 23), 1.0), ((0, 9, 12), 1 + 2.0 ** -10 if t == torch.float16 else 1 + 2.0 ** -7)):
        x, A, s = spread(T, R, n_in, bits, t, x_t)
        B = torch.zeros((2, n_out, R))
        B[0, torch.arange(n_out), k] = b * 2.0 ** (torch.arange(n_out) % 5 - 2)
        B[1] = -2 * B[0]
        out = torch.empty((T, n_out)).cuda()
        moe.adapter_mm(moe.Adapters(A.cuda(), B.to(t).cuda(), scale.cuda()), g.jobs, g.njobs, g.cap, x.cuda(), None, out)
        at = ids.long()
        want = scale[at].double()[:, None] * s[:, k] * B[at[:, None], torch.arange(n_out), k].double()
        assert torch.equal(out.cpu().double(), want)


@pytest.mark.parametrize("t, x_t", KINDS)
@pytest.mark.parametrize("T, R, n_in", SHAPES)
@pytest.mark.parametrize("power", [-118, -112, -106, 100])
def test_small_and_large_s(T, R, n_in, power, t, x_t):
    """the same where the scale takes s far down or up: its last bits are beyond 16-bit types' smallest values, and still count"""
    n_out, t, x_t = 145, TYPES[t], TYPES[x_t]
    ids, g = in_order(T, 2)
    scale = torch.tensor([2.0 ** power, -2.0 ** power])
    k = torch.arange(n_out) % R
    x, A, s = spread(T, R, n_in, (0, 9, 17, 23), t, x_t)
    B = torch.zeros((2, n_out, R))
    B[:, torch.arange(n_out), k] = 2.0 ** 15
    out = torch.empty((T, n_out)).cuda()
    moe.adapter_mm(moe.Adapters(A.cuda(), B.to(t).cuda(), scale.cuda()), g.jobs, g.njobs, g.cap, x.cuda(), None, out)
    want = scale[ids.long()].double()[:, None] * s[:, k] * 2.0 ** 15
    assert torch.equal(out.cpu().double(), want)


@pytest.mark.parametrize("T, R", [(2, 8), (2, 40), (3, 128), (1100, 16)])
def test_products_that_just_fit(T, R):
    """s = 5.19393e33 times f16's largest value, 65504, is 3.4022e38 and fits 32 bits; 65536 times s would not"""
    n_in, n_out = 256, 70
    ids, g = in_order(T, 1)
    A, B, x = torch.zeros((1, R, n_in)), torch.zeros((1, n_out, R)), torch.zeros((T, n_in))
    A[0, R - 1, 7], x[:, 7], B[0, :, R - 1] = 1.0, 5.19393e33, 65504.0
    assert float(x[0, 7]) * 65504 < torch.finfo(torch.float32).max < float(x[0, 7]) * 65536
    out = torch.empty((T, n_out)).cuda()
    moe.adapter_mm(moe.Adapters(A.half().cuda(), B.half().cuda()), g.jobs, g.njobs, g.cap, x.cuda(), None, out)
    want = torch.full((T, n_out), float(x[0, 7]) * 65504, dtype=torch.float64)
    within(out, want, 2 * STEP * want, torch.float32)   # a product as two, their sum


@pytest.mark.parametrize("t, x_t", KINDS)
@pytest.mark.parametrize("T, R", [(2, 8), (2, 40), (3, 128), (1100, 16)])
def test_smallest_values_of_16_bits(T, R, t, x_t):
    """x, A and B below their types' smallest normal numbers are not taken for zeros"""
    n_in, n_out, t, x_t = 256, 70, TYPES[t], TYPES[x_t]
    low, f = {torch.float16: (2.0 ** -23, 8.0), torch.bfloat16: (2.0 ** -130, 2.0 ** 40)}[t]
    ids, g = in_order(T, 1)
    for a, u, b in ((low, f, f), (f, low, f), (f, f, low)):
        A, x, B = torch.zeros((1, R, n_in)), torch.zeros((T, n_in)), torch.zeros((1, n_out, R))
        A[:, :, 9], x[:, 9], B[:, :, R - 1] = a, u, b
        out = torch.empty((T, n_out)).cuda()
        moe.adapter_mm(moe.Adapters(A.to(t).cuda(), B.to(t).cuda()), g.jobs, g.njobs, g.cap, x.to(x_t).cuda(), None, out)
        assert (out.cpu().double() == low * f * f).all(), (a, u, b)
