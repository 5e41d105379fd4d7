"""adapter_mm on job lists that no grouping makes."""
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
