"""The 16-bit experts' products (moe_mm_16, moe_mm_16_big) against 64 bits, within the bounds of fp32 sums."""
import random

import numpy as np
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403
from tests.test_gpu_f8 import close, dev, gen, job_tensors

pytestmark = pytest.mark.gpu


def case(T, E, K, n_in, n_out, t, seed):
    g, rng = gen(seed), np.random.default_rng(seed)
    W = (torch.randn((E + 1, n_out, n_in), generator=g) * 0.05).to(OUT[t])
    x = torch.randn((T, n_in), generator=g).to(OUT[t])
    return W, x, picks(rng, T, E, K, 0.1, hot=1), T * K + T


def run(fn, size, T, E, K, n_in, n_out, t, out_t, table, shuffle):
    W, x, topi, P = case(T, E, K, n_in, n_out, t, T + n_in)
    a, n, flat = jobs(topi, E, True, size, True, shuffle)
    jt, nt, cap = job_tensors(a, n)
    pitch = (n_out * n_in + 7) // 8 * 8 + 8   # experts apart
    buf = torch.zeros((E + 1, pitch), dtype=OUT[t])
    buf[:, : n_out * n_in] = W.view(E + 1, -1)
    d = dev(buf)
    A, sa = (torch.tensor([d.data_ptr() + 2 * e * pitch for e in range(E + 1)], dtype=torch.int64).cuda(), 0) if table else (d, 2 * pitch)
    out = torch.full((P, n_out), 77.0, dtype=OUT[out_t], device="cuda")
    fn(A, sa, n_in, n_out, jt, nt, cap, dev(x), out)
    want, bound, where = grouped(x.double(), W.double(), flat, False)
    close(out[where.cuda()], want, bound, OUT[out_t])
    rest = torch.ones(P, dtype=torch.bool)
    rest[where] = False
    assert (out.cpu()[rest] == 77).all()


@pytest.mark.parametrize("t, out_t", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T, E, K, n_in, n_out", [(1, 8, 3, 256, 128), (3, 5, 2, 8, 1), (7, 16, 4, 200, 145), (16, 32, 6, 1024, 512), (11, 4, 4, 584, 272)])
def test_window(T, E, K, n_in, n_out, t, out_t):
    run(moe.moe_mm_16, 16, T, E, K, n_in, n_out, t, out_t, table=T == 7, shuffle=random.Random(3))


@pytest.mark.parametrize("t, out_t", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T, E, K, n_in, n_out", [(1, 8, 3, 256, 128), (17, 5, 2, 8, 1), (65, 16, 4, 200, 145), (200, 12, 6, 1024, 512), (300, 4, 3, 584, 272),
                                               (300, 4, 3, 72, 8190), (380, 4, 3, 200, 8190)])   # the last two: groups of 1, 2 and 4 jobs
def test_prompt(T, E, K, n_in, n_out, t, out_t):
    run(moe.moe_mm_16_big, 64, T, E, K, n_in, n_out, t, out_t, table=T == 65, shuffle=random.Random(4) if T == 200 else None)
