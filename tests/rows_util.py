"""Plain forms, in 64 bits or whole numbers, of grouped and sorted rows and of adapters, and the bounds of their errors (on the CPU).

A product of two numbers of at most 24 bits and its addition by fmaf is off by at most half a step of the partial sum, 2^-24 of
it; matrix instructions may round each addition by up to a step, 2^-23.  A sum of n terms in any order is then off by at most
n 2^-23 times the sum of the terms' sizes (n 2^-24 by fmaf).  A rounding to the output's type adds half a step: 2^-24, 2^-11, 2^-8 of the
value for f32, f16, bf16, and at least half of the type's smallest step (2^-150, 2^-25, 2^-134)."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SUB = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
STEP, FMA = 2.0 ** -23, 2.0 ** -24
JOB = 64


def rounding(v, bound, t):
    """the bound of a value's error after its rounding to type t, from the bound of what is rounded"""
    return bound + HALF[t] * (v.abs() + bound) + SUB[t]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, shape, t):
    return torch.randn(shape, generator=g).to(t)


def group(ids, G):
    """(offsets, pos, order, groups' rows as lists)"""
    of = [[] for _ in range(G)]
    for i, g in enumerate(ids):
        if 0 <= g < G:
            of[g].append(i)
    order = [i for rows in of for i in rows]
    pos = [-1] * len(ids)
    for p, i in enumerate(order):
        pos[i] = p
    offsets = np.concatenate([[0], np.cumsum([len(r) for r in of])]).astype(np.int64)
    return offsets, pos, order, of


def jobs(of, offsets, in_place):
    """[(group, row numbers)] 64 rows a job"""
    out = []
    for g, rows in enumerate(of):
        num = rows if in_place else list(range(int(offsets[g]), int(offsets[g]) + len(rows)))
        out += [(g, num[k:k + JOB]) for k in range(0, len(num), JOB)]
    return out


def picks(rng, T, K, E, drop):
    """pos [T][K] of random distinct picks, `drop` of them elsewhere; and the number of rows"""
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]) if T else np.zeros((0, K), int)
    ids[rng.random(ids.shape) < drop] = -1
    offsets, pos, _, _ = group(ids.reshape(-1).tolist(), E)
    return torch.tensor(pos, dtype=torch.int32).view(T, K), int(offsets[-1])


def combine(ys, w, pos):
    """(y, the sum of its terms' sizes)"""
    T, K = pos.shape
    y, s = torch.zeros((T, ys.shape[1]), dtype=torch.float64), torch.zeros((T, ys.shape[1]), dtype=torch.float64)
    for k in range(K):
        t = (pos[:, k] >= 0).nonzero()[:, 0]
        v = w[t, k].double()[:, None] * ys[pos[t, k].long()].double()
        y[t] += v
        s[t] += v.abs()
    return y, s


def combine_backward(dy, ys, w, pos):
    """(dys, dw, the sum of dw's terms' sizes); dys of the rows no pos names are 0"""
    T, K = pos.shape
    dys = torch.zeros(ys.shape, dtype=torch.float64)
    dw, s = torch.zeros((T, K), dtype=torch.float64), torch.zeros((T, K), dtype=torch.float64)
    for k in range(K):
        t = (pos[:, k] >= 0).nonzero()[:, 0]
        p, d = pos[t, k].long(), dy[t].double()
        dys[p] = w[t, k].double()[:, None] * d
        v = d * ys[p].double()
        dw[t, k], s[t, k] = v.sum(1), v.abs().sum(1)
    return dys, dw, s


def adapted(x, A, B, scale, ids, base, x_bits=0.0):
    """(out, the bound of its error before the last rounding) of rows with adapters ids (-1: none)"""
    n, R, ni = A.shape
    out = base.double().clone() if base is not None else torch.zeros((x.shape[0], B.shape[1]), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for a in sorted(set(ids.tolist()) - {-1}):
        t = (ids == a).nonzero()[:, 0]
        xa, Aa, Ba = x[t].double(), A[a].double(), B[a].double()
        f = 1.0 if scale is None else scale[a].double()
        s, se = xa @ Aa.t(), ni * STEP * (xa.abs() @ Aa.abs().t())
        s, se = s * f, (se + 2 * FMA * (s.abs() + se)) * abs(f)   # the scale's rounding
        bound[t] += se @ Ba.abs().t() + (R + 1) * STEP * (out[t].abs() + (s.abs() + se) @ Ba.abs().t())
        out[t] += s @ Ba.t()
    return out, bound


def within(got, want, bound, t):
    """got (type t) is want within bound before its rounding; where want is not finite got is the same"""
    got, want = got.cpu(), want.cpu()
    assert got.dtype == t and got.shape == want.shape
    fin = torch.isfinite(want)
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert torch.equal(g[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    over = (g - want).abs()[fin] - rounding(want, bound, t)[fin]
    assert over.numel() == 0 or over.max() <= 0, f"{(over > 0).sum()} of {over.numel()} values off by up to {over.max():.3g} more than allowed"
