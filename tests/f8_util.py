"""Plain forms, in 64 bits, of the 8-bit and 16-bit products, and seeded inputs for their tests (on the CPU).

Tolerances are bounds: the 8-bit products of more than 16 rows into 16-bit outputs may keep 13 bits of the largest of 8
consecutive products (so each is off by at most 2^-13 of it), which bounds an output by 7 2^-13 of the sum of the terms' sizes,
and the whole result, whose errors do not add up in one direction, by 2^-13 sqrt(8 / 3) of its norm (a unit's error is at most
uniform over it, its rms 3^-1/2; the largest of 8 terms is at most the root of their square sum).  Every other product: a product of n terms summed in fp32 in whatever order is off by at most n 2^-23 times the sum of the
terms' sizes (one unit in the last place an addition, however it rounds; the 8-bit form sums 128 terms of a block and then
the blocks, with a rounding of the scales' product), and a final rounding to the output's type adds half a step."""
import numpy as np
import torch

from sfnx_amd import _abi

F8 = torch.float8_e4m3fn
BLK, F8_MAX, S_MIN = 128, 448.0, 2.0 ** -126
F8_INV = torch.tensor(1 / 448, dtype=torch.float32)
ULP = 2.0 ** -23
OUT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3_HALF, E4M3_SUB = 2.0 ** -4, 2.0 ** -10   # half a step: of a value, of the subnormals


def nb(n):
    return (n + BLK - 1) // BLK


def spread(s, cols):
    return s.repeat_interleave(BLK, -1)[..., :cols]


def quantize(x):
    """(q as float8, s) of rows of x (fp32 values): fp32 scales, the fp32 quotient rounded once"""
    x = x.float()
    rows, cols = x.shape
    v = torch.zeros((rows, nb(cols) * BLK))
    v[:, :cols] = x
    v = v.view(rows, nb(cols), BLK)
    fin = torch.isfinite(v)
    am = torch.where(fin, v.abs(), torch.zeros(())).amax(2)
    s = torch.clamp(am * F8_INV, min=S_MIN)
    t = torch.where(fin, torch.clamp(v / s[:, :, None], -F8_MAX, F8_MAX), torch.full((), float("nan")))
    return t.to(F8).view(rows, -1)[:, :cols].contiguous(), s


def dequantize(q, s):
    return q.double() * spread(s.double(), q.shape[1])


def matrices(g, n, rows, cols, std=0.05):
    """n matrices of the 8-bit store: (uint8 [n][stride], their values in 64 bits [n][rows][cols])"""
    stride = (rows * cols + 4 * nb(rows) * nb(cols) + 15) // 16 * 16
    blob = torch.zeros((n, stride), dtype=torch.uint8)
    q = (torch.randn((n, rows, cols), generator=g) * 100).clamp(-F8_MAX, F8_MAX).to(F8)
    s = (torch.rand((n, nb(rows), nb(cols)), generator=g) + 0.5) * std / 100
    blob[:, : rows * cols] = q.reshape(n, -1).view(torch.uint8)
    blob[:, rows * cols: rows * cols + 4 * nb(rows) * nb(cols)] = s.reshape(n, -1).view(torch.uint8)
    full = s.double().repeat_interleave(BLK, 1)[:, :rows].repeat_interleave(BLK, 2)[:, :, :cols]
    return blob, q.double() * full


def product(x, W, blocked, n=None):
    """(x W^T, its fp32 error bound) of 64-bit rows and matrix"""
    K = x.shape[1]
    terms = 128 + nb(K) + 3 if blocked else K
    return x @ W.t(), terms * ULP * (x.abs() @ W.abs().t())


COARSE, COARSE_NORM = 7 * 2.0 ** -13, 2.0 ** -13 * (8 / 3) ** 0.5


def half_step(t, v):
    """half a step of type t at the values v"""
    return torch.finfo(t).eps / 2 * v.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def swiglu(r, err, ff):
    """(h, bound) of gate|up rows r known to err: |silu'| <= 1.1; expf, the division and two products, 8 roundings"""
    g, u, eg, eu = r[:, :ff], r[:, ff:], err[:, :ff], err[:, ff:]
    si = g * torch.sigmoid(g)
    h = si * u
    return h, 1.1 * eg * (u.abs() + eu) + (si.abs() + 1.1 * eg) * eu + 8 * ULP * h.abs()


def jobs(topi, E, shared, size, gather, shuffle=None):
    """the routers' jobs of picks topi [T][K] (-1: none): (int32 array [jobs][2 + 2 size], njobs, [(expert, y, out)])"""
    T, K = topi.shape
    rows = [[] for _ in range(E + 1)]
    for p, e in enumerate(topi.reshape(-1).tolist()):
        if e >= 0:
            rows[e].append((p // K if gather else p, p))
    if shared:
        rows[E] = [(t if gather else T * K + t, T * K + t) for t in range(T)]
    js = [(e, rows[e][i:i + size]) for e in range(E + 1) for i in range(0, len(rows[e]), size)]
    if shuffle is not None:
        shuffle.shuffle(js)
    a = np.full((max(1, len(js)), 2 + 2 * size), -12345678, np.int32)   # entries past n are never to be used
    flat = []
    for i, (e, r) in enumerate(js):
        a[i, 0], a[i, 1] = e, len(r)
        a[i, 2:2 + len(r)] = [y for y, _ in r]
        a[i, 2 + size:2 + size + len(r)] = [o for _, o in r]
        flat += [(e, y, o) for y, o in r]
    return a, len(js), flat


def grouped(x, W, flat, blocked):
    """(outputs, bounds, output rows) of the jobs' rows in 64 bits"""
    outs, errs, where = [], [], []
    for e in sorted({f[0] for f in flat}):
        fs = [f for f in flat if f[0] == e]
        o, b = product(x[[f[1] for f in fs]], W[e], blocked)
        outs.append(o)
        errs.append(b)
        where += [f[2] for f in fs]
    return torch.cat(outs), torch.cat(errs), torch.tensor(where)


def picks(rng, T, E, K, none=0.0, hot=None):
    a = np.stack([rng.permutation(E)[:K] for _ in range(T)]) if T else np.zeros((0, K), int)
    if hot is not None:
        a[:, 0] = np.where((a[:, 1:] == hot).any(1), a[:, 0], hot)
    a[rng.random(a.shape) < none] = -1
    return a


__all__ = [n for n in dir() if not n.startswith("_")] + ["_abi"]
