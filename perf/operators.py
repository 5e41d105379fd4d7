"""Matrix products of 8-bit and 16-bit floating-point weights, dense and grouped by expert, as cases that can be timed and
checked: what a model whose experts are kept in block-scaled 8-bit floating point (or not quantized at all) asks of an MoE
layer.

The operators, with e4m3 the 8-bit type of 4 exponent and 3 mantissa bits (no infinities, largest value 448) and a block 128
consecutive columns of a row (the last one may be shorter):

  quantize     s[r][b] = max(max |x[r][block b]| / 448, 2^-126),  q[r][k] = e4m3(x[r][k] / s[r][k / 128])
  gemm         out[c][n] = sum_k (xq[c][k] xs[c][k / 128]) (wq[n][k] ws[n / 128][k / 128])
  gate_up      of a job (an expert w, activation rows y, output rows o): g, u = the expert's gate and up rows times row y (as
               gemm), h[o] = u g / (1 + exp(-g)); decode windows get h in 32 bits, prompt chunks quantized again
  down         the expert's down rows times h[o]; a decode window's h is quantized first
  mm16         the expert's rows times row y, both in 16 bits

A case is a dict: "op", and the sizes that op takes.  Weights are N(0, 0.02), activations N(0, 1) with a few large columns;
experts are picked with a Zipf skew over a random ranking.  The shared expert is expert E, with every token a row of it.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
BLK, F8_MAX, S_MIN = 128, 448.0, 2.0 ** -126
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
JOB_ROWS = {"decode": 16, "prompt": 64}   # rows of a job in a decode window and in a prompt chunk


def _moe(op, path, T, H, E, K, ff, out=None, type=None, skew=0.35):
    c = {"op": op, "path": path, "T": T, "H": H, "E": E, "K": K, "ff": ff, "skew": skew}
    return {**c, **({"out": out} if out else {}), **({"type": type} if type else {})}


def listed():
    return [
        # one token's activations in front of a layer: a launch and little else
        {"op": "quantize", "rows": 1, "cols": 2048, "type": "f32", "name": "quantize_1row"},
        # a long prompt chunk's activations as a model that runs in bf16 hands them over
        {"op": "quantize", "rows": 4096, "cols": 4096, "type": "bf16", "name": "quantize_4096rows_bf16"},
        # the shared expert's gate|up for a single token
        {"op": "gemm", "rows": 1, "n_in": 2048, "n_out": 1024, "out": "f32", "name": "gemm_1row"},
        # the end of a prompt through a dense matrix of odd sizes: the last blocks of rows and columns are short
        {"op": "gemm", "rows": 777, "n_in": 2000, "n_out": 1301, "out": "f16", "name": "gemm_777rows_odd"},
        # a long prompt chunk through a wide dense matrix
        {"op": "gemm", "rows": 4096, "n_in": 4096, "n_out": 4096, "out": "bf16", "name": "gemm_4096rows"},
        # one token a step: ten experts and the shared one read their gate|up rows
        _moe("gate_up", "decode", 1, 2048, 512, 10, 512) | {"name": "gate_up_1row"},
        # a verify window of the most rows a window holds
        _moe("down", "decode", 16, 2048, 512, 10, 512, out="bf16") | {"name": "down_16rows"},
        # the usual prompt chunk
        _moe("gate_up", "prompt", 2048, 2048, 512, 10, 512) | {"name": "gate_up_2048rows"},
        # the end of a prompt in a wider model with an FF of five blocks, picks without skew
        _moe("down", "prompt", 777, 2560, 256, 8, 640, out="f32", skew=0.0) | {"name": "down_777rows"},
        # a few sequences at once through a small model whose experts are not quantized
        _moe("mm16", "decode", 5, 1024, 64, 6, 512, out="f32", type="f16") | {"name": "mm16_5rows_f16"},
        # a long chunk over few experts, hundreds of rows each: the matrix cores carry it
        _moe("mm16", "prompt", 4096, 2048, 64, 6, 1024, out="bf16", type="bf16") | {"name": "mm16_4096rows_bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "gate_up", "gate_up", "down", "down", "mm16", "mm16"])
    out = rng.choice(sorted(TYPES))
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 4096), "cols": 16 * _log_int(rng, 4, 256), "type": out}
    if op == "gemm":
        return {"op": op, "rows": _log_int(rng, 1, 4096), "n_in": 16 * _log_int(rng, 8, 256), "n_out": _log_int(rng, 64, 4096),
                "out": out}
    path = rng.choice(["decode", "prompt", "prompt"])
    H = rng.choice([1024, 2048, 2048, 2560, 4096])
    ff = rng.choice([512, 512, 640, 1024, 16 * rng.randint(20, 64)])
    E = rng.randint(8, max(8, min(512, 512 * 512 * 2048 // (H * ff * (2 if op == "mm16" else 1)))))
    K = rng.randint(1, min(12, E))
    T = _log_int(rng, 1, 16) if path == "decode" else _log_int(rng, 17, 4096)
    while path == "prompt" and T * (K + 1) * H * ff > 4096 * 7 * 2048 * 1024:   # no more work than the largest listed
        T = T // 2 + 1
    skew = round(rng.uniform(0.0, 1.0), 2)
    if op == "gate_up":
        return _moe(op, path, T, H, E, K, ff, skew=skew)
    if op == "down":   # a window's h is quantized inside: its outputs are those of a model that keeps 16 bits
        return _moe(op, path, T, H, E, K, ff, out=rng.choice(["bf16", "f16"]) if path == "decode" else out, skew=skew)
    t = rng.choice(["f16", "bf16"])
    return _moe(op, path, T, H, E, K, ff, out=rng.choice(["f32", t]), type=t, skew=skew)


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _up(n, m):
    return (n + m - 1) // m * m


def _nb(n):
    return (n + BLK - 1) // BLK


def _activations(g, rows, cols):
    """N(0, 1) about a few columns that run ten times as large, as a model's residual stream has them"""
    x = torch.randn((rows, cols), device=DEV, generator=g)
    big = torch.rand((cols,), device=DEV, generator=g) < 0.005
    return torch.where(big, 10 * x, x)


def _quantize_rows(x):
    """(q, s) of rows of x: a block's scale max |x| / 448, its values x / s"""
    rows, cols = x.shape
    nb = _nb(cols)
    v = torch.nn.functional.pad(x.float(), (0, nb * BLK - cols)).view(rows, nb, BLK)
    s = (v.abs().amax(2) / F8_MAX).clamp_min(S_MIN)
    q = (v / s[:, :, None]).clamp(-F8_MAX, F8_MAX).to(F8)
    return q.view(rows, nb * BLK)[:, :cols].contiguous(), s


def _f8_matrices(g, n, rows, cols):
    """n matrices as the library's 8-bit store has them, uint8 [n][stride]: e4m3 values [rows][cols], then the f32 scales of
    the 128 x 128 blocks, [ceil(rows / 128)][ceil(cols / 128)]"""
    rb, cb = _nb(rows), _nb(cols)
    out = torch.zeros((n, _up(rows * cols + 4 * rb * cb, 16)), dtype=torch.uint8, device=DEV)
    for e0 in range(0, n, 64):
        m = min(64, n - e0)
        w = torch.randn((m, rows, cols), device=DEV, generator=g) * 0.02
        v = torch.nn.functional.pad(w, (0, cb * BLK - cols, 0, rb * BLK - rows)).view(m, rb, BLK, cb, BLK)
        s = v.abs().amax((2, 4)) / F8_MAX
        q = (v / s[:, :, None, :, None]).clamp(-F8_MAX, F8_MAX).to(F8).view(m, rb * BLK, cb * BLK)[:, :rows, :cols]
        out[e0:e0 + m, : rows * cols] = q.reshape(m, -1).view(torch.uint8)
        out[e0:e0 + m, rows * cols: rows * cols + 4 * rb * cb] = s.reshape(m, -1).view(torch.uint8)
    return out


def _picks(g, T, E, K, skew):
    """K distinct experts a token, drawn without replacement with weights rank^-skew over a random ranking"""
    rank = torch.randperm(E, device=DEV, generator=g).float() + 1
    gumbel = -torch.log(-torch.log(torch.rand((T, E), device=DEV, generator=g).clamp(1e-7, 1 - 1e-7)))
    return torch.topk(gumbel - skew * torch.log(rank), K, dim=1).indices


def _jobs(topi, E, size, gather):
    """The jobs of a window or chunk of T tokens: expert e's pairs p = t K + k in pair order, `size` rows a job, then the
    shared expert's (E) with rows t -> T K + t.  gather: activation rows are tokens, else pairs.  Returns the library's job
    array [jobs][2 + 2 size] int32, their count, and the same as index lists (rows sel of the padded [jobs * size] rows, their
    activation and output rows, the jobs' experts)."""
    T, K = topi.shape
    P = T * K
    e = torch.cat([topi.reshape(-1), torch.full((T,), E, device=DEV)])
    pair = torch.arange(P + T, device=DEV)
    token = torch.cat([torch.arange(P, device=DEV) // K, torch.arange(T, device=DEV)])
    order = torch.argsort(e, stable=True)
    cnt = torch.bincount(e, minlength=E + 1)
    nj = (cnt + size - 1) // size
    e = e[order]
    pos = torch.arange(P + T, device=DEV) - (torch.cumsum(cnt, 0) - cnt)[e]
    job = (torch.cumsum(nj, 0) - nj)[e] + pos // size
    sel, out = job * size + pos % size, pair[order]
    y = token[order] if gather else out
    J = int(nj.sum())
    w = torch.repeat_interleave(torch.arange(E + 1, device=DEV), nj)
    arr = torch.zeros((J, 2 + 2 * size), dtype=torch.int32, device=DEV)
    arr[:, 0] = w
    arr[:, 1] = torch.bincount(job, minlength=J)
    arr[job, 2 + pos % size] = y.int()
    arr[job, 2 + size + pos % size] = out.int()
    return {"jobs": arr.view(-1), "njobs": torch.tensor([J, 0], dtype=torch.int32, device=DEV), "cap": J, "w": w, "sel": sel,
            "y": y, "o": out, "size": size}


def prepare(case, seed):
    g = _gen(seed, 1)
    op, st = case["op"], dict(case)
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        st["x"] = _activations(g, rows, cols).to(TYPES[case["type"]])
        st["q"] = torch.empty((rows, cols), dtype=torch.uint8, device=DEV)
        st["s"] = torch.empty((rows, _nb(cols)), device=DEV)
        return st
    if op == "gemm":
        rows, n_in, n_out = case["rows"], case["n_in"], case["n_out"]
        st["W"] = _f8_matrices(g, 1, n_out, n_in)
        q, st["xs"] = _quantize_rows(_activations(g, rows, n_in))
        st["xq"] = q.view(torch.uint8)
        st["out_t"] = torch.empty((rows, n_out), dtype=TYPES[case["out"]], device=DEV)
        return st
    T, H, E, K, ff = case["T"], case["H"], case["E"], case["K"], case["ff"]
    st.update(_jobs(_picks(g, T, E, K, case["skew"]), E, JOB_ROWS[case["path"]], op != "down"))
    P = T * K + T
    st["n_in"], st["n_out"] = (ff, H) if op == "down" else (H, 2 * ff)
    if op == "mm16":
        t = TYPES[case["type"]]
        st["W"] = torch.empty((E + 1, 2 * ff, H), dtype=t, device=DEV)
        for e0 in range(0, E + 1, 64):
            st["W"][e0:e0 + 64] = torch.randn(st["W"][e0:e0 + 64].shape, device=DEV, generator=g) * 0.02
        st["x"] = _activations(g, T, H).to(t)
    else:
        st["W"] = _f8_matrices(g, E + 1, st["n_out"], st["n_in"])
        if op == "gate_up":
            q, st["xs"] = _quantize_rows(_activations(g, T, H))
            st["xq"] = q.view(torch.uint8)
        else:   # h = silu(gate) up of products of unit scale
            a, b = (0.9 * torch.randn((P, ff), device=DEV, generator=g) for _ in range(2))
            h = torch.nn.functional.silu(a) * b
            if case["path"] == "decode":
                st["h"] = h
            else:
                q, st["hs"] = _quantize_rows(h)
                st["hq"] = q.view(torch.uint8)
    if op == "gate_up":
        if case["path"] == "decode":
            st["h"] = torch.empty((P, ff), device=DEV)
        else:
            st["hq"] = torch.empty((P, ff), dtype=torch.uint8, device=DEV)
            st["hs"] = torch.empty((P, _nb(ff)), device=DEV)
    else:
        st["out_t"] = torch.empty((P, st["n_out"]), dtype=TYPES[case["out"]], device=DEV)
    return st


# ---------------------------------------------------------------------------------------------------- the plain forms
def _spread(s, rows, cols):
    """a block's scale for each of its values"""
    return s.repeat_interleave(BLK, -1)[..., :cols] if rows is None else \
        s.repeat_interleave(BLK, -2)[..., :rows, :].repeat_interleave(BLK, -1)[..., :cols]


def _weights(blob, rows, cols):
    """matrices of the 8-bit store in 32 bits"""
    rb, cb, n = _nb(rows), _nb(cols), blob.shape[0]
    q = blob[:, : rows * cols].contiguous().view(F8).view(n, rows, cols).float()
    s = blob[:, rows * cols: rows * cols + 4 * rb * cb].contiguous().view(torch.float32).view(n, rb, cb)
    return q * _spread(s, rows, cols)


def _rows(q, s, cols):
    return q.view(F8).float() * _spread(s, None, cols)


def _job_products(st, W, x):
    """the jobs' rows of x times their experts' matrices W [jobs][n_out][n_in], as rows in the order of st["o"]"""
    n, size = W.shape[0], st["size"]
    xp = torch.zeros((n * size, x.shape[1]), device=DEV)
    xp[st["sel"]] = x[st["y"]]
    o = torch.bmm(xp.view(n, size, -1), W.transpose(1, 2).contiguous())
    return o.view(n * size, -1)[st["sel"]]


def _plain(st):
    op = st["op"]
    if op == "quantize":
        q, s = _quantize_rows(st["x"])
        return {"q": q, "s": s}
    if op == "gemm":
        W, x = _weights(st["W"], st["n_out"], st["n_in"])[0], _rows(st["xq"], st["xs"], st["n_in"])
        return {"out": (x @ W.t()).to(TYPES[st["out"]])}
    n_in, n_out = st["n_in"], st["n_out"]
    if op == "mm16":
        W, x = st["W"][st["w"]].float(), st["x"].float()
    else:
        W = _weights(st["W"][st["w"]], n_out, n_in)
        if op == "gate_up":
            x = _rows(st["xq"], st["xs"], n_in)
        elif st["path"] == "decode":
            q, s = _quantize_rows(st["h"])
            x = _rows(q, s, n_in)
        else:
            x = _rows(st["hq"], st["hs"], n_in)
    r = _job_products(st, W, x)
    if op != "gate_up":
        out = st["out_t"]
        out[st["o"]] = r.to(out.dtype)
        return {"out": out}
    ff = st["ff"]
    g, u = r[:, :ff], r[:, ff:]
    h = torch.empty((r.shape[0], ff), device=DEV)
    h[st["o"]] = u * g / (1 + torch.exp(-g))
    if st["path"] == "decode":
        return {"h": h}
    q, s = _quantize_rows(h)
    return {"hq": q, "hs": s}


# ---------------------------------------------------------------------------------------------------- a pass
def run(st):
    if not own:
        return _plain(st)
    from sfnx_amd import moe
    op = st["op"]
    if op == "quantize":
        moe.quantize_f8(st["x"], st["q"], st["s"])
        return {"q": st["q"].view(F8), "s": st["s"]}
    if op == "gemm":
        moe.f8_gemm(st["W"], st["n_out"], st["n_in"], st["xq"], st["xs"], st["out_t"])
        return {"out": st["out_t"]}
    W, sa, n_in, n_out, ff = st["W"], st["W"].stride(0) * st["W"].element_size(), st["n_in"], st["n_out"], st["ff"]
    jobs, njobs, cap, decode = st["jobs"], st["njobs"], st["cap"], st["path"] == "decode"
    if op == "gate_up":
        if decode:
            moe.moe_gate_up_swiglu_f8(W, sa, n_in, ff, jobs, njobs, cap, st["xq"], st["xs"], st["h"])
            return {"h": st["h"]}
        moe.moe_gate_up_swiglu_f8_big(W, sa, n_in, ff, jobs, njobs, cap, st["xq"], st["xs"], st["hq"], st["hs"])
        return {"hq": st["hq"].view(F8), "hs": st["hs"]}
    if op == "down":
        if decode:
            moe.moe_down_f8(W, sa, n_in, n_out, jobs, njobs, cap, st["h"], st["out_t"])
        else:
            moe.moe_down_f8_big(W, sa, n_in, n_out, jobs, njobs, cap, st["hq"], st["hs"], st["out_t"])
    elif decode:
        moe.moe_mm_16(W, sa, n_in, n_out, jobs, njobs, cap, st["x"], st["out_t"])
    else:
        moe.moe_mm_16_big(W, sa, n_in, n_out, jobs, njobs, cap, st["x"], st["out_t"])
    return {"out": st["out_t"]}


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["type"]] + 1) + 4 * case["rows"] * _nb(case["cols"]), "flops": 2 * n}
    f8 = lambda rows, cols: rows * cols + 4 * rows * _nb(cols)   # activation rows with their scales
    mat = lambda rows, cols: rows * cols + 4 * _nb(rows) * _nb(cols)
    if op == "gemm":
        r, ni, no = case["rows"], case["n_in"], case["n_out"]
        return {"bytes": f8(r, ni) + mat(no, ni) + r * no * size[case["out"]], "flops": 2 * r * ni * no}
    T, H, E, K, ff = case["T"], case["H"], case["E"], case["K"], case["ff"]
    p = [(e + 1) ** -case["skew"] for e in range(E)]
    picked = 1 + sum(1 - (1 - min(1.0, K * w / sum(p))) ** T for w in p)   # experts with rows, the shared one among them
    P = T * K + T
    flops = 2 * P * (H * ff if op == "down" else 2 * H * ff)
    if op == "mm16":
        return {"bytes": picked * 4 * ff * H + 2 * T * H + P * 2 * ff * size[case["out"]], "flops": flops}
    if op == "gate_up":
        return {"bytes": picked * mat(2 * ff, H) + f8(T, H) + (4 * P * ff if case["path"] == "decode" else f8(P, ff)), "flops": flops}
    return {"bytes": picked * mat(H, ff) + (4 * P * ff if case["path"] == "decode" else f8(P, ff)) + P * H * size[case["out"]],
            "flops": flops}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _block_of(n):
    return torch.arange(n, device=DEV) // BLK


def _exact_quantize(x):
    """the quantizer's definition: its scale is a 32-bit value, the quotient is exact up to its one rounding"""
    cols = x.shape[1]
    s = torch.stack([c.abs().amax(1) for c in x.float().split(BLK, 1)], 1) / F8_MAX
    s = torch.clamp(s, min=S_MIN)
    q = x.double() / s.double()[:, _block_of(cols)]
    return torch.clamp(q, -F8_MAX, F8_MAX).to(F8), s


def _exact_matrix(st, e):
    if st["op"] == "mm16":
        return st["W"][e].double()
    r, c = st["n_out"], st["n_in"]
    m = st["W"][e]
    s = m[r * c: r * c + 4 * _nb(r) * _nb(c)].clone().view(torch.float32).view(_nb(r), _nb(c)).double()
    return m[: r * c].view(F8).view(r, c).double() * s[_block_of(r)][:, _block_of(c)]


def _exact_rows(st):
    op = st["op"]
    if op == "mm16":
        return st["x"].double()
    if op == "down" and st["path"] == "decode":
        q, s = _exact_quantize(st["h"])
    else:
        q, s = (st["hq"], st["hs"]) if op == "down" else (st["xq"], st["xs"])
    q = q.view(F8).double()
    return q * s.double()[:, _block_of(q.shape[1])]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        q, s = _exact_quantize(st["x"])
        return {"q": q, "s": s.double()}
    x = _exact_rows(st)
    if case["op"] == "gemm":
        return {"out": x @ _exact_matrix(st, 0).t()}
    r = torch.empty((st["o"].numel(), st["n_out"]), dtype=torch.float64, device=DEV)
    e_of_row = st["w"][st["sel"] // st["size"]]
    for e in torch.unique(e_of_row).tolist():   # the rows are in the order of their experts, one expert's together
        i = (e_of_row == e).nonzero()[:, 0]
        r[st["o"][i]] = x[st["y"][i]] @ _exact_matrix(st, e).t()
    if case["op"] != "gate_up":
        return {"out": r}
    g, u = r[:, : st["ff"]], r[:, st["ff"]:]
    h = u * g * torch.sigmoid(g)
    if case["path"] == "decode":
        return {"h": h}
    s = torch.stack([c.abs().amax(1) for c in h.split(BLK, 1)], 1) / F8_MAX
    s = torch.clamp(s, min=S_MIN)
    q = torch.clamp(h / s[:, _block_of(st["ff"])], -F8_MAX, F8_MAX)
    return {"hq": q.to(torch.float32).to(F8), "hs": s}
