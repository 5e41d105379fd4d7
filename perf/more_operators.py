"""Rows grouped by a number each carries, and what is done with them, as cases that can be timed and checked: tokens sorted by
expert and back with the router's weights applied, with its gradients, and low-rank adapters of many requests beside a
shared projection.

The operators (a pick or row whose id is outside [0, G) belongs to no group: its pos is -1, and it is left out everywhere):

  group         offsets[g] = the rows of groups before g;  pos[i] = offsets[ids[i]] + |{j < i: ids[j] = ids[i]}|;
                order[pos[i]] = i;  jobs: a group's rows 64 a job, in order, their row numbers pos (sorted) or i (in place)
  sort          xs[pos[t][k]] = x[t]
  sort_grad     dx[t] = sum_k dxs[pos[t][k]]
  combine       y[t] = sum_k w[t][k] ys[pos[t][k]]
  combine_grad  dys[pos[t][k]] = w[t][k] dy[t],  dw[t][k] = sum_h dy[t][h] ys[pos[t][k]][h]
  adapters      out[t] = base[t] + scale[a] B[a] (A[a] x[t]) for the row's adapter a, base[t] for a row without one

A case is a dict: "op", and the sizes that op takes.  Activations are N(0, 1) with a few large columns; experts are picked with
a Zipf skew over a random ranking, and `drop` of the picks belong to experts that live elsewhere.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
JOB = 64   # rows of a job


def _picked(op, T, K, E, H=0, type=None, out=None, skew=0.35, drop=0.0, in_place=False):
    c = {"op": op, "T": T, "K": K, "E": E, "skew": skew, "drop": drop}
    if op == "group":
        c["in_place"] = in_place
    return {**c, **({"H": H, "type": type} if H else {}), **({"out": out} if out else {})}


def _adapted(T, requests, n, rank, n_in, n_out, type, x, out, none=0.0):
    return {"op": "adapters", "T": T, "requests": requests, "n": n, "rank": rank, "n_in": n_in, "n_out": n_out, "type": type,
            "x": x, "out": out, "none": none}


def listed():
    return [
        # a decode window's picks: a launch and little else
        _picked("group", 16, 10, 512, in_place=True) | {"name": "group_16rows"},
        # a long prompt chunk's picks
        _picked("group", 4096, 10, 512) | {"name": "group_4096rows"},
        # a few sequences at once through a small model
        _picked("sort", 5, 6, 64, 1024, "f32") | {"name": "sort_5rows_f32"},
        # the usual prompt chunk
        _picked("sort", 2048, 10, 512, 2048, "bf16") | {"name": "sort_2048rows_bf16"},
        # a wider model whose experts are spread over four machines: three of four picks are another's
        _picked("sort_grad", 777, 8, 256, 2560, "f16", "f16", drop=0.75) | {"name": "sort_grad_777rows_f16"},
        # one token a step, its experts' rows in the router's type
        _picked("combine", 1, 10, 512, 2048, "f32", "f32") | {"name": "combine_1row"},
        # a long prompt chunk
        _picked("combine", 4096, 10, 512, 2048, "bf16", "bf16") | {"name": "combine_4096rows_bf16"},
        # a training step over few experts
        _picked("combine_grad", 4096, 6, 64, 2048, "bf16", "bf16") | {"name": "combine_grad_4096rows_bf16"},
        # one token a step beside the shared expert's gate|up, in the engine's 32-bit activations
        _adapted(1, 1, 64, 16, 2048, 1024, "bf16", "f32", "f32") | {"name": "adapters_1row"},
        # a window of the most rows, every row another request's
        _adapted(16, 16, 64, 16, 2048, 2048, "bf16", "bf16", "bf16") | {"name": "adapters_16rows"},
        # prompts of some requests in one chunk, a third of its rows without an adapter, an odd number of columns out
        _adapted(777, 9, 16, 8, 2560, 1301, "f16", "f16", "f32", none=0.33) | {"name": "adapters_777rows_odd"},
        # a long chunk of few requests beside a wide projection
        _adapted(4096, 4, 8, 64, 4096, 4096, "bf16", "bf16", "bf16") | {"name": "adapters_4096rows"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group", "sort", "sort_grad", "combine", "combine_grad", "combine_grad", "adapters", "adapters", "adapters"])
    if op == "adapters":
        T, n, t = _log_int(rng, 1, 4096), _log_int(rng, 1, 64), rng.choice(["f16", "bf16"])
        rank, n_in, n_out = rng.choice([8, 16, 16, 24, 32, 64, 128]), 8 * _log_int(rng, 16, 512), _log_int(rng, 64, 4096)
        x, out = rng.choice([t, t, "f32"]), rng.choice([t, t, "f32"])
        while max(T * rank * (n_in + n_out) / (4096 * 64 * 8192), T * (n_in * SIZE[x] + 2 * n_out * SIZE[out]) / (4096 * 4096 * 6)) > 1:
            T = T // 2 + 1   # no more than the largest listed
        return _adapted(T, rng.randint(1, min(T, 16)), n, rank, n_in, n_out, t, x, out,
                        none=rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)]))
    E, T = _log_int(rng, 2, 512), _log_int(rng, 1, 4096)
    K = rng.randint(1, min(12, E))
    skew, drop = round(rng.uniform(0.0, 1.0), 2), rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)])
    if op == "group":
        return _picked(op, T, K, E, skew=skew, drop=drop, in_place=rng.random() < 0.5)
    H = rng.choice([1024, 2048, 2048, 2560, 4096, rng.randint(65, 4096)])
    t, out = rng.choice(sorted(TYPES)), rng.choice(sorted(TYPES))
    while T * K * H * SIZE[t] > 4096 * 6 * 2048 * 2:   # no more than the largest listed
        T = T // 2 + 1
    return _picked(op, T, K, E, H, t, None if op == "sort" else out, skew, drop)


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _activations(g, rows, cols):
    """N(0, 1) about a few columns that run ten times as large, as a model's residual stream has them"""
    x = torch.randn((rows, cols), device=DEV, generator=g)
    big = torch.rand((cols,), device=DEV, generator=g) < 0.005
    return torch.where(big, 10 * x, x)


def _picks(g, T, E, K, skew, drop):
    """K distinct experts a token, drawn without replacement with weights rank^-skew over a random ranking, `drop` of them -1,
    and their weights, the softmax of K logits"""
    rank = torch.randperm(E, device=DEV, generator=g).float() + 1
    gumbel = -torch.log(-torch.log(torch.rand((T, E), device=DEV, generator=g).clamp(1e-7, 1 - 1e-7)))
    topi = torch.topk(gumbel - skew * torch.log(rank), K, dim=1).indices.int()
    topi[torch.rand((T, K), device=DEV, generator=g) < drop] = -1
    w = torch.exp(torch.randn((T, K), device=DEV, generator=g))
    return topi.contiguous(), w / w.sum(1, keepdim=True)


def _requests(g, case):
    """each row's adapter, -1 for none: a window's rows are one a request, a chunk's are its requests' prompts one after another"""
    T, r, n = case["T"], case["requests"], case["n"]
    ad = torch.randint(0, n, (r,), device=DEV, generator=g) if r > n else torch.randperm(n, device=DEV, generator=g)[:r]
    cut = torch.sort(torch.rand((r - 1,), device=DEV, generator=g) * T).values
    ids = ad[torch.searchsorted(cut, torch.arange(T, device=DEV).float())] if T > r else ad[torch.arange(T, device=DEV) % r]
    ids[torch.rand((T,), device=DEV, generator=g) < case["none"]] = -1
    return ids.int()


def _groups(ids, G):
    """(offsets, pos, order, valid rows first) of group, order filled up with -1"""
    n = ids.numel()
    key = torch.where((ids >= 0) & (ids < G), ids, torch.full_like(ids, G)).long()
    by = torch.argsort(key, stable=True)
    skey = key[by]
    offsets = torch.searchsorted(skey, torch.arange(G + 1, device=DEV)).int()
    at = torch.arange(n, device=DEV, dtype=torch.int32)
    in_group = skey < G
    pos = torch.empty_like(at)
    pos[by] = torch.where(in_group, at, torch.full_like(at, -1))
    return offsets, pos, torch.where(in_group, by.int(), torch.full_like(at, -1))


def _cap(n, G):
    return n // JOB + min(n, G) + 1


def _jobs(offsets, order, cap, in_place):
    """the library's job array [cap][2 + 2 * 64] int32 (a job: group, rows, their numbers twice) and the number of jobs"""
    n, G = order.numel(), offsets.numel() - 1
    off = offsets.long()
    nj = (off[1:] - off[:-1] + JOB - 1) // JOB
    first = torch.cumsum(nj, 0) - nj
    j = torch.arange(cap, device=DEV)
    last = torch.searchsorted(first + nj, j, right=True).clamp(max=G - 1)   # a job's group: the first that ends after it
    real = j < first[-1] + nj[-1]
    r0 = off[last] + (j - first[last]) * JOB
    rows = torch.where(real, (off[last + 1] - r0).clamp(max=JOB), 0)
    at = r0[:, None] + torch.arange(JOB, device=DEV)
    there = torch.arange(JOB, device=DEV) < rows[:, None]
    num = order[at.clamp(0, n - 1)] if in_place else at.int()
    num = torch.where(there, num, torch.zeros_like(num))
    head = torch.stack([torch.where(real, last, 0), rows], 1).int()
    count = torch.stack([first[-1] + nj[-1], torch.zeros_like(nj[0])]).int()
    return torch.cat([head, num, num], 1).view(-1), count


def prepare(case, seed):
    g = _gen(seed, 2)
    op, T, st = case["op"], case["T"], dict(case)
    if op == "adapters":
        n, R, ni, no, t = case["n"], case["rank"], case["n_in"], case["n_out"], TYPES[case["type"]]
        st["x"] = _activations(g, T, ni).to(TYPES[case["x"]])
        st["A"] = (torch.randn((n, R, ni), device=DEV, generator=g) / math.sqrt(ni)).to(t)
        st["B"] = (torch.randn((n, no, R), device=DEV, generator=g) / math.sqrt(R)).to(t)
        st["scale"] = 0.25 + torch.rand((n,), device=DEV, generator=g)
        st["base"] = torch.randn((T, no), device=DEV, generator=g).to(TYPES[case["out"]])
        st["out_t"] = torch.empty_like(st["base"])
        st["ids"] = _requests(g, case)
        listed_ids = torch.where(st["ids"] < 0, torch.full_like(st["ids"], n), st["ids"])   # rows without an adapter: group n
        offsets, _, order = _groups(listed_ids, n + 1)
        st["cap"] = _cap(T, n + 1)
        st["jobs"], st["njobs"] = _jobs(offsets, order, st["cap"], True)
        if own:
            from sfnx_amd import moe
            st["adapters"] = moe.Adapters(st["A"], st["B"], st["scale"])
        return st
    K, E = case["K"], case["E"]
    topi, st["w"] = _picks(g, T, E, K, case["skew"], case["drop"])
    n = T * K
    if op == "group":
        st["ids"], st["cap"] = topi.view(-1), _cap(n, E)
        if own:
            from sfnx_amd import moe
            st["groups"] = moe.RowGroups(n, E, in_place=st["in_place"])
        return st
    st["pos"] = _groups(topi.view(-1), E)[1].view(T, K)
    H, t = case["H"], TYPES[case["type"]]
    if op == "sort":
        st["x"] = _activations(g, T, H).to(t)
        st["xs"] = torch.zeros((n, H), dtype=t, device=DEV)
        return st
    out = TYPES[case["out"]]
    st["ys"] = _activations(g, n, H).to(t)
    if op == "combine_grad":
        st["dy"] = torch.randn((T, H), device=DEV, generator=g).to(out)
        st["dys"] = torch.zeros((n, H), dtype=t, device=DEV)
        st["dw"] = torch.empty((T, K), device=DEV)
    else:
        st["y"] = torch.empty((T, H), dtype=out, device=DEV)
    return st


# ---------------------------------------------------------------------------------------------------- the plain forms
def _grouped(offsets, pos, order, jobs, njobs):
    return {"offsets": offsets, "pos": pos, "order": order, "jobs": jobs, "njobs": njobs}


def _plain_adapters(st):
    """every adapter's products of every row, of which each row takes its own"""
    n, R = st["A"].shape[:2]
    T, x, ids = st["x"].shape[0], st["x"].float(), st["ids"].long()
    s = (x @ st["A"].float().view(n * R, -1).t()).view(T, n, R)
    mine = ids[:, None] == torch.arange(n, device=DEV)
    s = torch.where(mine[:, :, None], s * st["scale"][:, None], torch.zeros((), device=DEV)).view(T, n * R)
    B = st["B"].float().permute(0, 2, 1).reshape(n * R, -1)
    return {"out": (st["base"].float() + s @ B).to(st["out_t"].dtype)}


def _plain(st):
    op = st["op"]
    if op == "adapters":
        return _plain_adapters(st)
    if op == "group":
        offsets, pos, order = _groups(st["ids"], st["E"])
        jobs, njobs = _jobs(offsets, order, st["cap"], st["in_place"])
        return _grouped(offsets, pos, order, jobs, njobs)
    pos, T, K = st["pos"].long(), st["T"], st["K"]
    n = T * K
    there = (pos >= 0).view(T, K, 1)
    if op == "sort":
        xs = torch.zeros((n + 1, st["H"]), dtype=st["xs"].dtype, device=DEV)   # the row after the last takes the picks without one
        xs[torch.where(pos < 0, n, pos)] = st["x"][:, None]
        return {"xs": xs[:n]}
    if op == "combine_grad":
        dy, w = st["dy"].float()[:, None], st["w"][:, :, None]
        dys = torch.zeros((n + 1, st["H"]), dtype=st["dys"].dtype, device=DEV)
        dys[torch.where(pos < 0, n, pos)] = (w * dy).to(st["dys"].dtype)
        dw = torch.where(there, dy * st["ys"].float()[pos.clamp(min=0)], torch.zeros((), device=DEV)).sum(2)
        return {"dys": dys[:n], "dw": dw}
    rows = torch.where(there, st["ys"].float()[pos.clamp(min=0)], torch.zeros((), device=DEV))
    y = (rows if op == "sort_grad" else st["w"][:, :, None] * rows).sum(1)
    return {"y": y.to(st["y"].dtype)}


# ---------------------------------------------------------------------------------------------------- a pass
def run(st):
    if not own:
        return _plain(st)
    from sfnx_amd import moe
    op = st["op"]
    if op == "group":
        g = st["groups"]
        moe.group_rows(st["ids"], g)
        return _grouped(g.offsets, g.pos, g.order, g.jobs, g.njobs)
    if op == "sort":
        moe.moe_sort_rows(st["x"], st["pos"], st["xs"])
        return {"xs": st["xs"]}
    if op == "sort_grad":
        moe.moe_sort_rows_backward(st["ys"], st["pos"], st["y"])
        return {"y": st["y"]}
    if op == "combine":
        moe.moe_combine_sorted(st["ys"], st["w"], st["pos"], st["y"])
        return {"y": st["y"]}
    if op == "combine_grad":
        moe.moe_combine_sorted_backward(st["dy"], st["ys"], st["w"], st["pos"], st["dys"], st["dw"])
        return {"dys": st["dys"], "dw": st["dw"]}
    moe.adapter_mm(st["adapters"], st["jobs"], st["njobs"], st["cap"], st["x"], st["base"], st["out_t"])
    return {"out": st["out_t"]}


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    op, T = case["op"], case["T"]
    if op == "adapters":
        n_in, n_out, R = case["n_in"], case["n_out"], case["rank"]
        rows = T * (1 - case["none"])
        used = min(case["requests"], case["n"])
        return {"bytes": int(used * R * (n_in + n_out) * 2 + rows * n_in * SIZE[case["x"]] + 2 * T * n_out * SIZE[case["out"]] + 8 * T),
                "flops": int(2 * rows * R * (n_in + n_out) + T * n_out)}
    n = T * case["K"]
    valid = int(n * (1 - case["drop"]))
    if op == "group":   # ids in; offsets, pos, order and the jobs' rows out
        return {"bytes": 8 * n + 12 * valid + 4 * case["E"], "flops": n}
    H, b = case["H"], SIZE[case["type"]]
    if op == "sort":
        return {"bytes": T * H * b + valid * H * b + 4 * n, "flops": 0}
    o = SIZE[case["out"]]
    if op == "combine_grad":
        return {"bytes": T * H * o + 2 * valid * H * b + 12 * n, "flops": 3 * valid * H}
    return {"bytes": valid * H * b + T * H * o + (4 if op == "sort_grad" else 8) * n, "flops": (1 if op == "sort_grad" else 2) * valid * H}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op, T = case["op"], case["T"]
    if op == "adapters":
        out, x = st["base"].double(), st["x"].double()
        for a in sorted(set(st["ids"].tolist()) - {-1}):
            rows = (st["ids"] == a).nonzero()[:, 0]
            s = torch.mm(x[rows], st["A"][a].double().t().contiguous())
            out[rows] += st["scale"][a].double() * torch.mm(s, st["B"][a].double().t().contiguous())
        return {"out": out}
    if op == "group":   # whole numbers: from a list of each group's rows
        ids, E, n = st["ids"].tolist(), case["E"], T * case["K"]
        of = [[] for _ in range(E)]
        for i, e in enumerate(ids):
            if 0 <= e < E:
                of[e].append(i)
        order = [i for rows in of for i in rows]
        pos, offsets, jobs = [-1] * n, [0], []
        for p, i in enumerate(order):
            pos[i] = p
        for e, rows in enumerate(of):
            nums = rows if st["in_place"] else list(range(offsets[-1], offsets[-1] + len(rows)))
            for k in range(0, len(rows), JOB):
                part = nums[k:k + JOB]
                part = part + [0] * (JOB - len(part))
                jobs.append([e, min(JOB, len(rows) - k)] + part + part)
            offsets.append(offsets[-1] + len(rows))
        count = len(jobs)
        jobs += [[0] * (2 + 2 * JOB)] * (st["cap"] - count)
        as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        return _grouped(as_ints(offsets), as_ints(pos), as_ints(order + [-1] * (n - len(order))), as_ints(jobs).view(-1), as_ints([count, 0]))
    pos, K = st["pos"].long(), case["K"]
    if op == "sort":
        xs = torch.zeros((T * K, case["H"]), dtype=torch.float64, device=DEV)
        for k in range(K):
            t = (pos[:, k] >= 0).nonzero()[:, 0]
            xs[pos[t, k]] = st["x"][t].double()
        return {"xs": xs}
    if op == "combine_grad":
        dys = torch.zeros((T * K, case["H"]), dtype=torch.float64, device=DEV)
        dw = torch.zeros((T, K), dtype=torch.float64, device=DEV)
        for k in range(K):
            t = (pos[:, k] >= 0).nonzero()[:, 0]
            dy = st["dy"][t].double()
            dys[pos[t, k]] = st["w"][t, k].double()[:, None] * dy
            dw[t, k] = (dy * st["ys"][pos[t, k]].double()).sum(1)
        return {"dys": dys, "dw": dw}
    y = torch.zeros((T, case["H"]), dtype=torch.float64, device=DEV)
    for k in range(K):
        t = (pos[:, k] >= 0).nonzero()[:, 0]
        w = 1.0 if op == "sort_grad" else st["w"][t, k].double()[:, None]
        y[t] += w * st["ys"][pos[t, k]].double()
    return {"y": y}
