"""group_rows, moe_sort_rows, moe_combine_sorted and their gradients against plain forms."""
import numpy as np
import pytest
import torch

from sfnx_amd import _abi, moe
from tests.rows_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def dev(t):
    return t.cuda()


# ---------------------------------------------------------------------------------------------------- group_rows
def check_groups(ids, g, what=""):
    """g's buffers against the plain form, what is left as it was included (a fresh g)"""
    offsets, pos, order, of = group(ids, g.n_groups)
    assert g.offsets.tolist() == offsets.tolist(), what
    assert g.pos[:len(ids)].tolist() == pos, what
    assert g.order[:len(order)].tolist() == order, what
    js = jobs(of, offsets, g.in_place)
    assert g.njobs.tolist() == [len(js), 0], what
    a = g.jobs.view(-1, 2 + 2 * JOB)[:len(js)].cpu().numpy()
    assert a[:, 0].tolist() == [w for w, _ in js] and a[:, 1].tolist() == [len(r) for _, r in js], what
    for row, (_, r) in zip(a, js):
        assert row[2:2 + len(r)].tolist() == r and row[2 + JOB:2 + JOB + len(r)].tolist() == r, what
        assert not row[2 + len(r):2 + JOB].any() and not row[2 + JOB + len(r):].any(), what
    return len(order), len(js)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n, G", [(0, 3), (1, 1), (1, 4096), (63, 1), (64, 2), (65, 1), (160, 512), (255, 7), (256, 256), (257, 300), (1000, 1),
                                  (3000, 33), (5000, 4096), (40960, 512)])
def test_group(n, G, in_place):
    rng = np.random.default_rng(n + G)
    ids = np.minimum((G * rng.random(n) ** 2).astype(np.int64), G - 1)   # the first groups are the largest
    g = moe.RowGroups(n, G, in_place)
    moe.group_rows(torch.tensor(ids, dtype=torch.int32).cuda(), g)
    m, nj = check_groups(ids.tolist(), g)
    assert m == n and (g.order[m:] == -1).all() and not g.jobs.view(-1, 130)[nj:].any()


@pytest.mark.parametrize("n, G", [(1, 2), (130, 5), (700, 64), (2500, 3)])
def test_group_ids_outside(n, G):
    """ids that name no group: below 0, G and above, the type's ends; all of them"""
    rng = np.random.default_rng(n)
    ids = rng.integers(0, G, n)
    ids[::2] = rng.choice([-1, -2 ** 31, G, G + 1, 2 ** 31 - 1], len(ids[::2]))
    g = moe.RowGroups(n, G)
    moe.group_rows(torch.tensor(ids, dtype=torch.int32).cuda(), g)
    m, nj = check_groups(ids.tolist(), g)
    assert (g.order[m:] == -1).all() and not g.jobs.view(-1, 130)[nj:].any()
    g = moe.RowGroups(n, G)
    moe.group_rows(torch.full((n,), -7, dtype=torch.int32).cuda(), g)
    assert g.offsets.tolist() == [0] * (G + 1) and g.njobs.tolist() == [0, 0] and (g.pos == -1).all() and (g.order == -1).all()


def test_group_fewer_rows_and_no_lists():
    """a g made for more rows keeps what lies behind; pos, order and jobs may be left out"""
    ids = torch.randint(0, 9, (300,), generator=gen(1), dtype=torch.int32)
    g = moe.RowGroups(1000, 9)
    g.pos.fill_(5)
    moe.group_rows(ids.cuda(), g)
    check_groups(ids.tolist(), g)
    assert (g.pos[300:] == 5).all() and (g.order[300:] == -1).all()
    off = torch.full((10,), -1, dtype=torch.int32).cuda()
    d = ids.cuda()
    _abi.check(_abi.lib().sfnx_group_rows(d.data_ptr(), 300, 9, off.data_ptr(), None, None, None, None, 0, 0, None, 0, moe._st()))
    assert torch.equal(off, g.offsets)


@pytest.mark.parametrize("n, G", [(4096, 64), (65536, 64), (65537, 64), (131072, 512), (131073, 4096), (300001, 1), (1 << 20, 700)])
def test_group_many(n, G):
    """both forms' ends, chunks of several rounds; against a stable sort"""
    ids = torch.randint(-1, G, (n,), generator=gen(n), dtype=torch.int32)
    ids[n // 3:n // 3 + 3000] = G - 1
    g = moe.RowGroups(n, G, in_place=True)
    moe.group_rows(ids.cuda(), g)
    by = torch.argsort(torch.where(ids < 0, G, ids), stable=True)
    cnt = torch.bincount(ids[ids >= 0], minlength=G)
    m = int(cnt.sum())
    assert torch.equal(g.offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(cnt, 0)]).int())
    assert torch.equal(g.order.cpu()[:m], by[:m].int()) and (g.order[m:] == -1).all()
    pos = torch.full((n,), -1, dtype=torch.int32)
    pos[by[:m]] = torch.arange(m, dtype=torch.int32)
    assert torch.equal(g.pos.cpu(), pos)
    a, nj = g.jobs.cpu().view(-1, 2 + 2 * JOB), int(g.njobs[0])
    assert nj == int(((cnt + JOB - 1) // JOB).sum()) and int(a[:nj, 1].sum()) == m and not a[nj:].any()
    there = torch.arange(JOB) < a[:nj, 1:2]
    assert torch.equal(a[:nj, 2:2 + JOB][there], by[:m].int()) and torch.equal(a[:nj, 2 + JOB:][there], by[:m].int())
    assert torch.equal(torch.repeat_interleave(a[:nj, 0], a[:nj, 1]), ids[by[:m]])


def test_group_fewer_rows_in_chunks_of_another_size():
    """131072 rows take 128 chunks, one row more 65: a g for the latter serves the former"""
    g, ids = moe.RowGroups(131073, 40), torch.randint(0, 40, (131072,), generator=gen(4), dtype=torch.int32)
    moe.group_rows(ids.cuda(), g)
    by = torch.argsort(ids, stable=True).int()
    assert torch.equal(g.order[:131072].cpu(), by) and int(g.order[131072]) == -1


def test_group_in_a_graph():
    """captured and replayed on other ids, with eager calls between"""
    ids = torch.zeros(3000, dtype=torch.int32).cuda()
    g = moe.RowGroups(3000, 40)
    moe.group_rows(ids, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.group_rows(ids, g)
    for k in range(4):
        now = torch.randint(-1, 40, (3000,), generator=gen(k), dtype=torch.int32)
        ids.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        other = moe.RowGroups(3000, 40)
        moe.group_rows(ids, other)
        assert torch.equal(g.pos, other.pos) and torch.equal(g.offsets, other.offsets)
        offsets, pos, order, of = group(now.tolist(), 40)
        assert g.pos.tolist() == pos and g.njobs[0].item() == len(jobs(of, offsets, False))


# ---------------------------------------------------------------------------------------------------- sort
SORT_SIZES = [(1, 1, 1), (1, 10, 2048), (5, 6, 1024), (3, 17, 65), (33, 2, 1), (70, 4, 4099), (9, 64, 130), (100, 3, 2560)]   # T, K, H


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16, torch.uint8, torch.int32, torch.float8_e4m3fn])
@pytest.mark.parametrize("T, K, H", SORT_SIZES)
def test_sort(T, K, H, t):
    rng = np.random.default_rng(T * K + H)
    pos, rows = picks(rng, T, K, max(K, 70), 0.3 if T % 2 else 0.0)
    x = torch.randint(0, 256, (T, H * t.itemsize), generator=gen(T), dtype=torch.uint8).view(t)
    xs = torch.full((rows + 3, H * t.itemsize), 0x5A, dtype=torch.uint8).cuda().view(t)
    moe.moe_sort_rows(x.cuda(), pos.cuda(), xs)
    want = torch.full((rows + 3, H * t.itemsize), 0x5A, dtype=torch.uint8)
    for k in range(K):
        m = (pos[:, k] >= 0).nonzero()[:, 0]
        want[pos[m, k].long()] = x.view(torch.uint8)[m]
    assert torch.equal(xs.view(torch.uint8).cpu(), want)


@pytest.mark.parametrize("H, pad, off", [(64, 8, 0), (64, 3, 0), (64, 8, 1), (63, 1, 0), (2560, 16, 8)])
def test_sort_strided(H, pad, off):
    """rows apart, rows off their alignment, a flat pos, and rows of xs that pos names beyond its end"""
    T, K = 20, 4
    pos, rows = picks(np.random.default_rng(3), T, K, 12, 0.2)
    x = rand(gen(1), (T, H + pad), torch.bfloat16)
    xs = torch.full((rows - 5, H + pad), 7.0, dtype=torch.bfloat16).cuda()
    moe.moe_sort_rows(x.cuda()[:, off:off + H], pos.view(-1).cuda(), xs[:, off:off + H])
    want = torch.full((rows - 5, H + pad), 7.0, dtype=torch.bfloat16)
    for t in range(T):
        for k in range(K):
            p = int(pos[t, k])
            if 0 <= p < rows - 5:
                want[p, off:off + H] = x[t, off:off + H]
    assert torch.equal(xs.cpu(), want)


# ---------------------------------------------------------------------------------------------------- combine and the gradients
def data(T, K, H, a, b, seed, drop):
    """pos, ys (type a; rows no pos names are NaN), w, a tensor like y (type b)"""
    rng, g = np.random.default_rng(seed), gen(seed)
    pos, rows = picks(rng, T, K, max(K, 16), drop)
    ys = rand(g, (rows + 2, H), a)
    ys[rows:] = float("nan")
    return pos, rows, ys, torch.rand((T, K), generator=g), rand(g, (T, H), b)


PAIRS = [(a, b) for a in TYPES for b in TYPES]


@pytest.mark.parametrize("a, b", PAIRS)
@pytest.mark.parametrize("T, K, H", SORT_SIZES)
def test_combine_and_gradients(T, K, H, a, b):
    a, b = TYPES[a], TYPES[b]
    pos, rows, ys, w, dy = data(T, K, H, a, b, T + H, 0.4 if T % 2 else 0.0)
    y = torch.full((T, H), 9.0, dtype=b).cuda()
    moe.moe_combine_sorted(ys.cuda(), w.cuda(), pos.cuda(), y)
    want, size = combine(ys, w, pos)
    within(y, want, K * FMA * size, b)
    one = torch.ones_like(w)
    moe.moe_sort_rows_backward(ys.cuda(), pos.cuda(), y)
    want, size = combine(ys, one, pos)
    within(y, want, K * FMA * size, b)
    dys, dw = torch.full_like(ys, 9.0).cuda(), torch.full((T, K), 9.0).cuda()
    moe.moe_combine_sorted_backward(dy.cuda(), ys.cuda(), w.cuda(), pos.cuda(), dys, dw)
    wys, ww, size = combine_backward(dy, ys, w, pos)
    within(dys[:rows], wys[:rows], FMA * wys[:rows].abs(), a)
    assert (dys[rows:] == 9).all()
    within(dw, ww, H * FMA * size, torch.float32)


@pytest.mark.parametrize("a, b", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("H, pad, off", [(64, 8, 0), (64, 3, 0), (128, 8, 1), (63, 1, 0)])
def test_strided(H, pad, off, a, b):
    a, b, T, K = TYPES[a], TYPES[b], 11, 5
    pos, rows, ys, w, dy = data(T, K, H + pad, a, b, 5, 0.2)
    cut = lambda t: t[:, off:off + H]
    y = torch.full((T, H + pad), 9.0, dtype=b).cuda()
    moe.moe_combine_sorted(cut(ys.cuda()), w.cuda(), pos.cuda(), cut(y))
    want, size = combine(cut(ys), w, pos)
    within(cut(y), want, K * FMA * size, b)
    assert (y[:, :off] == 9).all() and (y[:, off + H:] == 9).all()
    dys, dw = torch.full_like(ys, 9.0).cuda(), torch.empty((T, K)).cuda()
    moe.moe_combine_sorted_backward(cut(dy.cuda()), cut(ys.cuda()), w.cuda(), pos.cuda(), cut(dys), dw)
    wys, ww, size = combine_backward(cut(dy), cut(ys), w, pos)
    within(cut(dys)[:rows], wys[:rows], FMA * wys[:rows].abs(), a)
    assert (dys[:, :off] == 9).all() and (dys[:, off + H:] == 9).all() and (dys[rows:] == 9).all()
    within(dw, ww, H * FMA * size, torch.float32)


def test_one_gradient_alone_and_in_place():
    pos, rows, ys, w, dy = data(40, 6, 512, torch.bfloat16, torch.bfloat16, 8, 0.3)
    d = dict(dy=dy.cuda(), w=w.cuda(), pos=pos.cuda())
    dys, dw = torch.full_like(ys, 9.0).cuda(), torch.empty((40, 6)).cuda()
    moe.moe_combine_sorted_backward(d["dy"], ys.cuda(), d["w"], d["pos"], dys, dw)
    a, b = torch.full_like(ys, 9.0).cuda(), torch.empty_like(dw)
    moe.moe_combine_sorted_backward(d["dy"], ys.cuda(), d["w"], d["pos"], a, None)
    moe.moe_combine_sorted_backward(d["dy"], ys.cuda(), d["w"], d["pos"], None, b)
    assert torch.equal(a, dys) and torch.equal(b, dw)
    c, b = ys.cuda(), torch.empty_like(dw)
    moe.moe_combine_sorted_backward(d["dy"], c, d["w"], d["pos"], c, b)   # the gradient over ys
    assert torch.equal(c[:rows], dys[:rows]) and torch.equal(b, dw) and torch.isnan(c[rows:]).all()


def test_rows_that_are_not_finite():
    """infinities and NaN stay with their tokens; tokens without any pick are 0"""
    T, K, H = 24, 4, 256
    pos, rows, ys, w, dy = data(T, K, H, torch.float16, torch.float32, 2, 0.5)
    pos[5] = -1
    ys[int(pos[pos >= 0][0]), 3], ys[int(pos[pos >= 0][-1]), 5] = float("inf"), float("nan")
    w[pos < 0] = float("nan")   # weights of picks that are left out
    y = torch.empty((T, H)).cuda()
    moe.moe_combine_sorted(ys.cuda(), w.cuda(), pos.cuda(), y)
    want, size = combine(ys, w, pos)
    within(y, want, K * FMA * size, torch.float32)
    assert (y[5] == 0).all() and torch.isfinite(want).sum() == T * H - 2
    dys, dw = torch.zeros_like(ys).cuda(), torch.empty((T, K)).cuda()
    moe.moe_combine_sorted_backward(dy.cuda(), ys.cuda(), w.cuda(), pos.cuda(), dys, dw)
    wys, ww, size = combine_backward(dy, ys, w, pos)
    within(dw, ww, H * FMA * size, torch.float32)
    named = torch.zeros(ys.shape[0], dtype=torch.bool)
    named[pos[pos >= 0].long()] = True
    within(dys[named.cuda()], wys[named], FMA * wys[named].abs(), torch.float16)
    assert (dys[~named.cuda()] == 0).all()


def test_gradients_against_differences():
    """combine is linear in ys and in w, sort in x: a difference quotient is exact but for the roundings"""
    T, K, H, h = 19, 5, 320, 0.5
    pos, rows, ys, w, dy = data(T, K, H, torch.float32, torch.float32, 4, 0.3)
    ys[rows:] = 0
    g = gen(9)
    v, u = torch.randn(ys.shape, generator=g), torch.randn(w.shape, generator=g)

    def comb(ys, w):
        y = torch.empty((T, H)).cuda()
        moe.moe_combine_sorted(ys.cuda(), w.cuda(), pos.cuda(), y)
        return y.cpu().double()

    dys, dw = torch.zeros_like(ys).cuda(), torch.empty((T, K)).cuda()
    moe.moe_combine_sorted_backward(dy.cuda(), ys.cuda(), w.cuda(), pos.cuda(), dys, dw)
    scale = float((dy.double().abs() * combine(ys.abs() + v.abs(), w.abs() + u.abs(), pos)[1]).sum())   # bounds every term below
    bound = (2 * K + 2) * 2.0 ** -23 * scale / h
    by_ys = ((comb(ys + h * v, w) - comb(ys - h * v, w)) / (2 * h) * dy.double()).sum()
    assert abs(by_ys - (dys.cpu().double() * v.double()).sum()) <= bound
    by_w = ((comb(ys, w + h * u) - comb(ys, w - h * u)) / (2 * h) * dy.double()).sum()
    assert abs(by_w - (dw.cpu().double() * u.double()).sum()) <= bound + H * FMA * scale

    def sort(x):
        xs = torch.zeros((rows, H)).cuda()
        moe.moe_sort_rows(x.cuda(), pos.cuda(), xs)
        return xs.cpu().double()

    x, z, dxs = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g), torch.randn((rows, H), generator=g)
    dx = torch.empty((T, H)).cuda()
    moe.moe_sort_rows_backward(dxs.cuda(), pos.cuda(), dx)
    by_x = ((sort(x + h * z) - sort(x - h * z)) / (2 * h) * dxs.double()).sum()
    scale = float((combine(dxs.abs(), torch.ones_like(w), pos)[1] * (x.abs() + z.abs()).double()).sum())
    assert abs(by_x - (dx.cpu().double() * z.double()).sum()) <= (K + 2) * 2.0 ** -23 * scale / h


def test_past_32_bit_offsets():
    """rows of 2^20 values, the last of them 2.1e9 values and 4.3e9 bytes behind the first"""
    H, rows, T, K = 1 << 20, 2080, 2, 2
    ys = torch.zeros((rows, H), dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor([[rows - 1, 0], [3, rows - 2]], dtype=torch.int32).cuda()
    x = torch.stack([torch.arange(H, device="cuda") % 251, torch.arange(H, device="cuda") % 127 + 1]).to(torch.bfloat16)
    moe.moe_sort_rows(x, pos, ys)
    assert torch.equal(ys[rows - 1], x[0]) and torch.equal(ys[0], x[0]) and torch.equal(ys[rows - 2], x[1]) and torch.equal(ys[3], x[1])
    assert not ys[1:3].any() and not ys[4:rows - 2].any()
    w = torch.tensor([[0.5, 0.25], [2.0, 1.0]]).cuda()
    y = torch.empty((T, H), device="cuda")
    moe.moe_combine_sorted(ys, w, pos, y)
    assert torch.equal(y[0], 0.75 * x[0].float()) and torch.equal(y[1], 3 * x[1].float())
    dw = torch.empty((T, K), device="cuda")
    moe.moe_combine_sorted_backward(x, ys, w, pos, ys, dw)
    sq = x.double().square().sum(1)
    assert ((dw.double() - sq[:, None]).abs() <= H * FMA * sq[:, None]).all()
    assert torch.equal(ys[rows - 1], (0.5 * x[0].float()).bfloat16()) and torch.equal(ys[rows - 2], x[1])


def test_nothing_to_do():
    """no tokens; no sorted rows at all"""
    pos, w = torch.zeros((0, 4), dtype=torch.int32).cuda(), torch.zeros((0, 4)).cuda()
    x, ys = torch.zeros((0, 64)).cuda(), torch.full((3, 64), 2.0).cuda()
    moe.moe_sort_rows(x, pos, ys)
    moe.moe_combine_sorted(ys, w, pos, x)
    moe.moe_combine_sorted_backward(x, ys, w, pos, ys, w)
    assert (ys == 2).all()
    pos, w, x = torch.full((3, 4), -1, dtype=torch.int32).cuda(), torch.zeros((3, 4)).cuda(), torch.ones((3, 64)).cuda()
    none, dw = torch.zeros((0, 64)).cuda(), torch.ones((3, 4)).cuda()
    moe.moe_sort_rows(x, pos, none)
    moe.moe_combine_sorted_backward(x, none, w, pos, none, dw)
    moe.moe_combine_sorted(none, w, pos, x)
    assert not x.any() and not dw.any()


def test_in_a_graph_and_on_other_streams():
    """the whole way there and back, captured, replayed on other inputs; two such at once on streams of their own"""
    T, K, E, H = 200, 6, 32, 1024

    class Way:
        def __init__(self):
            self.ids, self.x = torch.zeros((T, K), dtype=torch.int32).cuda(), torch.zeros((T, H), dtype=torch.bfloat16).cuda()
            self.w, self.y = torch.zeros((T, K)).cuda(), torch.zeros((T, H)).cuda()
            self.xs, self.g = torch.zeros((T * K, H), dtype=torch.bfloat16).cuda(), moe.RowGroups(T * K, E)
            self.dys, self.dw, self.dx = torch.zeros_like(self.xs), torch.zeros((T, K)).cuda(), torch.zeros((T, H)).cuda()

        def fill(self, seed):
            g = gen(seed)
            self.ids.copy_(torch.randint(-1, E, (T, K), generator=g, dtype=torch.int32))
            self.x.copy_(torch.randn((T, H), generator=g))
            self.w.copy_(torch.rand((T, K), generator=g))

        def run(self):
            moe.group_rows(self.ids, self.g)
            moe.moe_sort_rows(self.x, self.g.pos, self.xs)
            moe.moe_combine_sorted(self.xs, self.w, self.g.pos.view(T, K), self.y)
            moe.moe_combine_sorted_backward(self.y, self.xs, self.w, self.g.pos.view(T, K), self.dys, self.dw)
            moe.moe_sort_rows_backward(self.dys, self.g.pos.view(T, K), self.dx)

        def out(self):
            return [self.y.clone(), self.dw.clone(), self.dx.clone()]

    a, b, e = Way(), Way(), Way()
    graphs = []
    for way in (a, b):
        way.run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            way.run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(3):
        for i, way in enumerate((a, b)):
            way.fill(2 * k + i)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for i, way in enumerate((a, b)):
            e.fill(2 * k + i)
            e.run()
            for p, q in zip(way.out(), e.out()):
                assert torch.equal(p, q)


def test_python_refuses():
    f = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    A, B = f(2, 8, 16, t=torch.bfloat16), f(2, 24, 8, t=torch.bfloat16)
    ad, g = moe.Adapters(A, B), moe.RowGroups(4, 3, in_place=True)
    mm = lambda x=f(4, 16), base=None, out=f(4, 24), jobs=g.jobs, cap=g.cap: moe.adapter_mm(ad, jobs, g.njobs, cap, x, base, out)
    for call, msg in [
        (lambda: moe.group_rows(i(5), g), "ids: 5 rows"), (lambda: moe.group_rows(i(4, 2)[:, :1], g), "ids: not contiguous"),
        (lambda: moe.group_rows(i(4), moe.RowGroups(4, 3, device="cpu")), "g: not on"),
        (lambda: moe.group_rows(i(4), moe.RowGroups(4, 4097)), "n_groups out of range"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(4, 2), f(8, 9)), "xs: shape"), (lambda: moe.moe_sort_rows(f(4, 8), i(3, 2), f(8, 8)), "pos:"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(9), f(8, 8)), "pos:"), (lambda: moe.moe_sort_rows(f(4, 8), i(4, 65), f(8, 8)), "K out of range"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(4, 0), f(8, 8)), "K out of range"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(4, 2), f(8).expand(8, 8)), "xs: rows overlap"),
        (lambda: moe.moe_combine_sorted(f(8, 8), f(4, 2), i(4, 2), f(4, 9)), "y: shape"),
        (lambda: moe.moe_combine_sorted(f(8, 8), f(4, 3), i(4, 2), f(4, 8)), "topw: shape"),
        (lambda: moe.moe_combine_sorted(f(8, 8), f(4, 2).double(), i(4, 2), f(4, 8)), "topw: type"),
        (lambda: moe.moe_combine_sorted_backward(f(4, 8), f(8, 9), f(4, 2), i(4, 2), None, None), "ys: shape"),
        (lambda: moe.moe_combine_sorted_backward(f(4, 8), f(8, 8), f(4, 2), i(4, 2), f(7, 8), None), "dys: shape"),
        (lambda: moe.moe_combine_sorted_backward(f(4, 8), f(8, 8), f(4, 2), i(4, 2), None, f(8)), "dw: shape"),
        (lambda: moe.Adapters(A, f(2, 24, 16, t=torch.bfloat16)), "B: shape"), (lambda: moe.Adapters(A, B.half()), "B: type"),
        (lambda: moe.Adapters(A, B, f(3)), "scale: shape"), (lambda: moe.Adapters([A[0], A[1, :, :8]], [B[0], B[1]]), "A: shape"),
        (lambda: mm(x=f(4, 24)), "x: shape"), (lambda: mm(x=f(4, 16, t=torch.float16)), "x: type"), (lambda: mm(out=f(3, 24)), "out: shape"),
        (lambda: mm(base=f(4, 24, t=torch.float16)), "base: type"), (lambda: mm(base=f(4, 48)[:, :24]), "base: rows 48 values apart"),
        (lambda: mm(cap=100), "jobs: smaller"), (lambda: mm(jobs=g.jobs.long()), "jobs: type"), (lambda: mm(x=f(4, 17)[:, :16]), "ldx must be"),
    ]:
        with pytest.raises((ValueError, RuntimeError), match=msg):
            call()
    torch.cuda.synchronize()
