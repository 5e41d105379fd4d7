"""The operators on sorted rows and adapters together with the router, the experts' products and the layers."""
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import matrices as f8_matrices
from tests.rows_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def layer16(s, seed):
    g = gen(seed)
    n = s.E + (1 if s.shared else 0)
    return moe.MoeLayer16(s, (torch.randn((s.E + 1, s.H), generator=g) * 0.05).cuda(), (torch.randn((n, 2 * s.ff, s.H), generator=g) * 0.03).half().cuda(),
                          (torch.randn((n, s.H, s.ff), generator=g) * 0.05).half().cuda())


@pytest.mark.parametrize("T", [1, 20, 300])
def test_a_prompt_over_sorted_rows(T):
    """router, group, sort, the experts' products over sorted rows, combine: layer_16's values"""
    s = moe.LayerShape(H=1024, E=64, K=6, ff=512, shared=False)
    L, b = layer16(s, 1), moe.FloatBuffers(s, max(T, 17))
    x = torch.randn((b.T, s.H), generator=gen(T)).cuda()
    want = torch.empty_like(x)
    moe.layer_16(L, x, want, b)
    T = b.T
    P, g = T * s.K, moe.RowGroups(T * s.K, s.E)
    moe.group_rows(b.topi, g)
    xs, gu, h, ys = (torch.zeros((P, n), dtype=t, device="cuda") for n, t in ((s.H, torch.float16), (2 * s.ff, torch.float32), (s.ff, torch.float16), (s.H, torch.float32)))
    y = torch.zeros_like(x)
    moe.moe_sort_rows(b.xh, g.pos, xs)
    moe.moe_mm_16_big(L.gu_w, L.gu_stride, s.H, 2 * s.ff, g.jobs, g.njobs, g.cap, xs, gu)
    moe.swiglu_h16(gu, h, s.ff)
    moe.moe_mm_16_big(L.dn_w, L.dn_stride, s.ff, s.H, g.jobs, g.njobs, g.cap, h, ys)
    moe.moe_combine_sorted(ys, b.topw, g.pos.view(T, s.K), y)
    assert torch.equal(gu[g.pos.long()], b.gu[:P]) and torch.equal(ys[g.pos.long()], b.part[:P])
    assert torch.equal(y, want)


def test_a_prompt_over_sorted_8_bit_rows():
    """the same with 8-bit experts, whose rows and scales are sorted each, and the shared expert one more pick of every token"""
    s, T = moe.LayerShape(H=1024, E=64, K=6, ff=512), 200
    g = gen(3)
    gu_w, _ = f8_matrices(g, s.E + 1, 2 * s.ff, s.H)
    dn_w, _ = f8_matrices(g, s.E + 1, s.H, s.ff)
    L = moe.MoeLayerF8(s, (torch.randn((s.E + 1, s.H), generator=g) * 0.05).cuda(), gu_w.cuda(), dn_w.cuda())
    b, x = moe.FloatBuffers(s, T), torch.randn((T, s.H), generator=g).cuda()
    want = torch.empty_like(x)
    moe.layer_f8(L, x, want, b)
    ids = torch.cat([b.topi, torch.full((T, 1), s.E, dtype=torch.int32, device="cuda")], 1)
    gate = torch.sigmoid(b.logits[:, s.E:])
    n, K = T * (s.K + 1), s.K + 1
    r = moe.RowGroups(n, s.E + 1)
    moe.group_rows(ids, r)
    q, qs = torch.zeros((n, s.H), dtype=torch.uint8, device="cuda"), torch.zeros((n, s.H // 128), device="cuda")
    hq, hs = torch.zeros((n, s.ff), dtype=torch.uint8, device="cuda"), torch.zeros((n, s.ff // 128), device="cuda")
    ys, y = torch.zeros((n, s.H), device="cuda"), torch.zeros_like(x)
    moe.moe_sort_rows(b.xq, r.pos.view(T, K), q)
    moe.moe_sort_rows(b.xs, r.pos.view(T, K), qs)
    moe.moe_gate_up_swiglu_f8_big(L.gu_w, L.gu_stride, s.H, s.ff, r.jobs, r.njobs, r.cap, q, qs, hq, hs)
    moe.moe_down_f8_big(L.dn_w, L.dn_stride, s.ff, s.H, r.jobs, r.njobs, r.cap, hq, hs, ys)
    moe.moe_combine_sorted(ys, torch.cat([b.topw, gate], 1), r.pos.view(T, K), y)
    pos = r.pos.view(T, K).long()
    assert torch.equal(ys[pos[:, : s.K].reshape(-1)], b.part[: T * s.K]) and torch.equal(ys[pos[:, s.K]], b.part[T * s.K:])
    # the sigmoids may differ by some steps of 2^-24
    size = (ys[pos[:, s.K]].abs() * gate).double()
    assert ((y.double() - want.double()).abs() <= 8 * FMA * size + 2 * FMA * want.abs().double()).all()


def adapters(n, R, n_in, n_out, seed):
    g = gen(seed)
    A, B = (torch.randn((n, R, n_in), generator=g) / n_in ** 0.5).half(), (torch.randn((n, n_out, R), generator=g) / R ** 0.5).half()
    return A, B, torch.rand((n,), generator=g) + 0.5


@pytest.mark.parametrize("T, R, table", [(1, 16, False), (7, 8, True), (16, 64, False), (90, 16, False), (300, 32, True)])
def test_layer_with_adapters(T, R, table):
    """layer_16's shared expert with adapters of its three products: each addition within its bound of 64 bits, what follows from the
    layer's own calls, and rows without an adapter unchanged"""
    s, n = moe.LayerShape(H=1024, E=64, K=6, ff=512), 5
    L, b, b0 = layer16(s, 2), moe.FloatBuffers(s, T), moe.FloatBuffers(s, T)
    x = torch.randn((T, s.H), generator=gen(T)).cuda()
    y, y0 = torch.empty_like(x), torch.empty_like(x)
    ids = torch.randint(-1, n, (T,), generator=gen(T + 1), dtype=torch.int32)
    ids[0] = 3
    if T > 1:
        ids[1] = -1
    g = moe.RowGroups(T, n, in_place=True)
    moe.group_rows(ids.cuda(), g)
    cpu = {k: adapters(n, R, i, o, v) for v, (k, i, o) in enumerate((("gate", s.H, s.ff), ("up", s.H, s.ff), ("down", s.ff, s.H)))}
    gpu = {k: moe.Adapters([m.cuda() for m in A] if table else A.cuda(), [m.cuda() for m in B] if table else B.cuda(), f.cuda()) for k, (A, B, f) in cpu.items()}
    moe.layer_16(L, x, y0, b0)
    moe.layer_16(L, x, y, b, moe.SharedAdapters(**gpu, groups=g))
    P, f32 = T * s.K, torch.float32
    for k, c in (("gate", slice(0, s.ff)), ("up", slice(s.ff, 2 * s.ff))):
        want, bound = adapted(b.xh.cpu(), *cpu[k], ids, b0.gu[P:, c].cpu())
        within(b.gu[P:, c], want, bound, f32)
    assert torch.equal(b.gu[:P], b0.gu[:P])
    h, part = torch.empty_like(b.h16), torch.zeros_like(b.part)
    moe.swiglu_h16(b.gu, h, s.ff)
    assert torch.equal(h, b.h16)
    mm = moe.moe_mm_16_big if b.big else moe.moe_mm_16
    mm(L.dn_w, L.dn_stride, s.ff, s.H, b.jobs_dn, b.njobs, b.cap, h, part)
    want, bound = adapted(h[P:].cpu(), *cpu["down"], ids, part[P:].cpu())
    within(b.part[P:], want, bound, f32)
    moe.moe_combine(b.part, b.topw, b.topi, b.logits, part[:T], s.E, s.K, True)
    assert torch.equal(part[:T], y)
    none = (ids < 0).cuda()
    assert torch.equal(y[none], y0[none]) and not torch.equal(y[~none], y0[~none])
    moe.layer_16(L, x, y, b, moe.SharedAdapters(None, None, None, g))
    assert torch.equal(y, y0)


def test_layer_refuses_adapters():
    s = moe.LayerShape(H=1024, E=64, K=6, ff=512, shared=False)
    A, B, f = adapters(2, 8, 512, 1024, 1)
    ad = moe.Adapters(A.cuda(), B.cuda())
    x = torch.zeros((3, s.H)).cuda()
    for shape, sh, msg in ((s, moe.SharedAdapters(None, None, ad, moe.RowGroups(3, 2, in_place=True)), "no shared expert"),
                           (moe.LayerShape(H=1024, E=64, K=6, ff=512), moe.SharedAdapters(ad, None, None, moe.RowGroups(3, 2, in_place=True)), "adapters.gate: 512 -> 1024"),
                           (moe.LayerShape(H=1024, E=64, K=6, ff=512), moe.SharedAdapters(None, None, ad, moe.RowGroups(3, 2)), "adapters.groups")):
        with pytest.raises(ValueError, match=msg):
            moe.layer_16(layer16(shape, 1), x, torch.empty_like(x), moe.FloatBuffers(shape, 3), sh)


def test_a_tuning_step():
    """y = sum_k w_k f(x W_e): the gradients of the weights, the tokens and the experts' matrices through sorted rows, against torch's own
    over the same formula in 64 bits"""
    T, K, E, H, F = 50, 3, 6, 64, 96
    g = gen(5)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int()
    ids[3, 1] = -1
    w, x, W, dy = torch.rand((T, K), generator=g), torch.randn((T, H), generator=g), torch.randn((E, H, F), generator=g), torch.randn((T, F), generator=g)
    r = moe.RowGroups(T * K, E)
    moe.group_rows(ids.cuda(), r)
    pos, off = r.pos.view(T, K), r.offsets.tolist()
    V = off[-1]
    xs, ys, y = torch.zeros((V, H)).cuda(), torch.zeros((V, F)).cuda(), torch.zeros((T, F)).cuda()
    moe.moe_sort_rows(x.cuda(), pos, xs)
    for e in range(E):
        ys[off[e]:off[e + 1]] = xs[off[e]:off[e + 1]] @ W[e].cuda()
    moe.moe_combine_sorted(ys, w.cuda(), pos, y)
    dys, dw, dxs, dx, dW = torch.zeros_like(ys), torch.zeros((T, K)).cuda(), torch.zeros_like(xs), torch.zeros((T, H)).cuda(), torch.zeros((E, H, F)).cuda()
    moe.moe_combine_sorted_backward(dy.cuda(), ys, w.cuda(), pos, dys, dw)
    for e in range(E):
        dxs[off[e]:off[e + 1]] = dys[off[e]:off[e + 1]] @ W[e].t().contiguous().cuda()
        dW[e] = xs[off[e]:off[e + 1]].t().contiguous() @ dys[off[e]:off[e + 1]]
    moe.moe_sort_rows_backward(dxs, pos, dx)
    a, b, c = (v.double().requires_grad_() for v in (w, x, W))
    there = ids >= 0
    out = torch.stack([torch.stack([a[t, k] * (b[t] @ c[int(ids[t, k])]) for k in range(K) if there[t, k]]).sum(0) for t in range(T)])
    (out * dy.double()).sum().backward()
    # each value is a sum of at most H + F + T K products in 32 bits of unit sizes' products: 2^-23 of the sum of their sizes, which the norms bound
    n = H + F + T * K
    size = lambda *v: float(torch.stack([u.double().abs().max() for u in v]).prod()) * n
    for got, want, s in ((y, out.detach(), size(w, x, W)), (dw, a.grad, size(dy, x, W) * H), (dx, b.grad, size(w, dy, W)), (dW, c.grad, size(w, dy, x))):
        assert ((got.cpu().double() - want).abs() <= n * STEP * s).all()
    assert dw[3, 1] == 0
