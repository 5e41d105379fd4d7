"""Whole layers of 8-bit and of f16 experts through the framework's routing, products and combine (layer_f8, layer_16): each
stage against 64 bits from the stage before it, and the layer in a graph beside eager calls."""
import numpy as np
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403
from tests.gpu_util import job_array
from tests.test_gpu_f8 import close, dev, gen

pytestmark = pytest.mark.gpu


def rows_of(jobs, n, big):
    """[(expert, y, out)] of the jobs the router made"""
    js = job_array(jobs, big)[:n]
    return [(int(j["w"]), int(j["y"][i]), int(j["out"][i])) for j in js for i in range(int(j["n"]))]


def shape_of(E, K, H, ff, shared):
    return moe.LayerShape(H=H, E=E, K=K, ff=ff, shared=shared)


def combined(b, s):
    """(y, bound) of the kernel's own part rows in 64 bits"""
    T, K = b.topi.shape
    part, w = b.part.double().cpu(), b.topw.double().cpu()
    terms = w[:, :, None] * part[: T * K].view(T, K, -1)
    if s.shared:
        terms = torch.cat([terms, torch.sigmoid(b.logits[:, s.E:].double().cpu())[:, :, None] * part[T * K:][:, None]], 1)
    return terms.sum(1), (K + 8) * ULP * terms.abs().sum(1)


@pytest.mark.parametrize("T", [1, 5, 16, 17, 150])
@pytest.mark.parametrize("E, K, H, ff, shared", [(64, 6, 1024, 512, True), (128, 8, 2560, 640, True), (64, 3, 1024, 144, False)])
def test_layer_f8(T, E, K, H, ff, shared):
    s = shape_of(E, K, H, ff, shared)
    g = gen(T + H)
    n = E + int(shared)
    gu, Wg = matrices(g, n, 2 * ff, H)
    dn, Wd = matrices(g, n, H, ff)
    L = moe.MoeLayerF8(s, dev(torch.randn((E + 1, H), generator=g) * 0.02), dev(gu), dev(dn))
    x, y = dev(torch.randn((T, H), generator=g)), torch.empty((T, H), device="cuda")
    b = moe.FloatBuffers(s, T)
    moe.layer_f8(L, x, y, b)
    torch.cuda.synchronize()
    wq, ws = quantize(x.cpu())
    assert torch.equal(b.xq.cpu(), wq.view(torch.uint8)) and torch.equal(b.xs.cpu(), ws)
    n = int(b.njobs[0])
    flat = rows_of(b.jobs_gu, n, b.big)
    assert sorted(f[2] for f in flat) == list(range(T * K + (T if shared else 0)))
    r, e, where = grouped(dequantize(wq, ws), Wg, flat, True)
    want, bound = swiglu(r, e, ff)
    if b.big:
        h = dequantize(b.hq.cpu().view(F8), b.hs.cpu())
        sc = spread(b.hs.cpu()[where].double(), ff)
        assert ((h[where] - want).abs() <= bound + (E4M3_HALF + 2 * ULP) * (want.abs() + bound) + E4M3_SUB * sc).all()
    else:
        close(b.h[where.cuda()], want, bound, torch.float32)
        h = dequantize(*quantize(b.h.cpu()))
    want, bound, where = grouped(h, Wd, rows_of(b.jobs_dn, n, b.big), True)
    close(b.part[where.cuda()], want, bound, torch.float32)
    close(y, *combined(b, s), torch.float32)


@pytest.mark.parametrize("T", [1, 16, 100])
@pytest.mark.parametrize("shared", [True, False])
def test_layer_16(T, shared):
    E, K, H, ff = 64, 6, 1024, 272
    s = shape_of(E, K, H, ff, shared)
    g = gen(T)
    n = E + int(shared)
    Wg, Wd = ((torch.randn(shp, generator=g) * 0.05).half() for shp in ((n, 2 * ff, H), (n, H, ff)))
    L = moe.MoeLayer16(s, dev(torch.randn((E + 1, H), generator=g) * 0.02), dev(Wg), dev(Wd))
    x, y = dev(torch.randn((T, H), generator=g)), torch.empty((T, H), device="cuda")
    b = moe.FloatBuffers(s, T)
    moe.layer_16(L, x, y, b)
    torch.cuda.synchronize()
    n = int(b.njobs[0])
    r, e, where = grouped(x.cpu().half().double(), Wg.double(), rows_of(b.jobs_gu, n, b.big), False)
    close(b.gu[where.cuda()], r, e, torch.float32)
    want, bound, where = grouped(b.h16.cpu().double(), Wd.double(), rows_of(b.jobs_dn, n, b.big), False)
    close(b.part[where.cuda()], want, bound, torch.float32)
    close(y, *combined(b, s), torch.float32)


@pytest.mark.parametrize("T", [3, 60])
def test_layer_f8_in_a_graph_beside_eager_calls(T):
    E, K, H, ff = 64, 6, 1024, 256
    s = shape_of(E, K, H, ff, True)
    g = gen(T)
    gu, dn = matrices(g, E + 1, 2 * ff, H)[0], matrices(g, E + 1, H, ff)[0]
    L = moe.MoeLayerF8(s, dev(torch.randn((E + 1, H), generator=g) * 0.02), dev(gu), dev(dn))
    xs = [dev(torch.randn((T, H), generator=g)) for _ in range(3)]
    b, b2 = moe.FloatBuffers(s, T), moe.FloatBuffers(s, T)
    x, y, y2 = xs[0].clone(), torch.empty((T, H), device="cuda"), torch.empty((T, H), device="cuda")
    moe.layer_f8(L, x, y, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.layer_f8(L, x, y, b)
    for i, v in enumerate(xs + xs):
        x.copy_(v)
        y.zero_()
        graph.replay()
        moe.layer_f8(L, v, y2, b2)   # eager, with buffers of its own
        torch.cuda.synchronize()
        assert torch.equal(y, y2), i
