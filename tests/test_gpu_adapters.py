"""adapter_mm against 64 bits, within the bounds of 32-bit sums and one rounding."""
import numpy as np
import pytest
import torch

from sfnx_amd import _abi, moe
from tests.rows_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def matrices(n, R, n_in, n_out, t, seed=1):
    g = gen(seed)
    return rand(g, (n, R, n_in), t), rand(g, (n, n_out, R), t), torch.rand((n,), generator=g) - 0.3


def adapter_ids(T, n, seed, none=0.2, sorted_=False):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, n, T)
    ids = np.sort(ids) if sorted_ else ids
    ids[rng.random(T) < none] = -1
    return torch.tensor(ids, dtype=torch.int32)


def plan(ids, n, none_too=False):
    """the job list; none_too: rows without an adapter are listed as group n"""
    g = moe.RowGroups(ids.numel(), n + 1, in_place=True)
    moe.group_rows(torch.where(ids < 0, torch.full_like(ids, n), ids).cuda() if none_too else ids.cuda(), g)
    return g


def call(ad, g, x, base, out):
    moe.adapter_mm(ad, g.jobs, g.njobs, g.cap, x, base, out)


SIZES = [(1, 1, 8, 8, 1), (1, 3, 16, 2048, 1024), (3, 2, 8, 72, 33), (16, 20, 16, 1024, 512), (17, 4, 24, 264, 145), (64, 1, 32, 512, 320),
         (65, 2, 48, 200, 1000), (150, 5, 64, 640, 257), (40, 3, 104, 136, 64), (333, 7, 128, 328, 96), (700, 3, 16, 2560, 2048)]


@pytest.mark.parametrize("t, x_t, out_t", [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("bf16", "f32", "f32"), ("f16", "f32", "f32"),
                                           ("f16", "f16", "f32"), ("bf16", "f32", "f16"), ("f16", "f16", "bf16")])
@pytest.mark.parametrize("T, n, R, n_in, n_out", SIZES)
def test_product(T, n, R, n_in, n_out, t, x_t, out_t):
    t, x_t, out_t = TYPES[t], TYPES[x_t], TYPES[out_t]
    A, B, scale = matrices(n, R, n_in, n_out, t)
    ids, g = adapter_ids(T, n, T), gen(T)
    x, base = rand(g, (T, n_in), x_t), rand(g, (T, n_out), out_t)
    ad = moe.Adapters(A.cuda(), B.cuda(), scale.cuda())
    want, bound = adapted(x, A, B, scale, ids, base)
    out = torch.full((T, n_out), 9.0, dtype=out_t).cuda()
    call(ad, plan(ids, n, True), x.cuda(), base.cuda(), out)   # rows without an adapter become base's
    within(out, want, bound, out_t)
    assert torch.equal(out[(ids < 0).cuda()].cpu(), base[ids < 0])
    there = base.cuda()
    call(ad, plan(ids, n), x.cuda(), there, there)             # in place: they are in no job
    assert torch.equal(there, out)
    there = base.cuda()
    call(ad, plan(ids, n, True), x.cuda(), there, there)       # or in one that adds nothing
    assert torch.equal(there, out)
    want, bound = adapted(x, A, B, scale, ids, torch.zeros_like(base))
    call(ad, plan(ids, n, True), x.cuda(), None, out)          # the adapters alone
    within(out, want, bound, out_t)
    out.fill_(9)
    call(ad, plan(ids, n), x.cuda(), None, out)                # rows of no job are left as they were
    within(out[(ids >= 0).cuda()], want[ids >= 0], bound[ids >= 0], out_t)
    assert (out[(ids < 0).cuda()] == 9).all()


@pytest.mark.parametrize("out_t", ["f32", "bf16"])
@pytest.mark.parametrize("ldx, x0, ldo, o0", [(264, 0, 600, 0), (272, 8, 600, 256), (256, 0, 601, 3), (264, 8, 256, 0)])
def test_strided(ldx, x0, ldo, o0, out_t):
    """half of a stacked output, rows apart and off their alignment; what lies beside is left as it was"""
    T, n, R, n_in, n_out, out_t = 90, 3, 16, 256, 253, TYPES[out_t]
    A, B, _ = matrices(n, R, n_in, n_out, torch.bfloat16)
    ids, g = adapter_ids(T, n, 1, 0.0), gen(2)
    x, buf = rand(g, (T, ldx), torch.bfloat16), rand(g, (T, ldo), out_t)
    out = buf.cuda()
    call(moe.Adapters(A.cuda(), B.cuda()), plan(ids, n), x.cuda()[:, x0:x0 + n_in], out[:, o0:o0 + n_out], out[:, o0:o0 + n_out])
    want, bound = adapted(x[:, x0:x0 + n_in], A, B, None, ids, buf[:, o0:o0 + n_out])
    within(out[:, o0:o0 + n_out], want, bound, out_t)
    assert torch.equal(out[:, :o0].cpu(), buf[:, :o0]) and torch.equal(out[:, o0 + n_out:].cpu(), buf[:, o0 + n_out:])


def test_matrices_that_live_apart():
    T, n, R, n_in, n_out = 50, 4, 16, 512, 384
    A, B, scale = matrices(n, R, n_in, n_out, torch.float16)
    ids = adapter_ids(T, n, 5)
    x, base = rand(gen(1), (T, n_in), torch.float16).cuda(), rand(gen(2), (T, n_out), torch.float32).cuda()
    a, b = torch.empty_like(base), torch.empty_like(base)
    g = plan(ids, n, True)
    call(moe.Adapters(A.cuda(), B.cuda(), scale.cuda()), g, x, base, a)
    call(moe.Adapters([m.cuda() for m in A], [m.cuda() for m in B], scale.cuda()), g, x, base, b)
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("x_t", ["f32", "bf16"])
def test_rows_that_are_not_finite(T, x_t):
    """infinities and NaN of a row, of an adapter or of base go where the formula takes them, with a rank that fills no tile"""
    n, R, n_in, n_out, x_t = 3, 8, 264, 70, TYPES[x_t]
    A, B, scale = matrices(n, R, n_in, n_out, torch.bfloat16)
    ids = adapter_ids(T, n, 3, 0.0)
    ids[:3] = torch.tensor([0, 0, 1])
    x, base = rand(gen(1), (T, n_in), x_t), rand(gen(2), (T, n_out), torch.float32)
    x[0, 5], x[2, 263], base[1, 4], base[1, 69] = float("inf"), float("nan"), float("-inf"), float("nan")
    A[2, 7, 0] = float("inf")
    out = torch.empty_like(base).cuda()
    call(moe.Adapters(A.cuda(), B.cuda(), scale.cuda()), plan(ids, n), x.cuda(), base.cuda(), out)
    want, bound = adapted(x, A, B, scale, ids, base)
    within(out, want, bound, torch.float32)
    assert torch.isfinite(out[((ids == 0) & (torch.arange(T) > 1)).cuda()]).all()


@pytest.mark.parametrize("t, x_t, out_t", [("bf16", "bf16", "bf16"), ("f16", "f32", "f32"), ("f16", "f16", "f16"), ("bf16", "f32", "f32")])
@pytest.mark.parametrize("T, n, R, n_in, n_out", [(1025, 4, 8, 264, 145), (1100, 9, 32, 1000, 520), (1500, 2, 24, 2048, 333), (17, 3, 32, 512, 256), (2000, 40, 16, 136, 128)])
def test_many_rows(T, n, R, n_in, n_out, t, x_t, out_t):
    test_product(T, n, R, n_in, n_out, t, x_t, out_t)


@pytest.mark.parametrize("T, R", [(7, 16), (7, 48), (130, 64), (1100, 16), (90, 128)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_matrices_that_are_not_finite(T, R, t):
    """infinities and NaN in A and B, of adapters of their own: each output is the formula's, the other adapters' are untouched"""
    n, n_in, n_out, t = 5, 264, 200, TYPES[t]
    A, B, scale = matrices(n, R, n_in, n_out, t)
    A[1, R - 1, 3], A[2, 0, 263] = float("-inf"), float("nan")
    B[3, 7, R - 1], B[3, 199, 0], B[4, 100, 2] = float("inf"), float("-inf"), float("nan")
    ids = adapter_ids(T, n, T, 0.1)
    ids[:5] = torch.arange(5)
    x, base = rand(gen(1), (T, n_in), t), rand(gen(2), (T, n_out), torch.float32)
    x[3] = 0
    x[3, 8] = 1.0   # so that most of this row's s has few bits
    out = base.cuda()
    call(moe.Adapters(A.cuda(), B.cuda(), scale.cuda()), plan(ids, n), x.cuda(), out, out)
    want, bound = adapted(x, A, B, scale, ids, base)
    within(out, want, bound, torch.float32)
    assert torch.isfinite(out[(ids == 0).cuda()]).all() and torch.isinf(out[3, [7, 199]]).all()


@pytest.mark.parametrize("T, R", [(5000, 16), (3000, 64), (700, 128)])
def test_few_jobs_of_many_rows(T, R):
    """a list shorter than the rows would fill: the rows' workspace, whose guard behind it stays, and rows of no job"""
    n, n_in, n_out = 2, 2048, 96
    A, B, scale = matrices(n, R, n_in, n_out, torch.bfloat16)
    x, base = rand(gen(1), (T, n_in), torch.bfloat16), rand(gen(2), (T, n_out), torch.float32)
    rows = torch.tensor([0, 5, T - 1, T // 2], dtype=torch.int32)
    a = torch.zeros((1, 130), dtype=torch.int32)
    a[0, 0], a[0, 1], a[0, 2:6], a[0, 66:70] = 1, 4, rows, rows
    ids = torch.full((T,), -1, dtype=torch.int32)
    ids[rows.long()] = 1
    d = dict(A=A.cuda(), B=B.cuda(), f=scale.cuda(), x=x.cuda(), out=base.cuda(), jobs=a.view(-1).cuda(), njobs=torch.tensor([1, 0], dtype=torch.int32).cuda())
    need = _abi.lib().sfnx_adapter_workspace(T, R, n_in, _abi.BF16)
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    p = {k: v.data_ptr() for k, v in d.items()}
    _abi.check(_abi.lib().sfnx_adapter_mm(p["A"], 2 * R * n_in, p["B"], 2 * n_out * R, _abi.BF16, p["f"], n, R, n_in, n_out, p["jobs"], p["njobs"], 1,
                                          _abi.BF16, p["x"], n_in, p["out"], _abi.F32, p["out"], n_out, T, ws.data_ptr(), need, moe._st()))
    want, bound = adapted(x, A, B, scale, ids, base)
    within(d["out"], want, bound, torch.float32)
    assert torch.equal(d["out"][(ids < 0).cuda()].cpu(), base[ids < 0]) and need and (ws[need:] == 0xAB).all()


def test_past_32_bit_offsets_of_few_rows():
    """rows 2^22 values apart, 700 of them"""
    T, n_in, n_out, R, ld = 700, 256, 264, 8, 1 << 22
    x = torch.zeros(T * ld, dtype=torch.float16, device="cuda").as_strided((T, n_in), (ld, 1))
    out = torch.zeros(T * ld, dtype=torch.float16, device="cuda").as_strided((T, n_out), (ld, 1))
    A, B = torch.zeros((2, R, n_in), dtype=torch.float16), torch.zeros((2, n_out, R), dtype=torch.float16)
    A[1, 3, 255], B[1, :, 3] = 2.0, (torch.arange(n_out) % 100).half()
    x[T - 1, 255] = 3.0
    ids = torch.full((T,), -1, dtype=torch.int32)
    ids[T - 1], ids[5] = 1, 0
    call(moe.Adapters(A.cuda(), B.cuda()), plan(ids, 2), x, out, out)
    assert torch.equal(out[T - 1].cpu(), 6 * B[1, :, 3]) and not out[:T - 1].any()


def test_two_forms_at_once_and_one_workspace_each():
    """calls with a workspace on two streams at once, and replayed beside each other"""
    T, n, R, n_in, n_out = 500, 3, 64, 1024, 512
    A, B, scale = matrices(n, R, n_in, n_out, torch.bfloat16)
    ad, ids = moe.Adapters(A.cuda(), B.cuda(), scale.cuda()), adapter_ids(T, n, 1)
    g = plan(ids, n, True)
    xs = [rand(gen(k), (T, n_in), torch.bfloat16).cuda() for k in range(2)]
    base, outs = rand(gen(9), (T, n_out), torch.float32).cuda(), [torch.zeros((T, n_out)).cuda() for _ in range(2)]
    want = []
    for x, out in zip(xs, outs):
        call(ad, g, x, base, out)
        want.append(out.clone())
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for x, out in zip(xs, outs):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(ad, g, x, base, out)
    for k in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for st, gr, x, out in zip(streams, graphs, xs, outs):
            with torch.cuda.stream(st):
                for _ in range(3):
                    gr.replay() if k % 2 else call(ad, g, x, base, out)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_sums_that_only_32_bits_hold():
    """s of two large terms that cancel and a small one, and s itself beside a base of another size: 16 bits anywhere on the way would lose them"""
    n_in, n_out, R = 64, 32, 8
    A, B = torch.zeros((1, R, n_in)), torch.zeros((1, n_out, R))
    A[0, 0, 0], A[0, 0, 63], A[0, 0, 20] = 1.0, -1.0, 1.0
    B[0, :, 0] = 1.0
    A[0, 1, 30], A[0, 1, 31] = 1.0, 2.0 ** -9
    B[0, :, 1] = 1.0
    x = torch.zeros((2, n_in))
    x[0, 0], x[0, 63], x[0, 20] = 4096.0, 4096.0, 0.0625
    x[1, 30], x[1, 31] = 1.0, 1.0
    for t in (torch.float16, torch.bfloat16):
        for x_t in (t, torch.float32):
            out = torch.empty((2, n_out)).cuda()
            call(moe.Adapters(A.to(t).cuda(), B.to(t).cuda()), plan(torch.zeros(2, dtype=torch.int32), 1), x.to(x_t).cuda(), None, out)
            assert (out[0] == 0.0625).all() and (out[1] == 1 + 2.0 ** -9).all()


def test_rows_of_a_job_outside():
    """job rows that x and out do not have are left out; so are jobs past njobs, and jobs without rows"""
    T, n, R, n_in, n_out = 20, 2, 16, 128, 96
    A, B, _ = matrices(n, R, n_in, n_out, torch.bfloat16)
    x, base = rand(gen(1), (T, n_in), torch.bfloat16), rand(gen(2), (T, n_out), torch.float32)
    a = torch.zeros((4, 130), dtype=torch.int32)
    a[0, 0], a[0, 1] = 1, 6
    a[0, 2:8] = torch.tensor([0, -1, T, 3, 2 ** 31 - 1, 5])
    a[0, 66:72] = torch.tensor([0, 1, 2, T, 4, 5])
    a[1, 0], a[1, 1] = 0, 0
    a[2, 0], a[2, 1], a[2, 2], a[2, 66] = -5, 1, 7, 7      # no adapter
    a[3, 0], a[3, 1], a[3, 2], a[3, 66] = 0, 1, 9, 9       # past njobs
    out = torch.full((T, n_out), 9.0).cuda()
    moe.adapter_mm(moe.Adapters(A.cuda(), B.cuda()), a.view(-1).cuda(), torch.tensor([3, 0], dtype=torch.int32).cuda(), 4, x.cuda(), base.cuda(), out)
    ids = torch.full((T,), -1, dtype=torch.int32)
    ids[[0, 5]] = 1
    want, bound = adapted(x, A, B, None, ids, base)
    done = torch.zeros(T, dtype=torch.bool)
    done[[0, 5, 7]] = True
    within(out[done.cuda()], want[done], bound[done], torch.float32)
    assert (out[~done.cuda()] == 9).all()


def test_past_32_bit_offsets():
    """rows of x and out whose last are past 2^31 values; a store of adapters past 4 GiB"""
    T, n_in, n_out, R = 2080, 1 << 20, 1 << 20, 8
    x, out = torch.zeros((T, n_in), dtype=torch.float16, device="cuda"), torch.zeros((T, n_out), dtype=torch.float16, device="cuda")
    A, B = torch.zeros((260, R, n_in), dtype=torch.float16, device="cuda"), torch.zeros((260, n_out, R), dtype=torch.float16, device="cuda")
    A[259, 3, n_in - 1], x[T - 1, n_in - 1] = 2.0, 3.0
    B[259, :, 3] = (torch.arange(n_out, device="cuda") % 100).half()
    ids = torch.full((T,), -1, dtype=torch.int32)
    ids[T - 1], ids[0] = 259, 258
    call(moe.Adapters(A, B), plan(ids, 260), x, out, out)
    assert torch.equal(out[T - 1], 6 * B[259, :, 3]) and not out[:T - 1].any()


def test_no_rows():
    A, B, _ = matrices(1, 8, 64, 64, torch.bfloat16)
    x, out = torch.zeros((0, 64), dtype=torch.bfloat16).cuda(), torch.zeros((0, 64)).cuda()
    g = plan(torch.zeros(0, dtype=torch.int32), 1)
    call(moe.Adapters(A.cuda(), B.cuda()), g, x, out, out)
    x, out = torch.zeros((4, 64), dtype=torch.bfloat16).cuda(), torch.ones((4, 64)).cuda()
    moe.adapter_mm(moe.Adapters(A.cuda(), B.cuda()), g.jobs, g.njobs, 0, x, None, out)
    call(moe.Adapters(A.cuda(), B.cuda()), plan(torch.full((4,), -1, dtype=torch.int32), 1), x, None, out)
    assert (out == 1).all()


def test_in_a_graph_and_on_another_stream():
    T, n, R, n_in, n_out = 100, 6, 32, 1024, 640
    A, B, scale = matrices(n, R, n_in, n_out, torch.bfloat16)
    ad = moe.Adapters(A.cuda(), B.cuda(), scale.cuda())
    ids, x = torch.zeros(T, dtype=torch.int32).cuda(), torch.zeros((T, n_in), dtype=torch.bfloat16).cuda()
    base, out = torch.zeros((T, n_out), dtype=torch.bfloat16).cuda(), torch.zeros((T, n_out), dtype=torch.bfloat16).cuda()
    g = moe.RowGroups(T, n + 1, in_place=True)

    def step():
        moe.group_rows(ids, g)
        call(ad, g, x, base, out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    st = torch.cuda.Stream()
    for k in range(4):
        now = torch.randint(0, n + 1, (T,), generator=gen(k), dtype=torch.int32)
        ids.copy_(now)
        x.copy_(rand(gen(k), (T, n_in), torch.bfloat16))
        base.copy_(rand(gen(k + 9), (T, n_out), torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            step()
        st.synchronize()
        assert torch.equal(got, out)
        want, bound = adapted(x.cpu(), A, B, scale, torch.where(now == n, -torch.ones_like(now), now), base.cpu())
        within(got, want, bound, torch.bfloat16)
