"""What the calls on grouped and sorted rows and adapters refuse, on the host, before anything is launched."""
import pytest
import torch

from sfnx_amd import _abi, moe

P = 4096   # a device pointer that is never dereferenced
BIG = 1 << 40


def group(L, ids=P, n=10, G=4, off=P, pos=P, order=P, jobs=P, njobs=P, cap=10, ws=None, wb=0):
    return L.sfnx_group_rows(ids, n, G, off, pos, order, jobs, njobs, cap, 0, ws, wb, None)


def sort(L, elem=2, x=P, ldx=64, T=4, K=2, H=64, pos=P, xs=P, ldxs=64, rows=8):
    return L.sfnx_moe_sort_rows(elem, x, ldx, T, K, H, pos, xs, ldxs, rows, None)


def combine(L, a=1, ys=P, ldys=64, rows=8, w=P, pos=P, T=4, K=2, H=64, b=0, y=P, ldy=64):
    return L.sfnx_moe_combine_sorted(a, ys, ldys, rows, w, pos, T, K, H, b, y, ldy, None)


def backward(L, b=1, dy=P, lddy=64, a=1, ys=P, ldys=64, rows=8, w=P, pos=P, T=4, K=2, H=64, dys=P, lddys=64, dw=P):
    return L.sfnx_moe_combine_sorted_backward(b, dy, lddy, a, ys, ldys, rows, w, pos, T, K, H, dys, lddys, dw, None)


def adapter(L, A=P, sa=BIG, B=P, sb=BIG, t=30, scale=P, n=2, R=16, ni=64, no=64, jobs=P, njobs=P, cap=2, xt=30, x=P, ldx=64, base=P, ot=0, out=P, ldo=64,
            rows=4, ws=None, wb=0):
    return L.sfnx_adapter_mm(A, sa, B, sb, t, scale, n, R, ni, no, jobs, njobs, cap, xt, x, ldx, base, ot, out, ldo, rows, ws, wb, None)


@pytest.mark.parametrize("fn, args, msg", [
    (group, dict(n=-1), "n out of range"), (group, dict(n=(1 << 24) + 1, cap=1 << 20), "n out of range"), (group, dict(n=70000, cap=2000), "workspace smaller"),
    (group, dict(n=70000, cap=2000, ws=P, wb=4 * 4 * 128 - 1), "workspace smaller"), (group, dict(n=70000, cap=2000, ws=P + 2, wb=BIG), "4-byte aligned"),
    (group, dict(G=0), "n_groups out of range"), (group, dict(G=4097), "n_groups out of range"),
    (group, dict(ids=None), "null pointer"), (group, dict(off=None), "null pointer"),
    (group, dict(njobs=None), "go together"), (group, dict(jobs=None), "go together"),
    (group, dict(cap=3), "njobs_cap smaller"), (group, dict(n=130, G=1, cap=2), "njobs_cap smaller"), (group, dict(ids=P + 2), "4-byte aligned"),
    (sort, dict(elem=3), "1, 2 or 4 bytes"), (sort, dict(elem=8), "1, 2 or 4 bytes"), (sort, dict(T=-1), "T out of range"),
    (sort, dict(K=0), "K out of range"), (sort, dict(K=65), "K out of range"), (sort, dict(H=0), "H out of range"),
    (sort, dict(H=(1 << 20) + 1, ldx=BIG, ldxs=BIG), "H out of range"), (sort, dict(rows=-1), "rows out of range"), (sort, dict(pos=None), "null pointer"),
    (sort, dict(pos=P + 1), "4-byte aligned"), (sort, dict(x=None), "null pointer"), (sort, dict(xs=None), "null pointer"),
    (sort, dict(x=P + 1), "aligned to their type"), (sort, dict(ldx=63), "row stride"), (sort, dict(ldxs=-64), "row stride"),
    (sort, dict(T=2 ** 31 - 1, H=1 << 20, ldx=1 << 20, ldxs=1 << 20), "too many rows"),
    (combine, dict(a=2), "type must be"), (combine, dict(b=12), "type must be"), (combine, dict(w=None), "null pointer"), (combine, dict(w=P + 2), "4-byte aligned"),
    (combine, dict(y=None), "null pointer"), (combine, dict(ys=None), "null pointer"), (combine, dict(y=P + 2), "aligned to their type"),
    (combine, dict(ldy=10), "row stride"), (combine, dict(K=65), "K out of range"),
    (backward, dict(a=3), "type must be"), (backward, dict(b=3), "type must be"), (backward, dict(dy=None), "null pointer"), (backward, dict(ys=None), "null pointer"),
    (backward, dict(w=None), "null pointer"), (backward, dict(dw=P + 2), "4-byte aligned"), (backward, dict(dys=P + 1), "aligned to their type"),
    (backward, dict(lddys=3), "row stride"), (backward, dict(lddy=BIG * 4), "row stride"),
    (adapter, dict(t=0), "adapter type"), (adapter, dict(t=1), "x type must be"), (adapter, dict(xt=1), "x type must be"), (adapter, dict(ot=7), "out type"),
    (adapter, dict(n=0), "n_adapters out of range"), (adapter, dict(R=12), "rank must be"), (adapter, dict(R=136), "rank must be"), (adapter, dict(R=0), "rank must be"),
    (adapter, dict(ni=60), "input width"), (adapter, dict(ni=(1 << 20) + 8, ldx=BIG), "input width"), (adapter, dict(no=0), "n_out out of range"),
    (adapter, dict(no=(1 << 20) + 1, ldo=BIG), "n_out out of range"), (adapter, dict(sa=16), "stride smaller"), (adapter, dict(sb=16), "stride smaller"),
    (adapter, dict(sa=BIG + 8), "multiple of 16"), (adapter, dict(rows=-1), "rows out of range"), (adapter, dict(cap=-1), "njobs out of range"),
    (adapter, dict(A=None), "null pointer"), (adapter, dict(jobs=None), "null pointer"), (adapter, dict(out=None), "null pointer"),
    (adapter, dict(B=P + 8), "16-byte aligned"), (adapter, dict(x=P + 2), "16-byte aligned"), (adapter, dict(ldx=63), "ldx must be"), (adapter, dict(ldx=68), "ldx must be"),
    (adapter, dict(ldo=63), "ldo smaller"), (adapter, dict(out=P + 2), "aligned to their type"), (adapter, dict(base=P + 2), "aligned to their type"),
    (adapter, dict(R=40), "workspace smaller"), (adapter, dict(R=40, ws=P, wb=1023), "workspace smaller"), (adapter, dict(R=40, ws=P + 4, wb=BIG), "workspace must be"),
    (adapter, dict(scale=P + 2), "4-byte aligned"), (adapter, dict(jobs=P + 2), "4-byte aligned"),
])
def test_library_refuses(fn, args, msg):
    L = _abi.lib()
    assert fn(L, **args) == -1
    assert msg in L.sfnx_last_error().decode()


def test_python_refuses():
    """on a host without a GPU: whatever is right in type and shape is refused for its place"""
    f = lambda *s, t=torch.float32: torch.zeros(s, dtype=t)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    g = moe.RowGroups(10, 3, device="cpu")
    cases = [
        (lambda: moe.RowGroups(-1, 3, device="cpu"), "n below 0"), (lambda: moe.RowGroups(1, 0, device="cpu"), "no groups"),
        (lambda: moe.group_rows(i(5).long(), g), "ids: type"), (lambda: moe.group_rows(i(5), g), "ids: not on"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(4, 2), f(8, 8, t=torch.float16)), "expected the same"),
        (lambda: moe.moe_sort_rows(f(4, 8).double(), i(4, 2), f(8, 8).double()), "expected the same"),
        (lambda: moe.moe_sort_rows(f(4), i(4, 2), f(8, 8)), "1 dimensions"), (lambda: moe.moe_sort_rows(f(8, 4).t(), i(4, 2), f(8, 8)), "not contiguous"),
        (lambda: moe.moe_sort_rows(f(4, 8), i(4, 2), f(8, 8)), "not on the current GPU"),
        (lambda: moe.moe_combine_sorted(f(8, 8), f(4, 2), i(4, 2), f(4, 9)), "ys: not on"),
        (lambda: moe.moe_combine_sorted(f(8, 8).double(), f(4, 2), i(4, 2), f(4, 8)), "ys: type"),
        (lambda: moe.moe_sort_rows_backward(f(8, 8, t=torch.uint8), i(4, 2), f(4, 8)), "dxs: type"),
        (lambda: moe.Adapters(f(2, 8, 16), f(2, 5, 8)), "A: type"), (lambda: moe.Adapters(f(0, 8, 16), f(0, 5, 8)), "for every adapter"),
        (lambda: moe.Adapters(f(2, 8, t=torch.bfloat16), f(2, 5, 8, t=torch.bfloat16)), "A: 2 dimensions"),
        (lambda: moe.Adapters([f(8, 16, t=torch.bfloat16)], [f(8, t=torch.bfloat16)]), "B: 1 dimensions"),
        (lambda: moe.Adapters(f(2, 8, 16, t=torch.bfloat16), f(3, 5, 8, t=torch.bfloat16)), "for every adapter"),
        (lambda: moe.Adapters(f(2, 8, 16, t=torch.bfloat16), f(2, 5, 4, t=torch.bfloat16)), "B: shape|A: not on"),
    ]
    for k, (call, msg) in enumerate(cases):
        with pytest.raises(ValueError, match=msg):
            call()


def test_workspaces_grow_with_rows():
    """a workspace for the most rows serves fewer; none where one launch is used"""
    L = _abi.lib()
    for args in ((16, 1 << 20, 30), (40, 4096, 30), (128, 64, 0), (32, 2048, 0)):
        last = 0
        for rows in list(range(0, 9000, 7)) + [1 << 16, 1 << 20]:
            now = L.sfnx_adapter_workspace(rows, *args)
            assert now >= last
            last = now
    assert L.sfnx_adapter_workspace(1024, 32, 4096, 30) == 0 and L.sfnx_adapter_workspace(16, 32, 4096, 0) == 0 and L.sfnx_adapter_workspace(1, 40, 4096, 0) > 0
    last = 0
    for n in list(range(0, 300000, 997)) + [1 << 24]:
        now = L.sfnx_group_rows_workspace(n, 512)
        assert now >= last
        last = now
    assert L.sfnx_group_rows_workspace(65536, 4096) == 0 and last == 4 * 128 * 512
