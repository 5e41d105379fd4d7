"""What Adapters and RowGroups keep for the library's pointers and 32-bit sizes, on a host without a GPU."""
import gc
import weakref

import pytest
import torch

from sfnx_amd import moe


@pytest.fixture
def anywhere(monkeypatch):
    """tensors are taken where they are"""
    monkeypatch.setattr(moe, "_need", lambda *a, **k: None)


def bf(*s):
    return torch.ones(s, dtype=torch.bfloat16)


def test_adapters_hold_what_their_tables_name(anywhere):
    """a list whose entries are replaced, or cleared, after the tables were made: the matrices live as long as the adapters"""
    A, B = [bf(8, 16) for _ in range(3)], [bf(5, 8) for _ in range(3)]
    at = [m.data_ptr() for m in A], [m.data_ptr() for m in B]
    alive = [weakref.ref(m) for m in A + B]
    ad = moe.Adapters(A, B)
    A[1] = bf(8, 16)
    B.clear()
    A.pop()
    gc.collect()
    assert all(r() is not None for r in alive)
    assert ad._A.tolist() == at[0] and ad._B.tolist() == at[1]
    del ad
    gc.collect()
    assert alive[1]() is None and alive[2]() is None and alive[3]() is None


def test_adapters_hold_what_they_were_made_of(anywhere):
    """attributes given other tensors, or none: the addresses taken stay those of tensors that live"""
    A, B, scale = bf(3, 8, 16), bf(3, 5, 8), torch.ones(3)
    alive = [weakref.ref(m) for m in (A, B, scale)]
    ad = moe.Adapters(A, B, scale)
    a, b, s = A.data_ptr(), B.data_ptr(), scale.data_ptr()
    del A, B, scale
    ad.A = ad.B = ad.scale = None
    gc.collect()
    assert all(r() is not None for r in alive) and (ad._a, ad._b, ad._scale) == (a, b, s)


@pytest.mark.parametrize("n, G", [(2 ** 31, 3), (2 ** 32 + 5, 3), (5, 2 ** 31), (5, 2 ** 32 + 3)])
def test_groups_past_32_bits(n, G):
    """the library's n and n_groups are 32-bit integers, which would cut these to other sizes"""
    with pytest.raises(ValueError, match="more than 2147483647"):
        moe.RowGroups(n, G, device="meta")


def test_adapters_past_32_bits(anywhere):
    """so are rank, n_in, n_out"""
    meta = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="meta")
    for A, B in ((meta(1, 8, 2 ** 32 + 8), meta(1, 5, 8)), (meta(1, 8, 16), meta(1, 2 ** 32 + 5, 8)), (meta(1, 2 ** 32 + 8, 16), meta(1, 5, 2 ** 32 + 8)),
                 (meta(2 ** 32 + 1, 8, 16), meta(2 ** 32 + 1, 5, 8))):
        with pytest.raises(ValueError, match="more than 2147483647"):
            moe.Adapters(A, B)


@pytest.mark.parametrize("flat", [False, True])
def test_picks_past_32_bits(monkeypatch, flat):
    """and K, in both of the ways that a call's tensors are looked at"""
    monkeypatch.setattr(moe, "_current", lambda: -1)   # the place of the tensors below
    monkeypatch.setattr(moe, "_st", lambda: None)
    monkeypatch.setattr(moe, "lib", lambda: pytest.fail("passed on"))
    K = 2 ** 32 + 3
    f = lambda *s: torch.empty(s, device="meta")
    pos = torch.empty((K,) if flat else (1, K), dtype=torch.int32, device="meta")
    w, x, rows = f(1, K), f(1, 8), f(4, 8)
    for call in (lambda: moe.moe_sort_rows(x, pos, rows), lambda: moe.moe_sort_rows_backward(rows, pos, x), lambda: moe.moe_combine_sorted(rows, w, pos, x),
                 lambda: moe.moe_combine_sorted_backward(x, rows, w, pos, None, w)):
        with pytest.raises(ValueError, match="more than 2147483647"):
            call()
