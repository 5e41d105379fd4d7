"""Sizes that the library's 32-bit integers would cut, on a host without a GPU."""
import pytest
import torch

from sfnx_amd import moe


@pytest.fixture
def anywhere(monkeypatch):
    """tensors are taken where they are"""
    monkeypatch.setattr(moe, "_need", lambda *a, **k: None)


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
