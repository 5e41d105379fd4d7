"""MoeLayerF8.store: values and scales as model files hold them, laid out as the 8-bit store; on the CPU."""
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403


@pytest.mark.parametrize("n, rows, cols", [(1, 1, 16), (3, 130, 144), (2, 256, 384), (2, 129, 16)])
def test_store_lays_out_values_then_scales(n, rows, cols):
    """against the layout read back value by value: e4m3 codes row-major, the f32 scales after them, padding of zeros"""
    g = torch.Generator().manual_seed(rows)
    q = (torch.randn((n, rows, cols), generator=g) * 100).clamp(-F8_MAX, F8_MAX).to(F8)
    s = torch.rand((n, nb(rows), nb(cols)), generator=g)
    for form in (q, q.view(torch.uint8)):
        out = moe.MoeLayerF8.store(form, s)
        assert out.dtype == torch.uint8 and out.shape == (n, moe.f8_matrix_bytes(rows, cols)) and out.is_contiguous()
        at = rows * cols
        assert torch.equal(out[:, :at], q.view(torch.uint8).reshape(n, at))
        assert torch.equal(out[:, at: at + 4 * nb(rows) * nb(cols)].contiguous().view(torch.float32).view(s.shape), s)
        assert (out[:, at + 4 * nb(rows) * nb(cols):] == 0).all()


def test_store_of_strided_values_and_scales():
    """transposed and sliced tensors, as a loader that splits or reorders matrices hands them over"""
    g = torch.Generator().manual_seed(5)
    q = (torch.randn((2, 144, 130), generator=g) * 100).clamp(-F8_MAX, F8_MAX).to(F8)
    s = torch.rand((2, 2, 2), generator=g)
    qt, st = q.transpose(1, 2), s.transpose(1, 2)
    assert not qt.is_contiguous() and not st.is_contiguous()
    assert torch.equal(moe.MoeLayerF8.store(qt, st), moe.MoeLayerF8.store(qt.contiguous(), st.contiguous()))


@pytest.mark.parametrize("q, s", [(torch.zeros((1, 130, 144)), torch.zeros((1, 2, 2))),
                                  (torch.zeros((1, 130, 144), dtype=torch.uint8), torch.zeros((1, 2, 2), dtype=torch.float64)),
                                  (torch.zeros((1, 130, 144), dtype=torch.uint8), torch.zeros((1, 1, 2))),
                                  (torch.zeros((2, 130, 144), dtype=torch.uint8), torch.zeros((1, 2, 2)))])
def test_store_refuses(q, s):
    """values that are no codes, scales of another type, block count or matrix count"""
    with pytest.raises(ValueError, match="store:"):
        moe.MoeLayerF8.store(q, s)
