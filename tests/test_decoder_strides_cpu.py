"""What the decoder operators hand to their kernels: strides that are multiples of 16 bytes, whatever a dimension of one element
came with, and no copy where the layout can be read in place."""
import pytest
import torch

from configurable_hierarchical_allreduce_algorithms_b200.ops import decoder


@pytest.mark.parametrize("shape,strides", [((1, 4, 64), (259, 64, 1)), ((5, 1, 64), (64, 3, 1)), ((1, 1, 8), (1, 1, 1)),
                                           ((1, 4, 64), (256, 67, 1)), ((6, 1, 64), (67, 3, 1)), ((6, 4, 64), (0, 64, 1))])
def test_heads(shape, strides):
    t = torch.randn(2000).bfloat16().as_strided(shape, strides)
    got = decoder._heads(t)
    st, sh, one = got.stride()
    assert one == 1 and st % 8 == 0 and sh % 8 == 0 and st and sh and torch.equal(got, t)


def test_rows():
    for t in (torch.randn(1, 75).bfloat16()[:, :72], torch.randn(1, 72).bfloat16().expand(4, 72), torch.randn(4, 75).bfloat16()[:, :72]):
        got = decoder._rows(t)
        assert got.stride(0) % 8 == 0 and got.stride(0) >= 72 and got.stride(1) == 1 and torch.equal(got, t)


def test_read_in_place():
    rows = torch.randn(6, 3 * 128).bfloat16()
    for t in rows.split(128, 1):
        assert decoder._rows(t).data_ptr() == t.data_ptr()
        assert decoder._heads(t.view(6, 2, 64)).data_ptr() == t.data_ptr()
    one = rows[:1, :128].view(1, 2, 64)
    assert decoder._heads(one.as_strided((1, 2, 64), (131, 64, 1))).data_ptr() == one.data_ptr()
