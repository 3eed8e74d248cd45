"""Which tensors describe a paged cache (meta tensors: nothing is launched)."""
import pytest
import torch

import qe_amd as qe


def _pages(*shape):
    return torch.zeros(shape, dtype=torch.float16, device="meta")


def test_pages_that_lie_over_each_other():
    """One page seen as many (a stride of 0, which the library takes for pages behind each other)."""
    for one in (_pages(1, 2, 16, 128).expand(8, 2, 16, 128), _pages(9, 2, 16, 128).as_strided((8, 2, 16, 128), (2048, 2048, 128, 1))):
        for k, v in ((one, one), (one, _pages(8, 2, 16, 128)), (_pages(8, 2, 16, 128), one)):
            with pytest.raises(RuntimeError, match="strides"):
                qe.paged_cache(k, v)


def test_one_head_whatever_its_stride():
    """Pages of one head are the same memory in either order of heads and rows: what stops these is that they are on no GPU."""
    for one in (_pages(8, 16, 1, 128).transpose(1, 2), _pages(8, 2, 16, 128)[:, 1:], _pages(8, 1, 16, 128)):
        with pytest.raises(RuntimeError, match="must be on a GPU"):
            qe.paged_cache(one, one)
    with pytest.raises(RuntimeError, match="strides"):
        qe.paged_cache(*[_pages(8, 16, 2, 128).transpose(1, 2)] * 2)
