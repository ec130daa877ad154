"""Refusals of page bounds that come where the cache is made, without a GPU."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("D", [16, 80, 96, 112])
def test_bounds_of_a_head_size_that_has_none(D):
    """A cache whose append could not keep its bounds is refused when it is made, not after a step has
    written its keys and values."""
    from pallas_flash.kernels import paged
    with pytest.raises(ValueError, match="head size"):
        paged.DevicePagedKVCache(2, 2, D, num_pages=4, page_size=16, max_seq_len=32, bounds=True, device="cpu")
    with pytest.raises(ValueError, match="head size"):
        paged.empty_bounds(torch.zeros((4, 2, 16, D), dtype=torch.bfloat16))
    assert paged.DevicePagedKVCache(2, 2, D, num_pages=4, page_size=16, max_seq_len=32, device="cpu").bounds is None
