"""Edges of serving sequences of different lengths that need no GPU: the cache's bookkeeping."""
import pytest
import torch

from smlm_hip.paged import PagedKVCache


def test_a_cache_made_in_inference_mode_is_written_outside_of_it():
    with torch.inference_mode():
        c = PagedKVCache(1, 2, 40, 1, 32, 16, device="cpu")
        c.reserve([3, 0])
    c.advance([3, 0])
    c.reserve([1, 20])
    assert c.lengths.tolist() == [3, 0] and c.block_table[1, 1] >= 0
    c.clear()
    assert not c.layers[0].pages[0].is_inference() and not c.block_table.is_inference()


@pytest.mark.parametrize("size", [0, -16, 8, 24, 8192])
def test_page_sizes_that_there_are_not(size):
    with pytest.raises(ValueError, match="pages of"):
        PagedKVCache(1, 2, 40, 1, 32, size, device="cpu")
