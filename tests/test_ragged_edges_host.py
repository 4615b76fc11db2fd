"""Edges of serving sequences of different lengths that need no GPU: the cache's bookkeeping, the split walks' workspaces."""
import pytest
import torch

from smlm_hip import _lib
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


def test_walks_of_batches_that_fill_the_gpu_are_not_split():
    """2,304 workgroups (sequences times groups of up to 16 query heads) of eight or more sequences, 768 of fewer, take no workspace
    however long the table; one sequence less takes some for every head."""
    need = lambda B, H, Hk, most: _lib.lib().smlm_paged_attention_workspace(B, H, Hk, 64, 64, most)  # noqa: E731
    for most in (17, 2048, 100_000):
        assert need(384, 6, 6, most) == need(2304, 1, 1, most) == need(1152, 32, 1, most) == need(7, 110, 110, most) == 0
        for B, H, Hk in ((383, 6, 6), (2303, 1, 1), (1151, 32, 1), (7, 109, 109)):
            assert need(B, H, Hk, most) == B * H * 2 * (64 + 2) * 4
    assert need(1, 1, 1, 16) == 0 and need(1, 1, 1, 4) == 0            # 1,024 tokens and fewer are one workgroup's
    assert need(1, 1, 1, 1 << 24) == 256 * (64 + 2) * 4                # the most splits
