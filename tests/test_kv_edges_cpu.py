"""Edges of the rotary norm, the paged 8-bit cache and its attention that need no GPU."""
import pytest
import torch

from primus_dlrm_b200.ops.kv_cache import PagedKVCache


def test_copy_pages_outside_the_pool():
    c = PagedKVCache(4, 1, 32, 16)
    c.k_scale.copy_(torch.arange(4.0)[:, None] + 1)
    for src, dst in (([-1], [0]), ([0], [-1]), ([4], [0]), ([0], [4])):
        with pytest.raises(IndexError):
            c.copy_pages(torch.tensor(src), torch.tensor(dst))
    assert c.k_scale.flatten().tolist() == [1, 2, 3, 4]
    c.copy_pages(torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32))
    assert c.k_scale.flatten().tolist() == [2, 1, 3, 4]
