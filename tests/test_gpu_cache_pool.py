"""Sequences of a page pool are named from 0 on: anything else is refused and changes nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_sequences_out_of_range_are_refused(device):
    from dgl_amd.attention import PagedCache
    cache = PagedCache(3, 1, 16, 64, page_size=16, num_pages=6, device=device)
    cache.reserve(2, 20)
    x = torch.randn(3, 1, 20, 16, device=device)
    cache.append(x, x)
    table, lengths = cache.table.clone(), cache.lengths.clone()
    for sequence in (-1, -3, 3, 100):
        with pytest.raises(ValueError, match="sequence"):
            cache.release(sequence)
        with pytest.raises(ValueError, match="sequence"):
            cache.reserve(sequence, 33)
    assert torch.equal(cache.table, table) and torch.equal(cache.lengths, lengths)
    cache.release(2)
    assert cache.lengths.tolist() == [20, 20, 0] and int(cache.table[2].max()) == -1
    cache.reserve(0, 64)
    cache.reserve(1, 32)                                  # all six pages are free again
