"""LowRankAdapters.from_pairs refuses pairs whose ranks differ, before it lays anything out."""
import pytest
import torch

from netra_moe.adapters import LowRankAdapters


@pytest.mark.parametrize("shapes", [
    [((8, 6), (5, 8)), ((4, 6), (5, 6))], [((8, 6), (5, 8)), ((4, 6), (5, 3))], [((4, 6), (5, 8))], [((4, 6), (5, 2))],
    [((4, 6), (4,))], [((1, 4, 6), (5, 4))]])
def test_ranks_that_differ(shapes):
    with pytest.raises(ValueError, match=r"pairs\[\d\]: need a \[r, K\] and b \[N, r\]"):
        LowRankAdapters.from_pairs([(torch.zeros(a), torch.zeros(b)) for a, b in shapes])
