"""Shards of many adapters' factors: every column of B and row of A is in exactly one of them, or the split is refused."""

import pytest
import torch

from qextract_infer_b200.tp_shard import shard_adapters


@pytest.mark.parametrize("world", [1, 2, 3, 4])
def test_shards_cover_the_factors(world):
    A, B = torch.randn(2, 48 * world, 16), torch.randn(2, 16, 24 * world)
    cols = [shard_adapters(A, B, "col", r, world) for r in range(world)]
    assert all(a is A for a, _ in cols) and torch.equal(torch.cat([b for _, b in cols], 2), B)
    rows = [shard_adapters(A, B, "row", r, world) for r in range(world)]
    assert all(b is B for _, b in rows) and torch.equal(torch.cat([a for a, _ in rows], 1), A)


@pytest.mark.parametrize("split,k,n", [("col", 64, 64), ("col", 48, 40), ("row", 64, 48), ("row", 40, 48)])
def test_uneven_splits_are_refused(split, k, n):
    """as those of the quantised linear beside them; the rest of the columns or rows was left out"""
    with pytest.raises(ValueError, match="needs"):
        shard_adapters(torch.zeros(1, k, 8), torch.zeros(1, 8, n), split, 0, 3)
    with pytest.raises(ValueError, match="unknown split"):
        shard_adapters(torch.zeros(1, 48, 8), torch.zeros(1, 8, 48), "both", 0, 2)
