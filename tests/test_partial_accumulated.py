"""Rows of accumulated weights that share memory would be added to by several workgroups at once: refused, no GPU needed.  Rows in any order, with or without
gaps, are taken."""
import pytest
import torch

from aitherkvcache_amd.eviction import weights_for

FLAT = torch.zeros(8192)


@pytest.mark.parametrize("shape,strides", [((2, 2, 32), (64, 16, 1)), ((2, 2, 32), (40, 32, 1)), ((2, 2, 32), (1, 64, 1)), ((2, 2, 32), (64, 31, 1)), ((3, 2, 40), (40, 100, 1)),
                                           ((2, 2, 32), (1, 1, 1)), ((2, 2, 32), (0, 32, 1)), ((2, 2, 32), (32, 0, 1)), ((2, 1, 32), (31, 4000, 1))])
def test_rows_that_share_memory_are_refused(shape, strides):
    with pytest.raises(ValueError, match="share memory"):
        weights_for(FLAT.as_strided(shape, strides), 2, shape[1], 32, "cpu")


@pytest.mark.parametrize("shape,strides", [((2, 2, 32), (64, 32, 1)), ((2, 2, 32), (32, 64, 1)), ((2, 2, 32), (100, 40, 1)), ((3, 2, 40), (40, 120, 1)), ((1, 2, 32), (0, 32, 1)),
                                           ((2, 1, 32), (32, 1, 1)), ((1, 1, 32), (0, 0, 1))])
def test_rows_apart_are_taken(shape, strides):
    given = FLAT.as_strided(shape, strides)
    assert weights_for(given, 1, shape[1], 32, "cpu") is given
