"""Scores of blocks at the ends of what they can be."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, ends, filled, queries_for
from vectorlink_gpu import attend_selected, select_blocks

pytestmark = pytest.mark.gpu


# one token a tile, several, and scores in the workspace
@pytest.mark.parametrize("rows,blocks", [(2, None), (150, None), (2, 1100)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("far", [110, 121, -100, -121])
def test_scores_of_any_size(far, dim, rows, blocks):
    """Keys whose powers of two lie 2^far from 1: products with their bounds pass the range of float32 (above 2^128), or lie below
    what it holds with all bits.  Neighbouring pages differ by little, and by much."""
    lengths = [1500, 700]
    (cache, table, lengths, gen) = filled(lengths, 1, dim, 51, torch.float32, blocks=blocks)
    pages = cache.bound_scales.size(0)
    # the bounds alone are looked at: they are made larger, some by one power more
    cache.bound_scales += far
    cache.bound_scales += torch.randint(0, 3, (pages, 1), generator=gen, device=DEV, dtype=torch.int8)
    real = table[table >= 0].long()
    cache.bound_scales[real] = cache.bound_scales[real].clamp(-126, 121)
    at = ends([rows - 1, 1])
    q = queries_for(rows, 3, dim, gen, torch.float32)
    q[::2] *= -1
    for count in (2, 7):
        assert torch.equal(select_blocks(q, cache, table, lengths, count, at).cpu(), ref.selection(q, cache, table, lengths, count, at)), count
    if rows == 2:  # scores, choice and attention in one launch
        assert torch.equal(attend_selected(q, cache, table, lengths, 3, offsets=at)[1].cpu(), ref.selection(q, cache, table, lengths, 3, at))
