"""The choice of blocks for scores that a negative scale is multiplied with."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import TYPES, ends, filled, queries_for
from vectorlink_gpu import attend_selected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,group,blocks", [(1, 4, None), (150, 3, None), (140, 20, None), (1, 2, 16_000)])
def test_a_negative_scale_turns_the_choice(rows, group, blocks, dtype):
    """scale <query, key> of the negated queries is what is chosen by: both calls are the same attention."""
    (cache, table, lengths, gen) = filled([1500, 700], 2, 64, 53, dtype, blocks=blocks)
    at = ends([rows, 1])
    q = queries_for(rows + 1, 2 * group, 64, gen, dtype)
    (out, blocks) = attend_selected(q, cache, table, lengths, 4, offsets=at, scale=-0.2)
    assert torch.equal(blocks.cpu(), ref.selection(-q, cache, table, lengths, 4, at))
    ref.check_attention(out, ref.attention(q, cache, table, lengths, at, scale=-0.2, blocks=blocks.cpu()), dtype)
    (same, blocks2) = attend_selected(-q, cache, table, lengths, 4, offsets=at, scale=0.2)
    assert torch.equal(blocks, blocks2) and torch.equal(out, same)
