"""Attention over the cache in 8 bits and the weights of its tokens where scores, scales and powers are next to nothing or next to
everything."""
import math

import pytest
import torch

from test_gpu_attention8 import DEV, MAXINT, TYPES, attend_and_check, ends, filled, forms_of, queries_for, whole
from vectorlink_gpu import KVCache8, attend

pytestmark = pytest.mark.gpu


def wide(table, blocks):
    """The table with so many blocks more that four pages are a workgroup's where weights are made from the keys."""
    out = torch.full((table.size(0), blocks), -1, dtype=torch.int32, device=DEV)
    out[:, :table.size(1)] = table
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("blocks", [3, 600])
def test_no_scale_leaves_tokens_alike_whatever_their_products(dtype, blocks):
    """Products of queries and keys leave float32, and every token gets the same weight all the same."""
    cache, table, lengths, gen = filled([150, 64], 2, 64, 91, torch.float32)
    x = 1e30 * torch.randn((2, 214, 2, 64), generator=gen, device=DEV)
    cache.write(x[0], x[1] * 1e-30, table, whole(0, 0), ends([150, 64]))
    q = queries_for(49, 4, 64, gen, dtype, 1e4 if dtype == torch.float16 else 1e30)
    for form in forms_of(64, dtype):
        attend_and_check(cache, wide(table, blocks), lengths, q, ends([40, 9]), scale=0.0, form=form)
    attend_and_check(cache, wide(table, blocks), lengths, q[:2], scale=0.0)
