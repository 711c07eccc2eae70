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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("larger", [0, 1])
@pytest.mark.parametrize("blocks", [2, 900])
def test_a_scale_times_a_power_beyond_float32(dtype, larger, blocks):
    """Two pages whose powers are 2^119 and 2^115 under a scale of 2^12, which makes factors of 2^131 and 2^127 of their codes: products
    of 2^-16 and 2^-14 are scores of 2^115 and 2^113, and the first has all weight."""
    cache = KVCache8.empty(2, 1, 64, weighted=True)
    cache.weights.zero_()
    keys = torch.zeros((128, 1, 64), device=DEV)
    for block, code, power in ((larger, 2.0 ** -6, 2.0 ** 119), (1 - larger, 2.0 ** -4, 2.0 ** 115)):
        keys[block * 64 + 9, 0, 3] = code * power
        keys[block * 64 + 20, 0, 5] = 448 * power  # which no query looks at
    gen = torch.Generator(device=DEV).manual_seed(3)
    table = whole(1, 0)[None]
    cache.write(keys, torch.randn((128, 1, 64), generator=gen, device=DEV), table, whole(0), ends([128]))
    assert sorted(cache.scales[:, 0, 0].tolist()) == [115 + 127, 119 + 127]
    at = larger * 64 + 9
    value = cache.read(table, whole(at), 1, dtype=torch.float32)[1][0, 0]
    for rows, form in [(40, f) for f in forms_of(64, dtype)] + [(1, None)]:
        q = torch.zeros((rows, 4, 64), device=DEV, dtype=dtype)
        q[..., 3] = 2.0 ** -10
        cache.weights.zero_()
        (out, lse) = attend(q, cache, wide(table, blocks), whole(128), None if rows == 1 else ends([rows]), scale=2.0 ** 12, causal=False,
                            return_lse=True, form=form, accumulate=True)
        assert torch.equal(out, value.to(dtype).expand_as(out))  # one weight of 1: what the cache holds, rounded
        assert bool((lse.double() / 2.0 ** 115 - 1).abs().max() < 2.0 ** -22)
        want = torch.zeros_like(cache.weights)
        want[table[0, larger].long(), 0, 9] = 4 * rows
        assert torch.equal(cache.weights, want)
