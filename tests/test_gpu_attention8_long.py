"""Evictions that several wavefronts' registers or several workgroups share, and weights that a second launch adds up: tables that miss
pages, weights that are all alike or not finite, positions that are all the latest."""
import math

import pytest
import torch

import attention8_evictions as whole_heads
import attention8_reference as ref8
from test_gpu_attention8 import DEV, MAXINT, attend_and_check, filled, queries_for, weigh_at_random, whole
from vectorlink_gpu import _native as nv
from vectorlink_gpu import attention

pytestmark = pytest.mark.gpu


def parts_of(cache, table, lengths, q):
    """Bytes of the parts that a call's workgroups leave to be joined."""
    (tokens, queries) = (attention._tokens(q.size(0), table, lengths, None), attention._queries(q, cache, None, True, None, None))
    return nv.lib().vl_attend8_workspace_bytes(cache._ref, tokens, queries, 0)


@pytest.mark.parametrize("group", [1, 4, 5, 7, 8, 9, 16])
@pytest.mark.parametrize("dim, dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.float32)])
def test_scores_that_a_second_launch_adds_up(group, dim, dtype):
    """Single tokens over contexts that several workgroups share: ends inside a piece of 2,048 places and a word of four, pages that miss."""
    cache, table, lengths, gen = filled([5_003, 4_097, 70, 0, 2_048], 1, dim, group + dim, dtype, blocks=81)
    table[0, 5] = -1
    table[0, 33:36] = MAXINT
    table[0, 78] = cache.pages  # the last
    table[1, 64] = -7           # of one token
    q = queries_for(5, group, dim, gen, dtype)
    assert parts_of(cache, table, lengths, q) > 0
    attend_and_check(cache, table, lengths, q)


def evict_and_check(cache, table, lengths, keep, recent):
    model = ref8.Model(cache)
    was = lengths.clone()
    left = cache.evict(table, lengths, keep, recent)
    assert torch.equal(was, lengths)
    assert left.tolist() == whole_heads.evict(model, table, lengths, keep, recent)
    model.check(cache)
    return left


def miss_pages(table, lengths, keep):
    """Of the first sequence pages in front, where the new length ends and behind it; of the last all but two."""
    border = keep // 64
    table[0, 1] = -1
    table[0, border] = MAXINT
    table[0, min(border + 3, table.size(1) - 1)] = -1
    table[0, -(-int(lengths[0]) // 64) - 1] = -1  # the last
    last = table.size(0) - 1
    kept = table[last, [0, 9]].clone()
    table[last] = -1
    (table[last, 0], table[last, 9]) = kept.tolist()


@pytest.mark.parametrize("weights", ["random", "ties", "alike", "odd", "nan"])
@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("longest, keep, recent", [(9_000, 5_003, 100), (20_011, 64 * 128, 500), (32_768, 32_700, 0), (33_000, 1_000, 1_000),
                                                   (40_000, 16_384, 512), (70_001, 69_990, 64)])
def test_long_evictions(longest, keep, recent, weights, missing):
    """More than 128 blocks are a workgroup's of 16 wavefronts, more than 512 several workgroups'."""
    lengths = [longest, longest - 3_333 if longest > 8_000 else 10, 50, keep + 1, min(longest, 10_000)]
    cache, table, held, gen = filled(lengths, 2, 32, longest + keep)
    (k, v) = torch.randn((2, 5 * 30, 2, 32), generator=gen, device=DEV) * 10.0 ** torch.randint(-2, 5, (2, 5 * 30, 2, 1), generator=gen, device=DEV)
    (k[3, 0, 5], v[70, 1, 7]) = (math.nan, math.inf)
    cache.write(k, v, table, held - 30, whole(0, 30, 60, 90, 120, 150))  # tokens whose powers others need
    weigh_at_random(cache, gen, ties=weights == "ties")
    if weights == "alike":
        cache.weights.fill_(0.0)
        cache.positions[:, 1] = 7  # all are the latest
    if weights == "odd":
        odd = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, -1.0, -0.0, 0.0, 1e-40, 3.0], device=DEV)
        cache.weights.copy_(odd[torch.randint(0, 9, cache.weights.shape, generator=gen, device=DEV)])
    if weights == "nan":
        cache.weights.fill_(math.nan)
    if missing:
        miss_pages(table, held, keep)
    left = evict_and_check(cache, table, held, keep, recent)
    if missing:
        assert int(left[4]) == (min(keep, 128) if lengths[4] > keep else lengths[4])  # 128 of its tokens are on pages
    # a second time, from what the first left
    cache.weights[:, :, 3::5] += 1
    evict_and_check(cache, table, left, keep * 2 // 3, recent // 2)


@pytest.mark.parametrize("longest, keep", [(20_000, 0), (40_000, 0), (40_000, 1), (70_001, 70_000), (33_000, 33_000)])
def test_long_evictions_of_all_or_of_one(longest, keep):
    cache, table, held, gen = filled([longest, 5, longest - 1], 1, 32, keep)
    weigh_at_random(cache, gen)
    evict_and_check(cache, table, held, keep, min(keep, 1))
    table[0] = -1
    assert cache.evict(table, held, min(keep, 4), 0).tolist() == [0, min(keep, 4), min(keep, 4)]


def test_a_table_that_only_names_many_blocks():
    """Short sequences under a table of 600 blocks take the way of several workgroups."""
    cache, table, held, gen = filled([300, 0, 64, 65, 129], 3, 64, 3)
    wide = torch.full((5, 600), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    weigh_at_random(cache, gen)
    evict_and_check(cache, wide, held, 64, 7)
