"""The choice of blocks over contexts of hundreds to thousands of blocks: scores that no longer fit a wavefront's registers or a
workgroup's share of LDS.  Tables name few pages many times, so most scores are ties, which go to the lower block."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, MAXINT, ends, filled, queries_for
from vectorlink_gpu import _native as nv
from vectorlink_gpu import attend_blocks, attend_selected, attention, select_blocks

pytestmark = pytest.mark.gpu


def repeated(sequences, blocks, heads, dim, seed, pages=50, dtype=torch.bfloat16, holes=True):
    """A table [sequences, blocks] over `pages` full pages in any order; some entries name no page."""
    (cache, _, _, gen) = filled([64] * pages, heads, dim, seed, dtype, spare=0)
    table = torch.randint(0, pages, (sequences, blocks), generator=gen, device=DEV, dtype=torch.int32)
    if holes:
        table[torch.rand(table.shape, generator=gen, device=DEV) < 0.01] = -1
    return cache, table, gen


def selection(queries, cache, table, lengths, count, offsets):
    """attention_reference.selection, all blocks of a row at once"""
    q = queries.cpu().double()
    group = q.size(1) // cache.heads
    (table, lengths, offsets) = (table.cpu().long(), lengths.tolist(), offsets.tolist())
    out = torch.full((q.size(0), cache.heads, count), MAXINT, dtype=torch.int64)
    (edges, powers) = (cache.bounds.cpu().double(), torch.exp2(cache.bound_scales.cpu().double()))
    for b in range(table.size(0)):
        real = (table[b] >= 0) & (table[b] < cache.pages)
        page = table[b].clamp(0, cache.pages - 1)
        for row in range(offsets[b], offsets[b + 1]):
            place = lengths[b] - (offsets[b + 1] - offsets[b]) + row - offsets[b]
            own = min(place, table.size(1) * 64 - 1) // 64
            if place < 0:
                continue
            for h in range(cache.heads):
                u = q[row, h * group:(h + 1) * group]
                e = torch.frexp(u.abs().max()).exponent.double() - 7
                u = torch.clamp(torch.round(u * torch.exp2(-e)), -127, 127)
                of_page = ((u.clamp(min=0) @ edges[:, h, 0].T.contiguous() + u.clamp(max=0) @ edges[:, h, 1].T.contiguous()).amax(0) * powers[:, h])
                score = torch.where(real, of_page[page], -torch.inf)[:own + 1]
                score[own] = torch.inf
                best = torch.sort(score, descending=True, stable=True)
                ids = best.indices[:count][best.values[:count] > -torch.inf]
                out[row, h, :len(ids)] = ids.sort().values
    return out.to(torch.int32)


# (blocks, group, rows of each sequence): tokens that share a workgroup are fewer than fit a tile from 896 blocks with one query a
# head on; 800 x 16 and 3,200 x 4 scores are 51 KB of LDS
RAGGED = [(600, 1, [40, 3, 17]), (800, 1, [33, 70]), (900, 1, [40, 3, 17]), (1000, 1, [30, 1, 30]), (1000, 5, [20, 9]), (640, 16, [5, 30]),
          (3200, 4, [70, 60]), (3500, 4, [70, 60]), (14_000, 1, [130]), (700, 20, [9, 2])]


@pytest.mark.parametrize("blocks,group,counts", RAGGED)
def test_rows_of_prompts(blocks, group, counts):
    heads = 2
    (cache, table, gen) = repeated(len(counts), blocks, heads, 64, blocks + group)
    lengths = torch.tensor([blocks * 64 - 7 - 900 * i for i in range(len(counts))], dtype=torch.int32, device=DEV)
    q = queries_for(sum(counts), heads * group, 64, gen, torch.bfloat16)
    for count in (1, 4, 77, 600):
        got = select_blocks(q, cache, table, lengths, count, ends(counts))
        assert torch.equal(got.cpu(), selection(q, cache, table, lengths, count, ends(counts))), count


@pytest.mark.parametrize("blocks,counts", [(1025, [9, 2]), (4090, [1, 1]), (4097, [1]), (5000, [3, 1, 2]), (20_000, [2])])
def test_few_rows_over_many_blocks(blocks, counts):
    """Scores in the workspace, chosen from by 8 wavefronts together: 4,096 of them fit registers."""
    (cache, table, gen) = repeated(len(counts), blocks, 1, 32, blocks)
    lengths = torch.tensor([blocks * 64 - 3 - 64 * 40 * i for i in range(len(counts))], dtype=torch.int32, device=DEV)
    q = queries_for(sum(counts), 3, 32, gen, torch.float16)
    for count in (1, 32, 500, 4096):
        got = select_blocks(q, cache, table, lengths, count, ends(counts))
        assert torch.equal(got.cpu(), selection(q, cache, table, lengths, count, ends(counts))), count


@pytest.mark.parametrize("blocks,count", [(600, 40), (4097, 32), (6000, 5), (16_384, 1024)])
def test_in_one_launch(blocks, count):
    """64 rows and heads: a workgroup for each scores, chooses and attends."""
    counts = [30, 2]
    (cache, table, gen) = repeated(2, blocks, 2, 32, blocks)
    lengths = torch.tensor([blocks * 64 - 5, blocks * 64 - 1999], dtype=torch.int32, device=DEV)
    q = queries_for(32, 4, 32, gen, torch.bfloat16)
    at = ends(counts)
    need = nv.lib().vl_attend_selected_workspace_bytes(cache._ref, attention._tokens(32, table, lengths, at),
                                                       attention._queries(q, cache, None, True, None, None), count)
    assert need == 0
    (out, got) = attend_selected(q, cache, table, lengths, count, offsets=at)
    assert torch.equal(got.cpu(), selection(q, cache, table, lengths, count, at))
    # what it attends to is checked elsewhere: the call of its own over the same lists differs by the order of sums, which may move a
    # rounding of the result by its unit
    apart = attend_blocks(q, cache, table, lengths, got, offsets=at).double()
    assert ((out.double() - apart).abs() <= 2.0 ** -7 * apart.abs() + 2.0 ** -16).all()
