"""Scores far beyond what float32 holds to the unit: a row's largest has all weight, whatever is lost of the scores."""
import math

import pytest
import torch

from test_gpu_attention import TYPES, DEV, ends, queries_for
from vectorlink_gpu import KVCache, KVCache8, attend, attend_blocks

pytestmark = pytest.mark.gpu
LENGTHS = [130, 1, 300, 64]


def filled(kind, key_size, gen):
    blocks = 5
    cache = KVCache8.empty(4 * blocks, 2, 64, weighted=True) if kind == 8 else KVCache.empty(4 * blocks, 2, 64)
    table = torch.randperm(4 * blocks, generator=gen, device=DEV).view(4, blocks).to(torch.int32)
    x = torch.randn((2, sum(LENGTHS), 2, 64), generator=gen, device=DEV)
    zeros = torch.zeros(4, dtype=torch.int32, device=DEV)
    cache.write(x[0] * key_size, x[1], table, zeros, ends(LENGTHS))
    (k, v) = cache.read(table, zeros, sum(LENGTHS), ends(LENGTHS), dtype=torch.float32)
    return cache, table, torch.tensor(LENGTHS, dtype=torch.int32, device=DEV), k.cpu().double(), v.cpu()


def expected(q, k, v, counts, scale, causal):
    """Of every row and head of the queries: the least and the largest that an output may be, the place of the token that has all weight
    (-1: none, -2: it cannot be told), the largest score, and what float32 may lose of a score.

    A score is a sum of 64 products, each rounded at most three times in parts, so it is off by less than 200 half steps of the sum of
    their magnitudes.  A token whose score is below the largest by twice that and 200 more has no weight: e^-200 is no float32.
    What is left are values between the least and the largest of the tokens that are as near, most often one's."""
    (rows, heads, dim) = q.shape
    q = q.cpu().double()
    (low, high) = (torch.zeros(q.shape), torch.zeros(q.shape))
    best = torch.full((rows, heads), -1)
    (score, lost) = (torch.full((rows, heads), -math.inf, dtype=torch.float64), torch.zeros((rows, heads), dtype=torch.float64))
    (row, token) = (0, 0)
    for n, count in zip(LENGTHS, counts):
        for i in range(count):
            sees = min(max(n - count + i + 1, 0), n) if causal else n
            for g in range(heads if sees else 0):
                (keys, values) = (x[token:token + sees, g // (heads // 2)] for x in (k, v))
                s = keys @ q[row + i, g] * scale
                off = 200 * 2.0 ** -24 * float((keys.abs() @ q[row + i, g].abs()).max()) * abs(scale)
                near = s >= s.max() - 2 * off - 200
                (score[row + i, g], lost[row + i, g]) = (s.max(), off)
                best[row + i, g] = int(s.argmax()) if int(near.sum()) == 1 else -2
                (low[row + i, g], high[row + i, g]) = (values[near].amin(0), values[near].amax(0))
        (row, token) = (row + count, token + n)
    assert bool((best >= 0).sum() > 0.8 * (best != -1).sum())
    return low, high, best, score, lost


@pytest.mark.parametrize("kind", [4, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size, scale", [(1e6, 1.0), (1e6, -3.0), (1e14, 1e-2), (1e2, 1e9)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [5, 2, 9, 3]])
@pytest.mark.parametrize("form", ["few", "many"])
def test_the_largest_has_all(kind, dtype, size, scale, counts, form):
    gen = torch.Generator(device=DEV).manual_seed(5)
    (cache, table, lengths, k, v) = filled(kind, size, gen)
    q = queries_for(sum(counts), 8, 64, gen, dtype, min(size, 6e3) if dtype == torch.float16 else size)
    for causal in (True, False):
        (low, high, best, score, lost) = expected(q, k, v, counts, scale, causal)
        seen = best != -1
        assert float(score[seen].abs().max()) > 2.0 ** 33
        offsets = None if counts == [1, 1, 1, 1] and form == "few" else ends(counts)

        def check(out):
            out = out.cpu()
            assert bool(((out >= low.to(dtype)) & (out <= high.to(dtype))).all())

        (out, lse) = attend(q, cache, table, lengths, offsets, scale=scale, causal=causal, return_lse=True, form=form)
        check(out)
        lse = lse.cpu().double()
        assert torch.equal(lse == -math.inf, ~seen)
        assert bool(((lse - score).abs() <= lost + 2.0 ** -22 * score.abs() + 6)[seen].all())  # 6: the logarithm of 300
        if kind == 4 and causal:
            blocks = torch.arange(5, dtype=torch.int32, device=DEV).expand(sum(counts), 2, 5).contiguous()
            check(attend_blocks(q, cache, table, lengths, blocks, offsets, scale=scale))
        if kind == 8:
            cache.weights.zero_()
            assert torch.equal(attend(q, cache, table, lengths, offsets, scale=scale, causal=causal, form=form, accumulate=True), out)
            got = cache.weights.cpu()
            (least, most) = (torch.zeros(got.shape), torch.zeros(got.shape))
            for row, b in enumerate([b for b, n in enumerate(counts) for _ in range(n)]):
                for g in range(8):
                    place = int(best[row, g])
                    if place >= 0:
                        least[int(table[b, place // 64]), g // 4, place % 64] += 1
                    if place == -2:
                        most[table[b].long().cpu(), g // 4] += 1
            most += least
            # the scores that attention had give what they gave there; made once more they may end below what the row ends with
            assert bool((got >= (least if offsets is None else 0)).all()) and bool((got <= most).all())
