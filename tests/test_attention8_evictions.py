"""The definition of eviction for long sequences against the one that goes token by token."""
import copy
import math
from types import SimpleNamespace

import pytest
import torch

import attention8_evictions as whole_heads
from attention8_reference import Model, exponent


def cache_of(pages, heads, dim, gen):
    part = lambda *s: torch.randint(0, 256, (pages, heads, *s), generator=gen, dtype=torch.uint8)
    scales = torch.randint(100, 140, (pages, heads, 4), generator=gen, dtype=torch.uint8)
    scales[..., 2:] = 0
    keys = part(64, dim)
    values = part(16, dim, 4)
    for t in (keys, values):
        t[(t & 127) == 127] = 0
    keys[3, 0, 5] = 127  # a token that is not finite, in keys and values
    values[3, 0, 1, :, 1] = 127
    scales[3, 0, 2] = 1
    weights = torch.randint(0, 5, (pages, heads, 64), generator=gen).float()
    weights[torch.rand(weights.shape, generator=gen) < 0.05] = math.nan
    return SimpleNamespace(pages=pages, heads=heads, dim=dim, keys=keys, values=values, scales=scales, weights=weights,
                           positions=torch.argsort(torch.rand((heads, pages * 64), generator=gen)).view(heads, pages, 64).transpose(0, 1).to(torch.int32) - 50)


@pytest.mark.parametrize("keep, recent", [(0, 0), (1, 1), (64, 10), (200, 30), (333, 333), (639, 0)])
@pytest.mark.parametrize("missing", [False, True])
def test_both_say_the_same(keep, recent, missing):
    gen = torch.Generator().manual_seed(keep + missing)
    table = torch.randperm(34, generator=gen)[:33].view(3, 11).to(torch.int32)
    if missing:
        table[0, 2] = -1
        table[1, 10] = 1 << 30
        table[2, 1:] = -5
    (a, lengths) = (Model(cache_of(34, 2, 32, gen)), torch.tensor([640, 700, 130]))
    b = copy.deepcopy(a)
    assert a.evict(table, lengths, keep, recent) == whole_heads.evict(b, table, lengths, keep, recent)
    for x, y in zip((*a.codes, *a.e, a.marked, a.weights, a.positions), (*b.codes, *b.e, b.marked, b.weights, b.positions)):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())


def test_powers():
    x = torch.tensor([0.0, 448.0, 448.0001, 449, 1e-40, 1e38, 3.4e38, 2.0 ** -117 * 448, 2.0 ** -117 * 449, 1.0, 7.0, 7.001], dtype=torch.float64)
    assert whole_heads.exponents(x).tolist() == [exponent(float(t)) for t in x]
