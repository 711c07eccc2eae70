"""Rows of one wavefront whose maxima move at different tokens."""
import pytest
import torch

from test_gpu_attention import DEV, TYPES, ends, filled, queries_for
from vectorlink_gpu import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_does_not_depend_on_its_neighbours(dtype):
    """Rows of one wavefront whose maxima move at other pages: a row's result is the same whatever the others hold, to the last bit."""
    (cache, table, lengths, gen) = filled([900], 1, 64, 67, dtype)
    k = torch.randn((900, 1, 64), generator=gen, device=DEV) * torch.logspace(-1.5, 0.5, 900, device=DEV)[:, None, None]
    cache.write(k.to(dtype), k.to(dtype), table, lengths - 900, ends([900]))
    q = queries_for(256, 1, 64, gen, dtype, 2.0)
    at = ends([256])
    (out, lse) = attend(q, cache, table, lengths, offsets=at, causal=False, return_lse=True, form="many")
    for turn in (3.0, 0.1, -2.0):
        other = q.clone()
        keep = torch.arange(256, device=DEV) % 4 == 1
        other[~keep] = (other[~keep].float() * turn).to(dtype)
        (out2, lse2) = attend(other, cache, table, lengths, offsets=at, causal=False, return_lse=True, form="many")
        assert torch.equal(out[keep], out2[keep]) and torch.equal(lse[keep], lse2[keep])
        assert not torch.equal(out[~keep], out2[~keep])
