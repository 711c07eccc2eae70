"""Scales next to nothing."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, ends, filled, queries_for
from test_gpu_attention_many import check, dense
from vectorlink_gpu import attend, attend_blocks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["few", "many"])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-46, 1e-39, -4e-38, 1.2e-38, 3e-37])
def test_scales_next_to_nothing(scale, form):
    """Queries and keys of 2^58 each: a scale of 1e-38 is a small one there, and 0 leaves all tokens alike."""
    (cache, table, lengths, gen) = filled([700, 90], 1, 64, 61, torch.float32)
    x = 2.0 ** 58 * torch.randn((790, 1, 64), generator=gen, device=DEV)
    v = torch.randn((790, 1, 64), generator=gen, device=DEV)
    cache.write(x, v, table, lengths * 0, ends([700, 90]))
    q = 2.0 ** 58 * queries_for(60, 2, 64, gen, torch.float32)
    at = ends([50, 10])
    (out, lse) = attend(q, cache, table, lengths, offsets=at, scale=scale, return_lse=True, form=form)
    check(out, lse, dense(q, cache, table, lengths, at, scale), torch.float32, 64)
    blocks = torch.arange(11, dtype=torch.int32, device=DEV).expand(60, 1, 11).contiguous()
    ref.check_attention(attend_blocks(q, cache, table, lengths, blocks, at, scale=scale),
                        ref.attention(q, cache, table, lengths, at, scale=scale, blocks=blocks.cpu()), torch.float32)


@pytest.mark.parametrize("form", ["few", "many"])
def test_no_scale_leaves_what_is_not_finite(form):
    """0 times an infinity or a NaN is no score."""
    (cache, table, lengths, gen) = filled([300], 1, 64, 63, torch.float32)
    q = queries_for(40, 2, 64, gen, torch.float32)
    q[3, 0, 5] = torch.inf
    q[7, 1, 60] = torch.nan
    out = attend(q, cache, table, lengths, offsets=ends([40]), scale=0.0, form=form)
    bad = out.isnan().any(-1)
    assert bad.sum() == 2 and bad[3, 0] and bad[7, 1]
