"""Batches with a place for each of many sequences, of which few have new tokens: what few rows give, wherever they stand."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, ends, filled, queries_for
from test_gpu_attention_many import check, dense
from vectorlink_gpu import attend, attend_selected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [None, "few", "many"])
@pytest.mark.parametrize("counts", [{0: 1}, {130: 1}, {3: 1, 64: 70, 65: 1, 130: 2}, {5: 2, 6: 1, 100: 1}])
def test_few_sequences_of_many_have_rows(counts, form):
    places = sorted(counts)
    held = [333, 70, 131, 64][:len(places)]
    (cache, some, lengths, gen) = filled(held, 2, 64, 3)
    sequences = 131
    table = torch.full((sequences, some.size(1)), -1, dtype=torch.int32, device=DEV)
    table[places] = some
    every = torch.zeros(sequences, dtype=torch.int32, device=DEV)
    every[places] = lengths
    at = ends([counts.get(b, 0) for b in range(sequences)])
    rows = int(at[-1])
    (k, v) = (queries_for(rows, 2, 64, gen, torch.bfloat16) for _ in range(2))
    starts = every - (at[1:] - at[:-1])
    cache.write(k, v, table, starts, at)
    (gk, gv) = cache.read(table, starts, rows, at, dtype=torch.float32)
    assert torch.equal(gk.cpu().double(), ref.rounded(k)) and torch.equal(gv.cpu().double(), ref.rounded(v))
    q = queries_for(rows, 6, 64, gen, torch.bfloat16)
    (out, lse) = attend(q, cache, table, every, offsets=at, return_lse=True, form=form)
    check(out, lse, dense(q, cache, table, every, at), torch.bfloat16, 64)
    (out, blocks) = attend_selected(q, cache, table, every, 2, offsets=at)
    assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, every, 2, at))
    ref.check_attention(out, ref.attention(q, cache, table, every, at, blocks=blocks), torch.bfloat16)
