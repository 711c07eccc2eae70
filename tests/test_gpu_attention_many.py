"""Attention of many rows over the same tokens against its definition in 64 bits: prompts and pieces of prompts."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, TYPES, ends, filled, queries_for
from vectorlink_gpu import _native as nv
from vectorlink_gpu import attend

pytestmark = pytest.mark.gpu

# units of rounding: a type of b significant bits is off by 2^-b of the number at most; weights are rounded to 8, 16 or 24 bits
UNIT = {torch.bfloat16: (2.0 ** -8, 2.0 ** -8), torch.float16: (2.0 ** -16, 2.0 ** -11), torch.float32: (2.0 ** -23, 2.0 ** -24)}


def dense(queries, cache, table, lengths, offsets=None, scale=None, causal=True):
    """(out, lse, size, most): attention_reference.attention with all rows of a sequence and head at once"""
    q = queries.detach().cpu().double()
    (rows, heads, dim) = q.shape
    group = heads // cache.heads
    scale = dim ** -0.5 if scale is None else scale
    (lengths, offsets) = (lengths.cpu().tolist(), offsets.cpu().tolist())
    held = ref.Held(cache, table, lengths)
    (out, size) = (torch.zeros((rows, heads, dim), dtype=torch.float64) for _ in range(2))
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    most = torch.zeros((rows, heads), dtype=torch.float64)
    for b in range(table.size(0)):
        (first, end, n) = (offsets[b], offsets[b + 1], held.lengths[b])
        if first == end or n == 0:
            continue
        sees = torch.full((end - first,), n)
        if causal:
            sees = (lengths[b] - (end - first) + torch.arange(end - first) + 1).clamp(0, n)
        for h in range(cache.heads):
            (k, v) = (held.k[b, h], held.v[b, h])
            mask = (torch.arange(n) < sees[:, None]) & ~torch.isneginf(k[:, 0])
            spoilt = (k.isnan().any(1) | v.isnan().any(1))
            (k, v) = (torch.where(k.isfinite(), k, 0.0), torch.where(v.isfinite(), v, 0.0))
            for g in range(h * group, (h + 1) * group):
                s = (q[first:end, g] @ k.T) * scale
                p = torch.nan_to_num(torch.softmax(s.masked_fill(~mask, -math.inf), 1))
                bad = (mask & spoilt).any(1)
                out[first:end, g] = (p @ v).masked_fill(bad[:, None], math.nan)
                lse[first:end, g] = torch.logsumexp(s.masked_fill(~mask, -math.inf), 1).masked_fill(bad, math.nan)
                size[first:end, g] = p @ v.abs()
                most[first:end, g] = ((q[first:end, g].abs() @ k.abs().T) * abs(scale) * mask).amax(1)
    return out, lse, size, most


def check(got, lse, want, dtype, dim):
    (out, want_lse, size, most) = want
    (weight, last) = UNIT[dtype]
    score = ((dim + 8) * most + 32)[..., None] * 2.0 ** -24  # what scores and exponentials of 32 bits are off by
    got = got.cpu().double()
    assert torch.equal(got.isnan(), out.isnan())
    room = (weight + 2 * score) * size + 1.01 * last * out.abs() + weight * last * size + 2.0 ** -24
    bad = ((got - out).abs() > room) & ~out.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - out).abs() / room).nan_to_num().max()):.2f} times the bound"
    lse = lse.cpu().double()
    assert torch.equal(lse.isneginf(), want_lse.isneginf()) and torch.equal(lse.isnan(), want_lse.isnan())
    some = want_lse.isfinite()
    assert ((lse - want_lse).abs() <= 2 * score[..., 0] + 2.0 ** -20 + want_lse.abs() * 2.0 ** -22)[some].all()


def form(dim, dtype):
    """Asks for the form for many rows where it is there; the one for few takes the others."""
    return "many" if dim * nv.TYPES[dtype] <= 256 else None


def run(counts, lengths, heads, group, dim, dtype, seed, causal=True, scale=None):
    cache, table, lengths, gen = filled(lengths, heads, dim, seed, dtype)
    q = queries_for(sum(counts), heads * group, dim, gen, dtype)
    at = ends(counts)
    (out, lse) = attend(q, cache, table, lengths, offsets=at, causal=causal, scale=scale, return_lse=True, form=form(dim, dtype))
    check(out, lse, dense(q, cache, table, lengths, at, scale, causal), dtype, dim)
    assert torch.equal(out, attend(q, cache, table, lengths, offsets=at, causal=causal, scale=scale, form=form(dim, dtype)))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,heads,group", [(32, 1, 4), (64, 2, 7), (96, 3, 3), (128, 2, 4), (128, 1, 1), (192, 1, 5), (256, 1, 2)])
def test_prompts(dim, heads, group, causal, dtype):
    """Sequences of which all, some, one or no tokens are new; more new ones than tokens, which then see nothing."""
    run([600, 0, 333, 1, 450], [600, 77, 1001, 64, 300], heads, group, dim, dtype, dim + group, causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_fill_tiles_and_pages(dtype):
    run([64, 128, 256, 512], [64, 128, 320, 512], 1, 8, 128, dtype, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_few_tiles_over_many_pages(dtype):
    """One sequence of few rows and many tokens: split over workgroups and joined."""
    run([300], [9000], 1, 2, 64, dtype, 5)


@pytest.mark.parametrize("scale", [0.0, -0.2, 4.0])
def test_scales(scale):
    run([300], [500], 1, 4, 64, torch.bfloat16, 7, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_grow(dtype):
    """Keys that grow along the sequence: the maximum moves in nearly every page, by little and by much."""
    cache, table, lengths, gen = filled([700], 1, 64, 9, dtype)
    k = torch.randn((700, 1, 64), generator=gen, device=DEV) * torch.logspace(-2, 1.3, 700, device=DEV)[:, None, None]
    cache.write(k.to(dtype), k.to(dtype), table, lengths - 700, ends([700]))
    q = queries_for(400, 2, 64, gen, dtype, 3.0)
    (out, lse) = attend(q, cache, table, lengths, offsets=ends([400]), return_lse=True, form=form(64, dtype))
    check(out, lse, dense(q, cache, table, lengths, ends([400])), dtype, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_that_are_not_finite(dtype):
    """They spoil the rows that see them and no others, in the same tile too; pages without one are among those with one."""
    cache, table, lengths, gen = filled([500, 200], 2, 64, 11, dtype)
    k = torch.randn((400, 2, 64), generator=gen, device=DEV).to(dtype)
    v = torch.randn((400, 2, 64), generator=gen, device=DEV).to(dtype)
    k[350, 0, 3] = math.nan
    v[390, 1, 60] = math.inf
    cache.write(k, v, table, lengths - torch.tensor([400, 0], dtype=torch.int32, device=DEV), ends([400, 0]))
    q = queries_for(600, 4, 64, gen, dtype)
    (out, lse) = attend(q, cache, table, lengths, offsets=ends([400, 200]), return_lse=True, form=form(64, dtype))
    want = dense(q, cache, table, lengths, ends([400, 200]))
    assert want[0][:350].isfinite().all() and want[0][350:400, :2].isnan().all() and want[0][390:400].isnan().all() and want[0][400:].isfinite().all()
    check(out, lse, want, dtype, 64)


def test_pages_that_hold_nothing_take_no_part():
    cache, table, lengths, gen = filled([600, 600], 1, 128, 13)
    table[0, 0] = -1
    table[0, 5] = 2147483647
    table[1] = cache.pages
    q = queries_for(900, 2, 128, gen, torch.bfloat16)
    (out, lse) = attend(q, cache, table, lengths, offsets=ends([500, 400]), return_lse=True, form="many")
    check(out, lse, dense(q, cache, table, lengths, ends([500, 400])), torch.bfloat16, 128)
    assert not out[500:].any()


def test_strides_and_alignment():
    cache, table, lengths, gen = filled([500, 130], 2, 96, 15)
    flat = queries_for(430, 6, 96, gen, torch.bfloat16)
    at = ends([400, 30])
    want = attend(flat, cache, table, lengths, offsets=at, form="many")
    for q in (torch.empty((430, 10, 99), dtype=torch.bfloat16, device=DEV)[:, 2:8, 1:97],
              torch.empty((6, 430, 96), dtype=torch.bfloat16, device=DEV).transpose(0, 1)):
        q.copy_(flat)
        assert torch.equal(attend(q, cache, table, lengths, offsets=at, form="many"), want)


def test_single_tokens_in_the_form_for_many():
    """Without offsets, one row a sequence."""
    cache, table, lengths, gen = filled([300, 0, 77], 2, 128, 17)
    q = queries_for(3, 8, 128, gen, torch.bfloat16)
    (out, lse) = attend(q, cache, table, lengths, return_lse=True, form="many")
    check(out, lse, dense(q, cache, table, lengths, ends([1, 1, 1])), torch.bfloat16, 128)


def test_rows_behind_the_last_offset_are_left_alone():
    """Offsets that name fewer rows than there are, or more: nothing outside is read or written."""
    cache, table, lengths, gen = filled([300, 200], 1, 64, 19)
    q = queries_for(300, 2, 64, gen, torch.bfloat16)
    for f in ("few", "many"):
        want = attend(q[:250], cache, table, lengths, offsets=ends([150, 100]), form=f)
        got = attend(q, cache, table, lengths, offsets=ends([150, 100]), form=f)
        assert torch.equal(got[:250], want)
        over = ends([150, 100])
        over[2] = 1_000_000  # cut to the rows that there are
        attend(q[:250], cache, table, lengths, offsets=over, form=f)
