"""The cache in 8 bits, attention over it, the weights of its tokens and eviction against their definitions in 64 bits."""
import math

import pytest
import torch

import attention8_reference as ref8
from vectorlink_gpu import KVCache8, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
DIMS = [32, 64, 96, 128, 192, 256]
MAXINT = 2147483647


def ends(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEV)


def whole(*n):
    return torch.tensor(n, dtype=torch.int32, device=DEV)


def garbage(cache, gen):
    """A cache as recycled memory leaves it: any bytes, codes of NaN and powers that no page has among them."""
    for t in (cache.keys, cache.values, cache.scales):
        t.random_(0, 256, generator=gen)
    if cache.weights is not None:
        cache.weights.normal_(generator=gen)
        cache.positions.random_(-1000, 1000, generator=gen)


def filled(lengths, heads, dim, seed, dtype=torch.bfloat16, spare=2, blocks=None, weighted=True, pieces=1):
    """A cache over garbage with these sequences written to shuffled pages, and their table."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    blocks = max(1, -(-max(lengths) // 64)) if blocks is None else blocks
    pages = len(lengths) * blocks + spare
    cache = KVCache8.empty(pages, heads, dim, weighted=weighted)
    garbage(cache, gen)
    table = torch.randperm(pages, generator=gen, device=DEV)[:len(lengths) * blocks].view(len(lengths), blocks).to(torch.int32)
    rows = sum(lengths)
    x = torch.randn((2, rows, heads, dim), generator=gen, device=DEV) * torch.exp(torch.randn((2, 1, 1, dim), generator=gen, device=DEV) / 2)
    x = x.to(dtype)
    cache.write(x[0], x[1], table, whole(*[0] * len(lengths)), ends(lengths))
    return cache, table, whole(*lengths), gen


def queries_for(rows, heads, dim, gen, dtype, scale=1.0):
    return (scale * torch.randn((rows, heads, dim), generator=gen, device=DEV)).to(dtype)


# ---- writing and reading -------------------------------------------------------------------------

@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_write_then_read(dim, dtype):
    """Sequences that start at the beginning, inside, at the end of a block; none, one and many rows; strided inputs; powers that
    grow and powers that stay; positions of the caller's."""
    gen = torch.Generator(device=DEV).manual_seed(dim)
    (heads, starts, counts) = (3, [0, 63, 64, 17, 130, 5, 2], [65, 1, 0, 200, 64, 2, 1])
    blocks = 5
    cache = KVCache8.empty(7 * blocks + 1, heads, dim, weighted=True)
    garbage(cache, gen)
    wide = torch.randperm(7 * blocks + 1, generator=gen, device=DEV)[:7 * blocks].view(7, blocks).to(torch.int32)
    table = torch.full((7, blocks + 3), -7, dtype=torch.int32, device=DEV)[:, :blocks]
    table.copy_(wide)
    model = ref8.Model(cache)
    before = torch.randn((2, sum(starts), heads, dim), generator=gen, device=DEV).to(dtype)
    cache.write(before[0], before[1], table, whole(*[0] * 7), ends(starts))
    model.write(before, table, [0] * 7, ends(starts).tolist())
    model.check(cache)
    mixed = torch.randn((sum(counts), 2 * heads + 1, dim), generator=gen, device=DEV) * 10.0 ** torch.randint(-3, 4, (sum(counts), 2 * heads + 1, 1), generator=gen, device=DEV)
    mixed = mixed.to(dtype)
    (k, v) = (mixed[:, :heads], mixed[:, heads + 1:])
    positions = torch.randint(-5, 1 << 30, (sum(counts),), generator=gen, device=DEV).to(torch.int32)
    cache.write(k, v, table, whole(*starts), ends(counts), positions=positions)
    model.write((k, v), table, starts, ends(counts).tolist(), positions)
    model.check(cache)
    for kind in (torch.float32, dtype):
        (gk, gv) = cache.read(table, whole(*starts), sum(counts), ends(counts), dtype=kind)
        assert gk.dtype == kind
        row = 0
        for b, n in enumerate(counts):
            for i in range(n):
                (page, j) = (int(wide[b, (starts[b] + i) // 64]), (starts[b] + i) % 64)
                for got, which in ((gk, 0), (gv, 1)):
                    want = model.codes[which][page, :, j] * torch.exp2(model.e[which][page].double())[:, None]
                    assert torch.equal(got[row].cpu(), want.to(kind))
                row += 1


def test_write_rounds_to_the_nearest_code():
    """Ties and their neighbours, both signs, subnormal codes, at powers from the least to the largest; magnitudes at the border of a
    power; what no power holds."""
    base = torch.tensor([448.0, 449, 464, 447.9, 1.0625, 1.1875, 2.125, 17.0, 2 ** -6, 2 ** -7, 1.5 * 2 ** -9, 2 ** -10, 1.01 * 2 ** -10, 33.0, 0.0, -0.0])
    x = torch.cat((base, torch.nextafter(base, torch.tensor(900.0))))[:31]
    powers = [-149, -135, -126, -118, -117, -116, -60, -1, 0, 1, 9, 60, 110, 117, 118, 119]
    cache = KVCache8.empty(len(powers), 1, 32)
    garbage(cache, torch.Generator(device=DEV).manual_seed(1))
    model = ref8.Model(cache)
    rows = torch.zeros((len(powers), 1, 32))
    for i, e in enumerate(powers):
        y = (torch.cat((x, torch.tensor([7.0]))).double() * 2.0 ** e).clamp(max=3.4028234e38).float()
        rows[i, 0] = torch.where(torch.arange(32) % 2 == i % 2, -y, y)
    table = torch.arange(len(powers), dtype=torch.int32, device=DEV)[:, None]
    (rows, zeros) = (rows.to(DEV), whole(*[0] * len(powers)))
    cache.write(rows, -rows, table, zeros)
    model.write((rows, -rows), table, [0] * len(powers), list(range(len(powers) + 1)))
    model.check(cache)
    assert int(cache.scales[-1, 0, 0]) == 246 and int(cache.scales[0, 0, 0]) == 10
    (k, v) = cache.read(table, zeros, len(powers), dtype=torch.float32)
    assert bool(k.isfinite().all()) and torch.equal(k, -v)
    # one token's power for the others: 2^-20 of it and less is nothing
    more = rows.clone()
    more[:] = 2.0 ** 100
    cache.write(more, more, table, zeros + 1)
    model.write((more, more), table, [1] * len(powers), list(range(len(powers) + 1)))
    model.check(cache)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_spoils_its_token_alone(bad):
    cache, table, lengths, gen = filled([150], 2, 96, 3)
    model = ref8.Model(cache)
    (k, v) = torch.randn((2, 3, 2, 96), generator=gen, device=DEV)
    k[1, 0, 95] = bad
    v[2, 1, 0] = bad
    k[0] *= 1e4
    cache.write(k, v, table, lengths, ends([3]))
    model.write((k, v), table, [150], [0, 3])
    model.check(cache)
    (gk, gv) = cache.read(table, lengths, 3, ends([3]), dtype=torch.float32)
    assert int(gk.isnan().sum()) == 96 and int(gv.isnan().sum()) == 96
    assert bool(gk[1, 0].isnan().all()) and bool(gv[2, 1].isnan().all())
    assert cache.scales[table[0, 2].long(), :, 2].tolist() == [1, 1]
    # the page taken anew takes the mark away
    zero = whole(0)
    cache.write(k[:1], v[:1], table[:, 2:], zero)
    assert cache.scales[table[0, 2].long(), :, 2].tolist() == [0, 0]
    # a block of nothing else
    cache.write(torch.full_like(k, bad), torch.full_like(v, bad), table, zero, ends([3]))
    assert bool(cache.read(table, zero, 3, ends([3]))[0].isnan().all()) and cache.scales[table[0, 0].long(), 0].tolist() == [10, 10, 1, 0]


def test_pages_outside_the_cache_and_rows_of_no_sequence():
    cache, table, lengths, gen = filled([200, 100], 2, 64, 5)
    model = ref8.Model(cache)
    away = table.clone()
    away[0, 3] = MAXINT
    away[1, 1] = -1
    x = torch.randn((7, 2, 64), generator=gen, device=DEV)
    offsets = whole(2, 4, 5)  # rows 0, 1, 5, 6 are nobody's
    cache.write(x, x, away, lengths, offsets)
    model.write((x, x), away, lengths.tolist(), [2, 4, 5])
    model.check(cache)
    (k, v) = cache.read(away, lengths, 7, offsets)
    assert not bool(k.any()) and not bool(v.any())
    (k, v) = cache.read(table, lengths - 5, 7, offsets)
    assert not bool(k[:2].any()) and bool(k[2:5].any()) and not bool(k[5:].any())
    cache.write(x, x, away, whole(MAXINT, -5), offsets)  # behind what the table names; a length below 0 is 0
    model.write((x, x), away, [MAXINT, -5], [2, 4, 5])
    model.check(cache)


def test_far_pages():
    """Offsets past 2^32 bytes."""
    (pages, heads, dim) = (33_000, 8, 256)
    cache = KVCache8.empty(pages, heads, dim)
    cache.scales.zero_()
    gen = torch.Generator(device=DEV).manual_seed(8)
    table = whole(pages - 1, 0, pages - 2)[None]
    (k, v) = torch.randn((2, 130, heads, dim), generator=gen, device=DEV).bfloat16()
    cache.write(k, v, table, whole(0), ends([130]))
    small = KVCache8.empty(3, heads, dim)
    near = whole(0, 1, 2)[None]
    small.write(k, v, near, whole(0), ends([130]))
    for a, b in zip(cache.read(table, whole(0), 130, ends([130])), small.read(near, whole(0), 130, ends([130]))):
        assert torch.equal(a, b)
    for rows in (1, 130):
        q = torch.randn((rows, 16, dim), generator=gen, device=DEV).bfloat16()
        at = None if rows == 1 else ends([rows])
        for form in ("few", "many"):
            assert torch.equal(attend(q, cache, table, whole(130), at, form=form), attend(q, small, near, whole(130), at, form=form))


# ---- attention -----------------------------------------------------------------------------------

def forms_of(dim, dtype):
    return ["few", "many"] if dim * {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype] <= 256 else ["few"]


def attend_and_check(cache, table, lengths, q, offsets=None, scale=None, causal=True, form=None):
    """With and without weights: the same output, what the definition says; twice: the same bits."""
    want, added, room = ref8.attention(q, cache, table, lengths, offsets, scale, causal)
    before = cache.weights.clone()
    (out, lse) = attend(q, cache, table, lengths, offsets, scale=scale, causal=causal, return_lse=True, form=form)
    assert torch.equal(cache.weights, before)
    real = torch.zeros(q.size(0), dtype=torch.bool)
    real[:int(offsets[-1]) if offsets is not None else None] = True
    ref8.check_output(out[real.to(DEV)], [x[real] for x in want], q.dtype, form == "many")
    (w, off) = (want[1][real], (want[2][real] + 8) * 2.0 ** -23)
    lse = lse.cpu().double()[real]
    assert torch.equal(lse.isnan(), w.isnan()) and torch.equal(lse == -math.inf, w == -math.inf)
    fine = w.isfinite()
    assert bool(((lse - w).abs()[fine] <= off[fine] + w.abs()[fine] * 2.0 ** -22).all())
    again = attend(q, cache, table, lengths, offsets, scale=scale, causal=causal, form=form, accumulate=True)
    assert torch.equal(again.cpu()[real].nan_to_num(), out.cpu()[real].nan_to_num())
    ref8.check_weights(cache.weights, before, added, room)
    first = cache.weights.clone()
    cache.weights.copy_(before)
    attend(q, cache, table, lengths, offsets, scale=scale, causal=causal, form=form, accumulate=True)
    assert torch.equal(cache.weights, first)
    cache.weights.copy_(before)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 4, 7, 16, 20])
def test_single_tokens(dim, dtype, group):
    """Sequences of none, one, a page's border and more; tables wider than the lengths; a sequence that misses a page."""
    cache, table, lengths, gen = filled([0, 1, 64, 65, 300, 129], 2, dim, dim + group, dtype, blocks=7)
    table[5, 1] = MAXINT
    q = queries_for(6, 2 * group, dim, gen, dtype)
    attend_and_check(cache, table, lengths, q)
    if group == 4:
        attend_and_check(cache, table, lengths, q, scale=-0.3, causal=False)
        attend_and_check(cache, table, lengths, q, scale=0.0)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_prompts(dim, dtype, causal):
    (counts, lengths) = ([70, 0, 1, 33, 9], [200, 50, 65, 20, 64])  # the fourth has more rows than tokens
    cache, table, held, gen = filled(lengths, 2, dim, dim, dtype)
    table[0, 1] = -1
    q = queries_for(sum(counts) + 3, 6, dim, gen, dtype)[:, :6]
    for form in forms_of(dim, dtype):
        attend_and_check(cache, table, held, q, ends(counts), causal=causal, form=form)


@pytest.mark.parametrize("dtype", TYPES)
def test_split_over_workgroups(dtype):
    """Long sequences: parts are joined by a second launch; weights of many pages."""
    cache, table, lengths, gen = filled([5_000, 4_097], 1, 64, 6, dtype)
    q = queries_for(2, 3, 64, gen, dtype)
    attend_and_check(cache, table, lengths, q)
    counts = [3, 40]
    attend_and_check(cache, table, lengths, queries_for(43, 3, 64, gen, dtype), ends(counts))


@pytest.mark.parametrize("dim, dtype, group", [(64, torch.bfloat16, 4), (128, torch.float16, 7), (96, torch.float32, 16), (192, torch.bfloat16, 1)])
def test_many_short_sequences(dim, dtype, group):
    """A tile of rows is one wavefront's, which adds its tokens' weights itself; of prompts four pages are a workgroup's."""
    gen = torch.Generator().manual_seed(dim)
    lengths = torch.randint(0, 67, (700,), generator=gen).tolist()
    cache, table, held, gen = filled(lengths, 3, dim, dim, dtype, blocks=2)
    table[17, 0] = -1
    table[300:310, 1] = MAXINT
    attend_and_check(cache, table, held, queries_for(700, 3 * group, dim, gen, dtype))
    counts = [n % 3 for n in lengths]
    q = queries_for(sum(counts) + 2, 6, dim, gen, dtype)
    for form in forms_of(dim, dtype):
        attend_and_check(cache, table, held, q, ends(counts), form=form)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_weights_under_wide_tables(dim, dtype, causal):
    """Tables of many blocks, most of which hold nothing: pages that are marked, that miss, that some rows see; no rows, no tokens, more
    rows than tokens; as many rows as a step of the workgroup takes and one more."""
    (counts, lengths) = ([70, 0, 64, 33, 9, 1, 22], [300, 50, 65, 20, 0, 129, 400])
    cache, table, held, gen = filled(lengths, 2, dim, dim + 1, dtype)
    (k, v) = torch.randn((2, 30, 2, dim), generator=gen, device=DEV).to(dtype)
    k[9, 0, 3] = math.inf
    v[20, 1, 5] = math.nan
    cache.write(k, v, table, held - 30, whole(0, 30, 30, 30, 30, 30, 30, 30))
    wide = torch.full((7, 160), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    wide[6, 2] = cache.pages
    q = queries_for(sum(counts) + 3, 6, dim, gen, dtype)
    q[150, 2, 7] = math.nan
    for form in forms_of(dim, dtype):
        attend_and_check(cache, wide, held, q, ends(counts), causal=causal, form=form)


def test_tables_too_wide_for_scores():
    """Single tokens whose scores would take more than 4 GiB under their table."""
    cache, table, held, gen = filled([n % 150 for n in range(0, 64 * 7, 7)], 2, 32, 17)
    wide = torch.full((64, 17_000), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    attend_and_check(cache, wide, held, queries_for(64, 16, 32, gen, torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.4, 0.0, 7.0])
def test_scales(dtype, scale):
    """Scores that are turned round, that are all the same, and that leave one token all weight."""
    cache, table, lengths, gen = filled([150, 64, 5], 2, 64, 21, dtype)
    q = queries_for(60, 8, 64, gen, dtype)
    for form in forms_of(64, dtype):
        attend_and_check(cache, table, lengths, q, ends([40, 19, 1]), scale=scale, form=form)
    attend_and_check(cache, table, lengths, q[:3], scale=scale)


@pytest.mark.parametrize("form", [None, "many"])
def test_tokens_that_are_not_finite_are_seen_by_later_rows_alone(form):
    cache, table, lengths, gen = filled([90, 200], 2, 64, 12)
    (k, v) = torch.randn((2, 40, 2, 64), generator=gen, device=DEV).bfloat16()
    k[20, 0, 3] = math.inf
    v[25, 1, 60] = math.nan
    cache.write(k, v, table, lengths - 40, whole(0, 0, 40))
    counts = [1, 40]
    q = queries_for(41, 8, 64, gen, torch.bfloat16)
    attend_and_check(cache, table, lengths, q, ends(counts), form=form)
    if form is None:
        attend_and_check(cache, table, lengths, q[:2])
        attend_and_check(cache, table, lengths - 30, q[:2])
    # a query that is not finite gives no weight and spoils no other's
    q[5, 2, 7] = math.nan
    q[6, 3, 1] = math.inf
    attend_and_check(cache, table, lengths, q, ends(counts), form=form)
    q = queries_for(2, 8, 64, gen, torch.bfloat16)
    q[0, 5, 0] = math.nan
    attend_and_check(cache, table, lengths, q)


def test_scores_beyond_everything():
    """Scores that leave float32, and weights that vanish beside one."""
    cache, table, lengths, gen = filled([130], 1, 32, 9, torch.float32)
    q = queries_for(1, 2, 32, gen, torch.float32, scale=3e4)
    attend_and_check(cache, table, lengths, q)
    before = cache.weights.clone()
    big = torch.full((1, 1, 32), 1e38, device=DEV)
    cache.write(big, big, table, lengths - 1)
    before = cache.weights.clone()
    out = attend(big, cache, table, lengths, accumulate=True)  # inf - inf
    assert bool(out.isnan().all()) and torch.equal(cache.weights, before)


def test_strided_queries_and_rows_of_no_sequence():
    cache, table, lengths, gen = filled([100, 70], 2, 128, 4)
    mixed = queries_for(9, 11, 128, gen, torch.bfloat16)
    q = mixed[:, 1:9]
    offsets = whole(2, 4, 7)
    (out, lse) = attend(q, cache, table, lengths, offsets, return_lse=True)
    part = attend(q[2:7].contiguous(), cache, table, lengths, whole(0, 2, 5))
    assert torch.equal(out[2:7], part)
    off = torch.randn((9 * 8 * 128 + 1,), generator=gen, device=DEV).bfloat16()[1:].view(9, 8, 128)  # off every boundary but its own
    off.copy_(q)
    for form in ("few", "many"):
        assert torch.equal(attend(off, cache, table, lengths, offsets, form=form)[2:7], attend(q, cache, table, lengths, offsets, form=form)[2:7])


# ---- eviction ------------------------------------------------------------------------------------

def evict_and_check(cache, table, lengths, keep, recent):
    model = ref8.Model(cache)
    left = cache.evict(table, lengths, keep, recent)
    want = model.evict(table, lengths, keep, recent)
    assert left.tolist() == want
    model.check(cache)
    return left


def weigh_at_random(cache, gen, ties=False):
    w = torch.exp(2 * torch.randn(cache.weights.shape, generator=gen, device=DEV))
    w[torch.rand(w.shape, generator=gen, device=DEV) < 0.1] = 0.0
    if ties:
        w = torch.randint(0, 3, w.shape, generator=gen, device=DEV).float()
    cache.weights.copy_(w)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("keep, recent", [(0, 0), (1, 0), (1, 1), (63, 5), (64, 64), (65, 20), (128, 0), (150, 31), (299, 1), (300, 7)])
def test_eviction(dim, keep, recent):
    cache, table, lengths, gen = filled([0, 1, 64, 65, 200, 300], 2, dim, dim + keep, blocks=6)
    weigh_at_random(cache, gen)
    evict_and_check(cache, table, lengths, keep, recent)


@pytest.mark.parametrize("keep, recent", [(70, 0), (130, 40), (191, 191)])
def test_eviction_with_ties_and_weights_that_are_not_finite(keep, recent):
    cache, table, lengths, gen = filled([192, 260, 333], 3, 32, keep)
    weigh_at_random(cache, gen, ties=True)
    cache.weights[:, 0] = 1.0
    odd = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, -1.0, -0.0, 0.0, 1e-40], device=DEV)
    cache.weights[:, 2] = odd[torch.randint(0, 8, cache.weights[:, 2].shape, generator=gen, device=DEV)]
    cache.positions[:, 1] = 5  # all are the latest
    evict_and_check(cache, table, lengths, keep, recent)


def test_eviction_raises_powers():
    """Pages of small numbers that large ones move to, subnormal codes, and the border's page among them."""
    cache, table, lengths, gen = filled([500], 2, 64, 77)
    for first in range(0, 500, 20):
        (k, v) = torch.randn((2, 20, 2, 64), generator=gen, device=DEV) * 10.0 ** torch.randint(-12, 13, (2, 20, 2, 1), generator=gen, device=DEV)
        cache.write(k, v, table, whole(first), ends([20]))
    k[3, 0, 5] = math.nan
    v[4, 1, 6] = math.nan
    cache.write(k, v, table, whole(480), ends([20]))
    for keep in (333, 200, 100, 37):
        weigh_at_random(cache, gen)
        lengths = evict_and_check(cache, table, lengths, keep, 30)
    extremes = torch.tensor([2.0 ** -126, 3e38], device=DEV)[torch.randint(0, 2, (2, 130, 2, 1), generator=gen, device=DEV)].repeat(1, 1, 1, 64)
    cache.write(extremes[0], extremes[1], table, whole(0), ends([130]))
    for b in (0, 1, 2):  # powers at both ends
        cache.write(extremes[0, :1] * 0 + 2.0 ** (-120 + 100 * b), extremes[1, :1] * 0 + 2.0 ** (100 - 100 * b), table[:, b:b + 1], whole(0))
    weigh_at_random(cache, gen)
    evict_and_check(cache, table, whole(130), 100, 0)


def test_eviction_of_sequences_that_miss_pages():
    cache, table, lengths, gen = filled([300, 320, 100, 200], 2, 32, 13)
    table[0, 1] = -3
    table[1, 4] = MAXINT
    table[2] = -1
    table[3, 0] = cache.pages
    weigh_at_random(cache, gen)
    left = evict_and_check(cache, table, lengths, 90, 10)
    assert left.tolist() == [90, 90, 0, 90]
    table[3, 1:] = -1
    assert evict_and_check(cache, table, whole(MAXINT, 90, -4, 200), 89, 10).tolist() == [89, 89, 0, 0]


@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("keep", [1_470, 1_535, 1_472])
def test_eviction_of_few_of_many(dim, keep):
    """Several pages are one workgroup's: sequences that keep all, that end early or miss pages among others; tokens of all sizes, so that
    powers grow, and one that is not finite."""
    lengths = [1_536, 1_500, 0, 1_536, keep, keep + 1, 700] + [1_536] * 17
    cache, table, held, gen = filled(lengths, 4, dim, keep + dim, blocks=24)
    (k, v) = torch.randn((2, 10 * 24, 4, dim), generator=gen, device=DEV) * 10.0 ** torch.randint(-2, 5, (2, 10 * 24, 4, 1), generator=gen, device=DEV)
    k[3, 0, 5] = math.nan
    cache.write(k, v, table, (held - 10).clamp(min=0), ends([10] * 24))
    table[3, 5] = -1
    table[8, 23] = MAXINT
    weigh_at_random(cache, gen)
    evict_and_check(cache, table, held, keep, 12)


@pytest.mark.parametrize("length, keep, recent", [(20_000, 9_999, 500), (70_001, 1_000, 999), (70_001, 69_990, 0)])
def test_eviction_of_long_sequences(length, keep, recent):
    """By what holds of every eviction, and with sorts of the whole."""
    cache, table, lengths, gen = filled([length, 50], 2, 32, length)
    weigh_at_random(cache, gen)
    cache.weights[:, 1] = cache.weights[:, 1].round()  # many ties
    pages = table[0].long()
    (w, p) = (t[pages].transpose(0, 1).flatten(1)[:, :length].clone() for t in (cache.weights, cache.positions))
    (k, v) = (x.view(length, 2, 32) for x in cache.read(table[:1], whole(0), length, ends([length]), dtype=torch.float32))
    late = p > p.amax(1, keepdim=True) - recent
    order = torch.sort(torch.where(late, math.inf, w), dim=1, descending=True, stable=True).indices
    stay = torch.zeros_like(late).scatter(1, order[:, :keep], True)
    left = cache.evict(table, lengths, keep, recent)
    assert left.tolist() == [keep, 50]
    (gk, gv) = cache.read(table[:1], whole(0), keep, ends([keep]), dtype=torch.float32)
    for h in range(2):
        source = torch.arange(keep, device=DEV)
        source[~stay[h, :keep]] = torch.arange(keep, length, device=DEV)[stay[h, keep:]]
        assert torch.equal(cache.weights[pages, h].flatten()[:keep], w[h, source])
        assert torch.equal(cache.positions[pages, h].flatten()[:keep], p[h, source])
        for got, was in ((gk, k), (gv, v)):  # rounded again at most over a power that a larger token needed
            off = (got[:, h] - was[source, h]).abs()
            assert bool((off <= was[:, h].abs().max() * 2.0 ** -17).all()) and float((off > 0).float().mean()) < 0.01


def test_read_in_weigh_evict_and_go_on():
    """A program's steps: a prompt in pieces, weights, an eviction, then a token at a time with an eviction every 16."""
    (heads, group, dim, keep, recent) = (2, 4, 64, 100, 20)
    gen = torch.Generator(device=DEV).manual_seed(31)
    cache = KVCache8.empty(14, heads, dim, weighted=True)
    garbage(cache, gen)
    table = torch.randperm(14, generator=gen, device=DEV).view(2, 7).to(torch.int32)
    (lengths, texts) = (whole(0, 0), 0)
    for piece in (150, 64, 33):
        (k, v) = torch.randn((2, 2 * piece, heads, dim), generator=gen, device=DEV).bfloat16()
        cache.write(k, v, table, lengths, ends([piece] * 2))
        lengths = lengths + piece
        texts += piece
        attend_and_check(cache, table, lengths, queries_for(2 * piece, heads * group, dim, gen, torch.bfloat16), ends([piece] * 2))
        attend(queries_for(2 * piece, heads * group, dim, gen, torch.bfloat16), cache, table, lengths, ends([piece] * 2), accumulate=True)
    lengths = evict_and_check(cache, table, lengths, keep, recent)
    assert lengths.tolist() == [keep, keep]
    for step in range(33):
        (k, v) = torch.randn((2, 2, heads, dim), generator=gen, device=DEV).bfloat16()
        cache.write(k, v, table, lengths, positions=whole(texts, texts))
        lengths = lengths + 1
        texts += 1
        q = queries_for(2, heads * group, dim, gen, torch.bfloat16)
        attend_and_check(cache, table, lengths, q)
        attend(q, cache, table, lengths, accumulate=True)
        if step % 16 == 15:
            lengths = evict_and_check(cache, table, lengths, keep, recent)
            for b in range(2):  # the latest stay in every head
                places = cache.positions[table[b].long()].transpose(0, 1).flatten(1)[:, :keep]
                for h in range(heads):
                    assert set(range(texts - recent, texts)) <= set(places[h].tolist())


def test_captured_steps():
    """A step captured into a graph and replayed, with the program's own work between, gives what eager calls give."""
    cache, table, lengths, gen = filled([300, 150], 2, 128, 55, blocks=8)
    weigh_at_random(cache, gen)
    parts = ("keys", "values", "scales", "weights", "positions")
    start = {n: getattr(cache, n).clone() for n in parts}
    other = KVCache8(**{n: t.clone() for n, t in start.items()})
    (k, v) = torch.randn((2, 2, 2, 128), generator=gen, device=DEV).bfloat16()
    q = queries_for(2, 8, 128, gen, torch.bfloat16)
    many = queries_for(100, 8, 128, gen, torch.bfloat16)
    (now, then) = (lengths.clone(), lengths.clone())
    texts = whole(300, 300)

    def step(cache, now, texts):
        cache.write(k, v, table, now, positions=texts)
        now += 1
        texts += 1
        a = attend(q, cache, table, now, accumulate=True)
        b = attend(many, cache, table, now, ends50, accumulate=True)
        now.copy_(cache.evict(table, now, 140, 16))
        return a, b, attend(q, cache, table, now)

    ends50 = ends([50, 50])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(cache, now, texts.clone())
    torch.cuda.synchronize()
    for n in parts:
        getattr(cache, n).copy_(start[n])
    now.copy_(lengths)
    count = texts.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, now, count)
    for i in range(4):
        graph.replay()
        want = step(other, then, texts)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        for n in parts:
            assert torch.equal(getattr(cache, n), getattr(other, n)), (i, n)
        k.normal_(generator=gen)
        q.normal_(generator=gen)


def test_nothing_to_look_at():
    """Tables of no blocks, a cache of no pages, no sequences: zeros, and lengths that are cut to what there is."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    q = queries_for(2, 4, 64, gen, torch.bfloat16)
    (kv, held) = (queries_for(2, 2, 64, gen, torch.bfloat16), whole(100, 7))
    full = filled([100], 2, 64, 5)[0]
    none = KVCache8.empty(0, 2, 64, weighted=True)
    for cache, table, left in [(full, torch.empty((2, 0), dtype=torch.int32, device=DEV), [0, 0]), (none, whole(0, 1, 2, 3).view(2, 2), [0, 7]),
                               (full, torch.full((2, 2), -1, dtype=torch.int32, device=DEV), [0, 7])]:
        was = [t.clone() for t in (cache.keys, cache.values, cache.scales, cache.weights, cache.positions)]
        for offsets in (None, whole(0, 1, 2), whole(0, 0, 0)):
            cache.write(kv, kv, table, held, offsets)
            assert not any(bool(t.any()) for t in cache.read(table, held, 2, offsets))
            out = attend(q, cache, table, held, offsets, accumulate=True)
            assert not bool(out[:0 if offsets is not None and not int(offsets[-1]) else None].any())
        assert cache.evict(table, held, 10, 3).tolist() == left
        assert cache.evict(table, held, 0).tolist() == [0, 0]
        for a, b in zip(was, (cache.keys, cache.values, cache.scales, cache.weights, cache.positions)):
            assert torch.equal(a.nan_to_num() if a.is_floating_point() else a, b.nan_to_num() if b.is_floating_point() else b)
    nothing = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    full.write(kv[:0], kv[:0], nothing, held[:0])
    assert attend(q[:0], full, nothing, held[:0], accumulate=True).shape == (0, 4, 64)
    assert full.evict(nothing, held[:0], 5).shape == (0,)


def test_two_streams():
    """Two caches worked on at once."""
    jobs = []
    for seed in (1, 2):
        cache, table, lengths, gen = filled([3_000, 2_000], 2, 64, seed)
        weigh_at_random(cache, gen)
        jobs.append((cache, table, lengths, queries_for(2, 8, 64, gen, torch.bfloat16), torch.cuda.Stream()))
    copies = [KVCache8(*(t.clone() for t in (c.keys, c.values, c.scales, c.weights, c.positions))) for c, *_ in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for cache, table, lengths, q, stream in jobs:
            with torch.cuda.stream(stream):
                got.append(attend(q, cache, table, lengths, accumulate=True))
                cache.evict(table, lengths, 1_500, 100)
    torch.cuda.synchronize()
    at = 0
    for _ in range(5):
        for copy, (cache, table, lengths, q, _) in zip(copies, jobs):
            assert torch.equal(attend(q, copy, table, lengths, accumulate=True), got[at])
            copy.evict(table, lengths, 1_500, 100)
            at += 1
    for copy, (cache, *_) in zip(copies, jobs):
        for name in ("keys", "values", "scales", "weights", "positions"):
            assert torch.equal(getattr(copy, name), getattr(cache, name)), name


def test_refusals_on_the_gpu():
    cache, table, lengths, gen = filled([100], 2, 64, 1, weighted=False)
    q = queries_for(1, 4, 64, gen, torch.bfloat16)
    attend(q, cache, table, lengths)
    with pytest.raises(AssertionError):
        attend(q, cache, table, lengths, accumulate=True)
    with pytest.raises(AssertionError):
        cache.evict(table, lengths, 50)
    with pytest.raises(RuntimeError):
        attend(q, cache, table, lengths.cpu())
    with pytest.raises(RuntimeError):
        cache.write(q[:, :2], q[:, :2], table.cpu(), lengths)
    with pytest.raises(AssertionError):
        attend(queries_for(1, 4, 64, gen, torch.float32), cache, table, lengths, form="most")
