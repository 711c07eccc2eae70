"""The cache in 4 bits and attention over it against their definitions in 64 bits."""
import math

import pytest
import torch

import attention_reference as ref
from vectorlink_gpu import KVCache, attend, attend_blocks, attend_selected, select_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
MAXINT = 2147483647


def garbage(cache, gen):
    """A cache as recycled memory leaves it: any bytes, scales of 255 among them."""
    for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
        t.random_(0, 256, generator=gen)
    cache.key_scales[torch.rand(cache.key_scales.shape, generator=gen, device=DEV) < 0.2] = 255
    cache.value_scales[torch.rand(cache.value_scales.shape, generator=gen, device=DEV) < 0.2] = 255
    cache.bounds.random_(-128, 128, generator=gen)
    cache.bound_scales.random_(-128, 128, generator=gen)


def filled(lengths, heads, dim, seed, dtype=torch.bfloat16, spare=2, blocks=None):
    """A cache over garbage with these sequences written to shuffled pages, and their table."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    blocks = max(1, -(-max(lengths) // 64)) if blocks is None else blocks
    pages = len(lengths) * blocks + spare
    cache = KVCache.empty(pages, heads, dim)
    garbage(cache, gen)
    table = torch.randperm(pages, generator=gen, device=DEV)[:len(lengths) * blocks].view(len(lengths), blocks).to(torch.int32)
    rows = sum(lengths)
    offsets = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=DEV)
    x = torch.randn((2, rows, heads, dim), generator=gen, device=DEV) * torch.exp(torch.randn((2, 1, 1, dim), generator=gen, device=DEV) / 2)
    x = x.to(dtype)
    cache.write(x[0], x[1], table, torch.zeros(len(lengths), dtype=torch.int32, device=DEV), offsets)
    return cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), gen


def queries_for(rows, heads, dim, gen, dtype, scale=1.0):
    return (scale * torch.randn((rows, heads, dim), generator=gen, device=DEV)).to(dtype)


def ends(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEV)


# ---- writing and reading -------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_write_then_read(dim, dtype):
    """Sequences that start at the beginning, inside, at the end of a block; none, one and many rows; strided inputs."""
    gen = torch.Generator(device=DEV).manual_seed(dim)
    (heads, starts, counts) = (3, [0, 63, 64, 17, 130, 5], [65, 1, 0, 200, 64, 2])
    blocks = 5
    cache = KVCache.empty(6 * blocks + 1, heads, dim)
    garbage(cache, gen)
    wide = torch.randperm(6 * blocks + 1, generator=gen, device=DEV)[:6 * blocks].view(6, blocks).to(torch.int32)
    table = torch.full((6, blocks + 3), -7, dtype=torch.int32, device=DEV)[:, :blocks]
    table.copy_(wide)
    zeros = torch.zeros(6, dtype=torch.int32, device=DEV)
    before = torch.randn((2, sum(starts), heads, dim), generator=gen, device=DEV).to(dtype)
    cache.write(before[0], before[1], table, zeros, ends(starts))
    mixed = torch.randn((sum(counts), 2 * heads + 1, dim), generator=gen, device=DEV) * 10.0 ** torch.randint(-3, 4, (1, 1, dim), generator=gen, device=DEV)
    mixed = mixed.to(dtype)
    (k, v) = (mixed[:, :heads], mixed[:, heads + 1:])
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    cache.write(k, v, table, at, ends(counts))
    (gk, gv) = cache.read(table, at, sum(counts), ends(counts), dtype=torch.float32)
    (wk, wv) = (ref.rounded(k), ref.rounded(v))
    assert torch.equal(gk.cpu().double(), wk) and torch.equal(gv.cpu().double(), wv)
    (gk, gv) = cache.read(table, at, sum(counts), ends(counts), dtype=dtype)
    assert gk.dtype == dtype and torch.equal(gk.cpu(), wk.to(dtype)) and torch.equal(gv.cpu(), wv.to(dtype))
    (gk, gv) = cache.read(table, zeros, sum(starts), ends(starts), dtype=torch.float32)
    assert torch.equal(gk.cpu().double(), ref.rounded(before[0])) and torch.equal(gv.cpu().double(), ref.rounded(before[1]))
    lengths = [a + n for a, n in zip(starts, counts)]
    held = ref.Held(cache, table, lengths)
    bounds = cache.read_bounds(table).cpu().double()
    for b, n in enumerate(lengths):
        for i in range(-(-n // 64)):
            for h in range(heads):
                (hi, lo, e) = ref.bounds_of(held.k[b, h][i * 64:i * 64 + 64], held.v[b, h][i * 64:i * 64 + 64])
                page = int(table[b, i])
                assert int(cache.bound_scales[page, h]) == e
                assert torch.equal(bounds[b, i, h, 0], hi * 2.0 ** e) and torch.equal(bounds[b, i, h, 1], lo * 2.0 ** e)


def test_write_rounds_to_the_nearest_code():
    """Every tie and its neighbours, both signs, at scales from the least to the largest; values that are too small become zero."""
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.99, 4.0, 0.1, 0.0, -0.0], dtype=torch.float32)
    x = torch.cat((base, torch.nextafter(base, torch.tensor(9.0)), torch.nextafter(base, torch.tensor(-9.0))))[:31]
    rows = torch.zeros((16, 1, 32))
    for i, e in enumerate((-149, -130, -126, -124, -123, -60, -1, 0, 1, 2, 3, 10, 60, 120, 124, 125)):
        y = (torch.cat((x, torch.tensor([7.0]))).double() * 2.0 ** e).float()
        rows[i, 0] = torch.where(torch.arange(32) % 2 == i % 2, -y, y)
    cache = KVCache.empty(1, 1, 32)
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.write(rows.to(DEV), -rows.to(DEV), table, start, ends([16]))
    (k, v) = cache.read(table, start, 16, ends([16]), dtype=torch.float32)
    assert torch.equal(k.cpu().double(), ref.rounded(rows)) and torch.equal(v.cpu().double(), ref.rounded(-rows))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_spoils_its_token_alone(bad):
    cache, table, lengths, gen = filled([150], 2, 96, 3)
    k = torch.randn((3, 2, 96), generator=gen, device=DEV)
    v = torch.randn((3, 2, 96), generator=gen, device=DEV)
    k[1, 0, 95] = bad
    v[2, 1, 0] = bad
    cache.write(k, v, table, lengths, ends([3]))
    (gk, gv) = cache.read(table, lengths, 3, ends([3]), dtype=torch.float32)
    assert torch.equal(gk.cpu().double().isnan(), ref.rounded(k).isnan()) and torch.equal(gv.cpu().double().isnan(), ref.rounded(v).isnan())
    assert int(gk.isnan().sum()) == 96 and int(gv.isnan().sum()) == 96
    assert cache.bound_scales[table[0, 2].long()].tolist() == [127, 127]
    edges = cache.read_bounds(table[0, 2:])
    assert torch.equal(edges[0, :, 0], torch.full((2, 96), math.inf, device=DEV)) and torch.equal(edges[0, :, 1], torch.full((2, 96), -math.inf, device=DEV))
    # a step back takes it out again
    cache.write(k[:1], v[:1], table, lengths, None)
    assert 127 not in cache.bound_scales[table[0, 2].long()].tolist()


def test_pages_outside_the_cache_hold_nothing():
    cache, table, lengths, gen = filled([200, 100], 2, 64, 5)
    images = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.bounds, cache.bound_scales)]
    away = table.clone()
    away[0, 3] = MAXINT
    away[1, 1] = -1
    k = torch.randn((30, 2, 64), generator=gen, device=DEV)
    cache.write(k, k, away, lengths, ends([20, 10]))
    for t, was in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.bounds, cache.bound_scales), images):
        assert torch.equal(t, was)
    (gk, gv) = cache.read(away, lengths, 30, ends([20, 10]))
    assert not gk.any() and not gv.any()
    assert not cache.read_bounds(torch.tensor([-1, MAXINT, cache.pages], dtype=torch.int32, device=DEV)).any()
    # places behind the table's last block
    cache.write(k[:2], k[:2], table, torch.tensor([256, 10_000], dtype=torch.int32, device=DEV))
    for t, was in zip((cache.keys, cache.values), images):
        assert torch.equal(t, was)


def test_a_token_at_a_time_is_the_same_as_all_at_once():
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn((2, 130, 2, 128), generator=gen, device=DEV).bfloat16()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    (one, two) = (KVCache.empty(3, 2, 128), KVCache.empty(3, 2, 128))
    for c in (one, two):
        for t in (c.keys, c.values, c.key_scales, c.value_scales, c.bounds, c.bound_scales):
            t.zero_()
    one.write(x[0], x[1], table, torch.zeros(1, dtype=torch.int32, device=DEV), ends([130]))
    for i in range(130):
        two.write(x[0, i:i + 1], x[1, i:i + 1], table, torch.tensor([i], dtype=torch.int32, device=DEV))
    for name in ("keys", "values", "key_scales", "value_scales", "bounds", "bound_scales"):
        assert torch.equal(getattr(one, name), getattr(two, name)), name


# ---- attention -----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 5, 16, 20])
def test_single_tokens(dim, group, dtype):
    """Lengths around the ends of blocks, none among them, a length that the table cuts; over garbage."""
    lengths = [0, 1, 2, 63, 64, 65, 128, 200, 333]
    cache, table, lengths, gen = filled(lengths, 2, dim, dim + group, dtype)
    q = queries_for(len(lengths), 2 * group, dim, gen, dtype)
    (out, lse) = attend(q, cache, table, lengths, return_lse=True)
    want = ref.attention(q, cache, table, lengths)
    ref.check_attention(out, want, dtype)
    assert torch.equal(lse.cpu().isneginf(), want[1].isneginf())
    some = ~want[1].isneginf()
    assert ((lse.cpu().double() - want[1]).abs() <= (want[2] + 16) * 2.0 ** -24)[some].all()
    assert torch.equal(out, attend(q, cache, table, lengths))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,heads,group", [(128, 2, 4), (64, 1, 7), (256, 1, 2), (96, 3, 1)])
def test_several_tokens(dim, heads, group, causal, dtype):
    """Rows of a sequence from none to more than its tokens (the first then see nothing)."""
    lengths = [70, 0, 5, 257, 64, 131]
    counts = [9, 0, 8, 40, 64, 1]
    cache, table, lengths, gen = filled(lengths, heads, dim, 17, dtype)
    q = queries_for(sum(counts), heads * group, dim, gen, dtype)
    out = attend(q, cache, table, lengths, offsets=ends(counts), causal=causal)
    ref.check_attention(out, ref.attention(q, cache, table, lengths, ends(counts), causal=causal), dtype)


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
def test_scales(scale):
    cache, table, lengths, gen = filled([300, 77], 2, 128, 4)
    q = queries_for(2, 8, 128, gen, torch.bfloat16)
    ref.check_attention(attend(q, cache, table, lengths, scale=scale), ref.attention(q, cache, table, lengths, scale=scale), torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores of thousands: one token has all the weight, and the maximum grows from block to block."""
    cache, table, lengths, gen = filled([640, 641], 1, 64, 6, dtype)
    q = queries_for(2, 3, 64, gen, dtype, 200.0)
    ref.check_attention(attend(q, cache, table, lengths), ref.attention(q, cache, table, lengths), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_that_are_not_finite(dtype):
    """They spoil the rows that see them and no others, in the same tile too."""
    cache, table, lengths, gen = filled([200, 90], 2, 64, 7, dtype)
    k = torch.randn((12, 2, 64), generator=gen, device=DEV).to(dtype)
    v = torch.randn((12, 2, 64), generator=gen, device=DEV).to(dtype)
    k[5, 0, 3] = math.nan
    v[7, 1, 60] = math.inf
    cache.write(k, v, table, lengths - 12, ends([12, 0]))
    q = queries_for(17, 8, 64, gen, dtype)
    out = attend(q, cache, table, lengths, offsets=ends([12, 5]))
    want = ref.attention(q, cache, table, lengths, ends([12, 5]))
    assert want[0][4].isfinite().all() and want[0][5, :4].isnan().all() and want[0][5, 4:].isfinite().all() and want[0][7].isnan().all()
    ref.check_attention(out, want, dtype)


def test_pages_that_hold_nothing_take_no_part():
    cache, table, lengths, gen = filled([300, 64], 2, 128, 9)
    table[0, 1] = MAXINT
    table[0, 4] = -3
    table[1, 0] = cache.pages
    q = queries_for(2, 4, 128, gen, torch.bfloat16)
    out = attend(q, cache, table, lengths)
    ref.check_attention(out, ref.attention(q, cache, table, lengths), torch.bfloat16)
    assert not out[1].any()


def test_strides_and_alignment():
    """Queries that lie between other things, off 16-byte boundaries, heads before rows; a table cut out of a wider one."""
    cache, table, lengths, gen = filled([300, 64, 130], 2, 64, 10)
    wide = torch.full((3, 11), -1, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + table.size(1)] = table
    cut = wide[:, 3:3 + table.size(1)]
    dense = queries_for(3, 6, 64, gen, torch.bfloat16)
    want = attend(dense, cache, table, lengths)
    mixed = torch.empty((3, 10, 67), dtype=torch.bfloat16, device=DEV)[:, 2:8, 1:65]
    turned = torch.empty((6, 3, 64), dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    for q in (mixed, turned):
        q.copy_(dense)
        assert torch.equal(attend(q, cache, cut, lengths), want)
        (out, blocks) = attend_selected(q, cache, cut, lengths, 2)
        (out2, blocks2) = attend_selected(dense, cache, table, lengths, 2)
        assert torch.equal(out, out2) and torch.equal(blocks, blocks2)


def test_parts_are_joined_by_their_sums():
    """Two halves of a context, each attended on its own, give the whole by lse."""
    cache, table, lengths, gen = filled([640], 2, 128, 11, torch.float32)
    q = queries_for(1, 8, 128, gen, torch.float32)
    (whole, lse) = attend(q, cache, table, lengths, return_lse=True)
    half = torch.tensor([320], dtype=torch.int32, device=DEV)
    (a, la) = attend(q, cache, table[:, :5], half, return_lse=True)
    (b, lb) = attend(q, cache, table[:, 5:].contiguous(), half, return_lse=True)
    both = torch.logaddexp(la, lb)
    assert torch.allclose(both, lse, rtol=0, atol=2e-5)
    assert torch.allclose(a * (la - both).exp()[..., None] + b * (lb - both).exp()[..., None], whole, rtol=0, atol=5e-5)


def test_a_cache_of_more_than_4_gib():
    """Pages whose bytes lie behind 2^32 and 2^33; one sequence also at the front."""
    (heads, dim, pages) = (1, 256, 1_100_000)  # 8 KiB of keys a page: 9 GB
    cache = KVCache.empty(pages, heads, dim)
    gen = torch.Generator(device=DEV).manual_seed(12)
    lengths = torch.tensor([150, 129], dtype=torch.int32, device=DEV)
    table = torch.tensor([[pages - 1, 3, 600_000], [524_288, 1_048_576, pages - 2]], dtype=torch.int32, device=DEV)
    x = torch.randn((2, 279, heads, dim), generator=gen, device=DEV).bfloat16()
    cache.write(x[0], x[1], table, torch.zeros(2, dtype=torch.int32, device=DEV), ends([150, 129]))
    (k, v) = cache.read(table, torch.zeros(2, dtype=torch.int32, device=DEV), 279, ends([150, 129]), dtype=torch.float32)
    assert torch.equal(k.cpu().double(), ref.rounded(x[0])) and torch.equal(v.cpu().double(), ref.rounded(x[1]))
    q = queries_for(2, 4, dim, gen, torch.bfloat16)
    ref.check_attention(attend(q, cache, table, lengths), ref.attention(q, cache, table, lengths), torch.bfloat16)
    (out, blocks) = attend_selected(q, cache, table, lengths, 2)
    assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, 2))
    ref.check_attention(out, ref.attention(q, cache, table, lengths, blocks=blocks), torch.bfloat16)


def test_a_long_context():
    """20,000 tokens, split over workgroups and joined."""
    cache, table, lengths, gen = filled([20_000, 70], 1, 128, 13)
    q = queries_for(2, 4, 128, gen, torch.bfloat16)
    ref.check_attention(attend(q, cache, table, lengths), ref.attention(q, cache, table, lengths), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_few_tokens_over_a_long_context(dtype):
    """Rows of one sequence that see differently many, tiles split over workgroups; 48 rows of a head are three tiles."""
    cache, table, lengths, gen = filled([5000, 3001], 2, 64, 14, dtype)
    q = queries_for(19, 6, 64, gen, dtype)
    out = attend(q, cache, table, lengths, offsets=ends([16, 3]))
    ref.check_attention(out, ref.attention(q, cache, table, lengths, ends([16, 3])), dtype)


@pytest.mark.parametrize("dim,group", [(64, 2), (128, 5), (96, 17)])
def test_so_many_tiles_that_every_wavefront_has_one(dim, group):
    lengths = [i * 37 % 150 for i in range(300)]
    cache, table, lengths, gen = filled(lengths, 8, dim, 16, blocks=3)
    q = queries_for(300, 8 * group, dim, gen, torch.bfloat16)
    (out, lse) = attend(q, cache, table, lengths, return_lse=True)
    some = torch.arange(0, 300, 7, device=DEV)  # the rest has the same code and the reference is slow
    want = ref.attention(q[some], cache, table[some], lengths[some])
    ref.check_attention(out[some], want, torch.bfloat16)
    assert torch.equal(lse[some].cpu().isneginf(), want[1].isneginf())
    (out, blocks) = attend_selected(q, cache, table, lengths, 2)
    assert torch.equal(blocks[some].cpu(), ref.selection(q[some], cache, table[some], lengths[some], 2))
    ref.check_attention(out[some], ref.attention(q[some], cache, table[some], lengths[some], blocks=blocks[some]), torch.bfloat16)


# ---- the choice of blocks ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 3, 16, 24])
def test_choice_of_single_tokens(dim, group, dtype):
    lengths = [0, 1, 64, 65, 640, 900, 1999]
    cache, table, lengths, gen = filled(lengths, 2, dim, dim + group, dtype)
    q = queries_for(len(lengths), 2 * group, dim, gen, dtype)
    for count in (1, 3, 8, 40):
        blocks = select_blocks(q, cache, table, lengths, count)
        assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, count)), count
    (out, blocks) = attend_selected(q, cache, table, lengths, 5)
    assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, 5))
    ref.check_attention(out, ref.attention(q, cache, table, lengths, blocks=blocks), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group", [(128, 2, 4), (96, 1, 6), (64, 2, 1), (256, 1, 17)])
def test_choice_of_several_tokens(dim, heads, group, dtype):
    lengths = [700, 0, 5, 450, 64]
    counts = [33, 0, 8, 130, 1]
    cache, table, lengths, gen = filled(lengths, heads, dim, 19, dtype)
    q = queries_for(sum(counts), heads * group, dim, gen, dtype)
    (out, blocks) = attend_selected(q, cache, table, lengths, 4, offsets=ends(counts))
    assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, 4, ends(counts)))
    ref.check_attention(out, ref.attention(q, cache, table, lengths, ends(counts), blocks=blocks), dtype)


def test_choice_among_many_blocks():
    """More blocks than a workgroup scores at once, counts up to all of them."""
    cache, table, lengths, gen = filled([64 * 1100 + 7, 64 * 300], 1, 32, 23)
    q = queries_for(2, 2, 32, gen, torch.bfloat16)
    for count in (1, 32, 257, 1100, 1101, 1500):
        blocks = select_blocks(q, cache, table, lengths, count)
        assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, count)), count


def test_ties_go_to_the_lower_block():
    cache = KVCache.empty(40, 1, 64)
    table = torch.randperm(40, device=DEV).to(torch.int32)[None]
    x = torch.ones((40 * 64, 1, 64), device=DEV)
    x[20 * 64] = 2.0  # one block is better than the rest
    cache.write(x, x, table, torch.zeros(1, dtype=torch.int32, device=DEV), ends([40 * 64]))
    lengths = torch.tensor([40 * 64], dtype=torch.int32, device=DEV)
    blocks = select_blocks(torch.ones((1, 4, 64), device=DEV), cache, table, lengths, 6)
    assert blocks.tolist() == [[[0, 1, 2, 3, 20, 39]]]
    # queries that are zero or not finite: all scores are zero
    for bad in (0.0, math.nan, math.inf):
        blocks = select_blocks(torch.full((1, 4, 64), bad, device=DEV), cache, table, lengths, 3)
        assert blocks.tolist() == [[[0, 1, 39]]]


def test_scores_below_zero():
    """A head's queries that fill no whole tile of 16: what is beside them is no score of zero."""
    for group in (3, 20):
        cache, table, lengths, gen = filled([1000], 1, 64, 29)
        x = 1 + torch.rand((1000, 1, 64), generator=gen, device=DEV)
        cache.write(x, x, table, torch.zeros(1, dtype=torch.int32, device=DEV), ends([1000]))
        q = -1 - torch.rand((1, group, 64), generator=gen, device=DEV)
        for count in (2, 7):
            assert torch.equal(select_blocks(q, cache, table, lengths, count).cpu(), ref.selection(q, cache, table, lengths, count))


def test_blocks_without_bounds_come_first():
    cache, table, lengths, gen = filled([1000], 2, 64, 31)
    bad = torch.full((1, 2, 64), math.nan, device=DEV, dtype=torch.bfloat16)
    bad[:, 1] = 1.0
    cache.write(bad, bad, table, torch.tensor([7 * 64], dtype=torch.int32, device=DEV))  # block 7 then holds one token
    q = queries_for(1, 4, 64, gen, torch.bfloat16)
    blocks = select_blocks(q, cache, table, lengths, 3)
    assert 7 in blocks[0, 0].tolist()
    assert torch.equal(blocks.cpu(), ref.selection(q, cache, table, lengths, 3))
    table[0, 3] = -1
    assert torch.equal(select_blocks(q, cache, table, lengths, 15).cpu(), ref.selection(q, cache, table, lengths, 15))


def test_lists_of_blocks_of_any_order():
    cache, table, lengths, gen = filled([1000, 128, 30], 2, 128, 37)
    q = queries_for(3, 8, 128, gen, torch.bfloat16)
    blocks = torch.tensor([[[15, 3, MAXINT, 0], [7, -1, 99, 2]], [[0, 1, 5, 6], [MAXINT] * 4], [[0, 1, 2, 3], [3, 2, 1, 0]]],
                          dtype=torch.int32, device=DEV)
    (out, lse) = attend_blocks(q, cache, table, lengths, blocks, return_lse=True)
    want = ref.attention(q, cache, table, lengths, blocks=blocks)
    ref.check_attention(out, want, torch.bfloat16)
    assert not out[1, 4:].any() and lse[1, 4:].isneginf().all()


# ---- how calls are made --------------------------------------------------------------------------

def test_empty_calls():
    cache = KVCache.empty(2, 2, 64)
    none = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    zero = torch.empty(0, dtype=torch.int32, device=DEV)
    kv = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    cache.write(kv, kv, none, zero)
    assert cache.read(none, zero, 0)[0].shape == (0, 2, 64)
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    assert attend(q, cache, none, zero).shape == (0, 4, 64)
    assert attend_selected(q, cache, none, zero, 3)[1].shape == (0, 2, 3)
    assert cache.read_bounds(zero).shape == (0, 2, 2, 64)
    # tables without a block, caches without a page
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=DEV)
    table = torch.empty((2, 0), dtype=torch.int32, device=DEV)
    lengths = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    assert not attend(q, cache, table, lengths).any()
    (out, blocks) = attend_selected(q, cache, table, lengths, 2)
    assert not out.any() and (blocks == MAXINT).all()
    nothing = KVCache.empty(0, 2, 64)
    table = torch.zeros((2, 1), dtype=torch.int32, device=DEV)
    nothing.write(q[:, :2], q[:, :2], table, lengths)
    assert not attend(q, nothing, table, lengths).any()


def test_on_a_stream_of_its_own():
    cache, table, lengths, gen = filled([3000, 400], 2, 128, 41)
    q = queries_for(2, 8, 128, gen, torch.bfloat16)
    want = attend_selected(q, cache, table, lengths, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            late = torch.empty_like(q)
            torch.cuda._sleep(1_000_000)
            late.copy_(q)  # the call has to wait for this
            (out, blocks) = attend_selected(late, cache, table, lengths, 4)
        side.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(blocks, want[1])


def test_captured_steps():
    """A step of an answer - write a token, attend to everything, attend to chosen blocks - as a graph, replayed with new inputs."""
    cache, table, lengths, gen = filled([3000, 401, 63], 2, 128, 43, blocks=48)
    (q, k, v) = (queries_for(3, n, 128, gen, torch.bfloat16) for n in (8, 2, 2))
    state = lengths.clone()

    def step():
        cache.write(k, v, table, state)
        state.add_(1)
        return (attend(q, cache, table, state), *attend_selected(q, cache, table, state, 4))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    state.copy_(lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for t in (q, k, v):
            t.normal_(generator=gen)
        before = lengths + i
        state.copy_(before)
        want = [t.clone() for t in step()]
        image = cache.keys.clone()
        state.copy_(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(cache.keys, image)
        assert torch.equal(state, before + 1)


def test_the_example_runs():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vectorlink-gpu_amd", "attend.py")
    spec = importlib.util.spec_from_file_location("attend_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    options = example.parse(["-c", "1500", "-b", "2", "-n", "2", "-d", "64", "-k", "8", "-p", "600", "-s", "4"])
    report = example.main(options)
    # codes of three magnitude bits: a quarter of a step of a sixth at most, and the token's subject dominates what is chosen
    assert report["blocks"] == 24 and 0.0 < report["keys_off"] < 0.2 and 0.0 < report["values_off"] < 0.2
    assert 0.0 < report["chosen_off"] < 1.0
    # all blocks chosen: the same tokens, joined in another order
    everything = example.main(dict(options, count=24))
    assert everything["chosen_off"] < 2.0 ** -7
