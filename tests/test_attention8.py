"""The cache in 8 bits without a GPU: calls that are refused on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from test_attention import BAD_QUERIES, BAD_TOKENS, queries, tokens
from vectorlink_gpu import _native as nv
from vectorlink_gpu import attention


@pytest.fixture(scope="module")
def lib():
    return nv.lib()


def cache(**kw):
    p = dict(pages=10, heads=2, dim=128, keys=256, values=256, scales=256, weights=256, positions=256)
    p.update(kw)
    return C.byref(nv.Cache8(**p))


BAD_CACHES = [dict(dim=80), dict(dim=0), dict(dim=512), dict(heads=0), dict(heads=70_000), dict(pages=-1), dict(pages=1 << 31), dict(keys=None),
              dict(values=None), dict(scales=None), dict(weights=None), dict(positions=None), dict(values=264), dict(weights=260)]
MUCH = 1 << 50


def write(lib, c, t, kind=1, keys=256, values=256, positions=None):
    return lib.vl_cache8_write(c, t, kind, keys, 256, 128, values, 256, 128, positions, None)


def test_cache_and_tokens_are_checked_by_every_call(lib):
    for c, t in [(cache(**kw), tokens()) for kw in BAD_CACHES] + [(cache(), tokens(**kw)) for kw in BAD_TOKENS] + [(None, tokens()), (cache(), None)]:
        assert write(lib, c, t) == -1
        assert lib.vl_cache8_read(c, t, 1, 256, 256, None) == -1
        for accumulate in (0, 1):
            assert lib.vl_attend8(c, t, queries(), accumulate, 256, MUCH, None) == -1
            assert lib.vl_attend8_workspace_bytes(c, t, queries(), accumulate) == -1
        assert lib.vl_attend8_form(c, t, queries()) == -1
        assert lib.vl_cache8_evict_workspace_bytes(c, t, 64) == -1
        assert lib.vl_cache8_evict(c, t, 64, 0, 256, 256, MUCH, None) == -1


def test_queries_are_checked(lib):
    for kw in BAD_QUERIES:
        assert lib.vl_attend8(cache(), tokens(), queries(**kw), 0, 256, MUCH, None) == -1
        assert lib.vl_attend8(cache(), tokens(), queries(**kw), 1, 256, MUCH, None) == -1
    assert lib.vl_attend8(cache(), tokens(), None, 0, 256, MUCH, None) == -1


def test_rows_that_are_written_or_read_are_checked(lib):
    assert write(lib, cache(), tokens(), kind=0) == -1 and write(lib, cache(), tokens(), kind=4) == -1
    assert write(lib, cache(), tokens(), keys=None) == -1 and write(lib, cache(), tokens(), kind=3, keys=258) == -1
    assert write(lib, cache(), tokens(), positions=258) == -1
    assert lib.vl_cache8_read(cache(), tokens(), 1, 256, 264, None) == -1
    assert lib.vl_cache8_read(cache(), tokens(), 5, 256, 256, None) == -1


def test_evictions_are_checked(lib):
    for keep, recent in ((-1, 0), (1 << 31, 0), (64, -1), (64, 65)):
        assert lib.vl_cache8_evict(cache(), tokens(), keep, recent, 256, 256, MUCH, None) == -1
    assert lib.vl_cache8_evict(cache(), tokens(), 64, 0, None, 256, MUCH, None) == -1
    for new in (1_024, 1_032, 1_016):  # three lengths of 4 bytes; other workgroups still read them
        assert lib.vl_cache8_evict(cache(), tokens(lengths=1_024), 64, 0, new, 256, MUCH, None) == -1 and b"overlap" in lib.vl_last_error()
    assert lib.vl_cache8_evict(cache(), tokens(offsets=256), 64, 0, 256, 256, MUCH, None) == -1
    plain = cache(weights=None, positions=None)
    assert lib.vl_cache8_evict(plain, tokens(), 64, 0, 256, 256, MUCH, None) == -1 and b"weights" in lib.vl_last_error()
    assert lib.vl_attend8(plain, tokens(), queries(), 1, 256, MUCH, None) == -1 and b"weights" in lib.vl_last_error()


def test_workspaces_are_checked(lib):
    t = tokens(blocks=40_000, table_stride=40_000)
    for accumulate in (0, 1):
        need = lib.vl_attend8_workspace_bytes(cache(), t, queries(), accumulate)
        assert need > 0 and need % 256 == 0
        assert lib.vl_attend8(cache(), t, queries(), accumulate, 256, need - 1, None) == -3 and b"workspace" in lib.vl_last_error()
        assert lib.vl_attend8(cache(), t, queries(), accumulate, 264, need, None) == -1
    need = lib.vl_cache8_evict_workspace_bytes(cache(), t, 64)
    assert need > 0 and need % 256 == 0
    assert lib.vl_cache8_evict(cache(), t, 64, 0, 256, 256, need - 1, None) == -3
    assert lib.vl_cache8_evict(cache(), t, 64, 0, 256, None, need, None) == -3
    assert lib.vl_cache8_evict(cache(), t, 64, 0, 256, 264, need, None) == -1
    # an eviction's lists are bounded by what stays and by half of what there is
    (one, all_) = (lib.vl_cache8_evict_workspace_bytes(cache(), t, keep) for keep in (1, (1 << 31) - 1))
    # two lists of 8 bytes an entry, the first hole of every block, and what workgroups that share a sequence and head tell each other
    (entries, chunks) = (40_000 * 64 // 2, -(-40_000 // 128))
    assert one < need < all_ < 3 * 2 * (2 * entries * 8 + 40_002 * 4 + chunks * (8 + 16 * 16) + 3 * 2048 * 4 + 2048)


def test_scores_take_4_gib_at_most(lib):
    """Tables of many blocks that mostly name nothing: weights are made from the keys once more."""
    def need(blocks):
        return lib.vl_attend8_workspace_bytes(cache(heads=8), tokens(rows=64, sequences=64, blocks=blocks, table_stride=blocks), queries(heads=32), 1)
    assert 1 << 32 <= need(8_192) < (1 << 32) + (1 << 28) and need(8_193) < 1 << 28


def test_a_cache_without_pages_keeps_no_scores(lib):
    """There would be no weights to add them to."""
    (few, wide) = (tokens(), tokens(blocks=40_000, table_stride=40_000))
    for t in (few, wide):
        assert lib.vl_attend8_workspace_bytes(cache(pages=0), t, queries(), 1) == lib.vl_attend8_workspace_bytes(cache(pages=0), t, queries(), 0)
        assert lib.vl_attend8_workspace_bytes(cache(), t, queries(), 1) > lib.vl_attend8_workspace_bytes(cache(), t, queries(), 0)


def test_calls_without_rows_succeed(lib):
    t = tokens(rows=0, sequences=0, table=None, lengths=None)
    assert lib.vl_cache8_write(cache(), t, 1, None, 0, 0, None, 0, 0, None, None) == 0
    assert lib.vl_cache8_read(cache(), t, 1, None, None, None) == 0
    assert lib.vl_attend8(cache(), t, queries(queries=None, out=None), 1, None, 0, None) == 0
    assert lib.vl_cache8_evict(cache(), t, 4, 0, None, None, 0, None) == 0


def on_cpu(pages=4, heads=2, dim=64):
    u8 = lambda *s: torch.zeros((pages, heads, *s), dtype=torch.uint8)
    return dict(keys=u8(64, dim), values=u8(16, dim, 4), scales=u8(4), weights=torch.zeros((pages, heads, 64)),
                positions=torch.zeros((pages, heads, 64), dtype=torch.int32))


def test_tensors_of_a_cache_are_checked():
    with pytest.raises(RuntimeError):
        attention.KVCache8(**on_cpu())  # right, but on the CPU
    with pytest.raises(RuntimeError):
        attention.KVCache8.empty(4, 2, 64, device="cpu")
    with pytest.raises(AssertionError):
        attention.KVCache8.empty(4, 2, 80, device="cpu")
    for name in on_cpu():
        for spoil in (lambda t: t.to(torch.int64), lambda t: t[:3], lambda t: torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype)[..., ::2]):
            parts = on_cpu()
            parts[name] = spoil(parts[name])
            with pytest.raises(AssertionError):
                attention.KVCache8(**parts)
    for name in ("weights", "positions"):
        parts = on_cpu()
        parts[name] = None
        with pytest.raises(AssertionError):
            attention.KVCache8(**parts)
    parts = on_cpu()
    parts["weights"].requires_grad_()
    with pytest.raises(AssertionError):
        attention.KVCache8(**parts)


def stands_for(weighted=True, pages=4, heads=2, dim=64):
    """A cache where only its sizes are looked at."""
    c = attention.KVCache8.__new__(attention.KVCache8)
    (c.pages, c.heads, c.dim, c._ref, c.gpu) = (pages, heads, dim, None, 0)
    c.weights = c.positions = torch.zeros((pages, heads, 64)) if weighted else None
    return c


def test_arguments_are_checked():
    (q, table, lengths) = (torch.zeros((3, 4, 64)), torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    c = stands_for()
    for spoil in (dict(queries=q[:, :3]), dict(queries=q[..., :32]), dict(table=table.float()), dict(lengths=lengths[:2]),
                  dict(queries=torch.zeros((3, 4, 64), requires_grad=True))):
        args = dict(queries=q, table=table, lengths=lengths)
        args.update(spoil)
        for accumulate in (False, True):
            with pytest.raises(AssertionError):
                attention.attend(args["queries"], c, args["table"], args["lengths"], accumulate=accumulate)
    with pytest.raises(AssertionError):  # before the GPU is looked for
        c.evict(table, lengths, 4, recent=5)
    with pytest.raises(AssertionError):
        c.evict(table, lengths, -1)
    with pytest.raises(AssertionError):
        c.evict(table, lengths[:2], 4)
    with pytest.raises(AssertionError):
        stands_for(weighted=False).evict(table, lengths, 4)
    kv = torch.zeros((3, 2, 64))
    with pytest.raises(AssertionError):
        stands_for(weighted=False).write(kv, kv, table, lengths, positions=lengths)
    for positions in (lengths[:2], lengths.long(), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(AssertionError):
            c.write(kv, kv, table, lengths, positions=positions)
    for f in (lambda: attention.select_blocks(q, c, table, lengths, 2), lambda: attention.attend_selected(q, c, table, lengths, 2),
              lambda: attention.attend_blocks(q, c, table, lengths, torch.zeros((3, 2, 2), dtype=torch.int32))):
        with pytest.raises(AssertionError, match="bounds"):
            f()
    for call in (lambda: attention.attend(q, c, table, lengths), lambda: c.evict(table, lengths, 4), lambda: c.write(kv, kv, table, lengths),
                 lambda: c.read(table, lengths, 3)):
        with pytest.raises(RuntimeError):  # right, but on the CPU
            call()
