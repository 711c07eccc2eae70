"""Attention over the cache without a GPU: calls that are refused on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from vectorlink_gpu import _native as nv
from vectorlink_gpu import attention


@pytest.fixture(scope="module")
def lib():
    return nv.lib()


def cache(**kw):
    p = dict(pages=10, heads=2, dim=128, keys=256, key_scales=256, values=256, value_scales=256, bounds=256, bound_scales=256)
    p.update(kw)
    return C.byref(nv.Cache(**p))


def tokens(**kw):
    p = dict(rows=3, sequences=3, blocks=4, table_stride=4, table=256, lengths=256, offsets=None)
    p.update(kw)
    return C.byref(nv.Tokens(**p))


def queries(**kw):
    p = dict(heads=8, row_stride=1024, head_stride=128, queries=256, out=256, lse=None, scale=1.0, type=1, causal=1, form=0)
    p.update(kw)
    return C.byref(nv.Queries(**p))


BAD_CACHES = [dict(dim=80), dict(dim=0), dict(dim=512), dict(heads=0), dict(heads=70_000), dict(pages=-1), dict(keys=None),
              dict(bounds=None), dict(values=264)]
BAD_TOKENS = [dict(rows=-1), dict(rows=4), dict(sequences=-1), dict(blocks=-1), dict(table_stride=3), dict(table=None), dict(lengths=None),
              dict(rows=3, sequences=0, offsets=256)]
BAD_QUERIES = [dict(heads=3), dict(heads=0), dict(type=0), dict(type=4), dict(queries=None), dict(out=None), dict(queries=257),
               dict(out=264), dict(scale=float("nan")), dict(scale=float("inf")), dict(form=3), dict(form=-1)]


def test_cache_and_tokens_are_checked_by_every_call(lib):
    for c, t in [(cache(**kw), tokens()) for kw in BAD_CACHES] + [(cache(), tokens(**kw)) for kw in BAD_TOKENS]:
        assert lib.vl_cache_write(c, t, 1, 256, 256, 128, 256, 256, 128, None) == -1
        assert lib.vl_cache_read(c, t, 1, 256, 256, None) == -1
        assert lib.vl_attend(c, t, queries(), 256, 1 << 40, None) == -1
        assert lib.vl_attend_workspace_bytes(c, t, queries()) == -1
        assert lib.vl_select_blocks(c, t, queries(), 4, 256, 256, 1 << 40, None) == -1
        assert lib.vl_attend_blocks(c, t, queries(), 256, 4, 256, 1 << 40, None) == -1
        assert lib.vl_attend_selected(c, t, queries(), 4, 256, 256, 1 << 40, None) == -1
    for kw in BAD_CACHES:
        assert lib.vl_cache_read_bounds(cache(**kw), 256, 1, 256, None) == -1
    assert lib.vl_attend(None, tokens(), queries(), 256, 1 << 40, None) == -1
    assert lib.vl_attend(cache(), None, queries(), 256, 1 << 40, None) == -1
    assert lib.vl_attend(cache(), tokens(), None, 256, 1 << 40, None) == -1


def test_queries_are_checked(lib):
    for kw in BAD_QUERIES:
        assert lib.vl_attend(cache(), tokens(), queries(**kw), 256, 1 << 40, None) == -1
        assert lib.vl_attend_blocks(cache(), tokens(), queries(**kw), 256, 4, 256, 1 << 40, None) == -1
        assert lib.vl_attend_selected(cache(), tokens(), queries(**kw), 4, 256, 256, 1 << 40, None) == -1
    for count in (0, -1, 1 << 30):
        assert lib.vl_select_blocks(cache(), tokens(), queries(), count, 256, 256, 1 << 40, None) == -1
        assert lib.vl_attend_blocks(cache(), tokens(), queries(), 256, count, 256, 1 << 40, None) == -1
    assert lib.vl_select_blocks(cache(), tokens(), queries(), 4, None, 256, 1 << 40, None) == -1
    assert lib.vl_attend_blocks(cache(), tokens(), queries(), None, 4, 256, 1 << 40, None) == -1


def test_rows_that_are_written_or_read_are_checked(lib):
    assert lib.vl_cache_write(cache(), tokens(), 0, 256, 256, 128, 256, 256, 128, None) == -1
    assert lib.vl_cache_write(cache(), tokens(), 1, None, 256, 128, 256, 256, 128, None) == -1
    assert lib.vl_cache_write(cache(), tokens(), 3, 258, 256, 128, 256, 256, 128, None) == -1
    assert lib.vl_cache_read(cache(), tokens(), 1, 256, 264, None) == -1
    assert lib.vl_cache_read_bounds(cache(), None, 1, 256, None) == -1
    assert lib.vl_cache_read_bounds(cache(), 256, -1, 256, None) == -1


def test_workspaces_are_checked(lib):
    t = tokens(blocks=40_000, table_stride=40_000)
    sizes = [(lib.vl_attend_workspace_bytes(cache(), t, queries()), lambda n: lib.vl_attend(cache(), t, queries(), 256, n, None)),
             (lib.vl_select_blocks_workspace_bytes(cache(), t, queries(), 4),
              lambda n: lib.vl_select_blocks(cache(), t, queries(), 4, 256, 256, n, None)),
             (lib.vl_attend_blocks_workspace_bytes(cache(), t, queries(), 40),
              lambda n: lib.vl_attend_blocks(cache(), t, queries(), 256, 40, 256, n, None))]
    for need, call in sizes:
        assert need > 0 and need % 256 == 0
        assert call(need - 1) == -3 and b"workspace" in lib.vl_last_error()
    both = lib.vl_attend_selected_workspace_bytes(cache(), t, queries(), 40)
    assert both == sizes[1][0] + sizes[2][0]
    assert lib.vl_attend_selected(cache(), t, queries(), 40, 256, 256, sizes[1][0] - 1, None) == -3


def test_form_by_sizes(lib):
    """Single tokens and a few go to the one form, prompts to the other where it is there."""
    def form(rows, length, type=1, dim=128, heads=8, group=4, batch=1, **kw):
        blocks = -(-length // 64)
        t = tokens(rows=rows * batch, sequences=batch, blocks=blocks, table_stride=blocks, offsets=None if rows == 1 else 256)
        return lib.vl_attend_form(cache(dim=dim, heads=heads), t, queries(heads=heads * group, type=type, **kw))

    (few, many) = (1, 2)
    assert form(1, 131_072) == few and form(1, 8192, batch=64) == few and form(5, 2050, type=3, dim=256) == few
    assert form(2048, 16_384) == many and form(2048, 16_384, dim=256) == many and form(2048, 8192, type=2) == many
    assert form(2048, 8192, type=3, dim=64) == many
    assert form(2048, 8192, type=3) == few and form(2048, 8192, type=2, dim=192) == few
    assert form(1, 64, form=many) == many and form(2048, 16_384, form=few) == few
    assert form(2048, 8192, type=3, form=many) == -1


def test_calls_without_rows_succeed(lib):
    t = tokens(rows=0, sequences=0, table=None, lengths=None)
    assert lib.vl_cache_write(cache(), t, 1, None, 0, 0, None, 0, 0, None) == 0
    assert lib.vl_cache_read(cache(), t, 1, None, None, None) == 0
    assert lib.vl_attend(cache(), t, queries(queries=None, out=None), None, 0, None) == 0
    assert lib.vl_attend_selected(cache(), t, queries(queries=None, out=None), 4, None, None, 0, None) == 0


def on_cpu(pages=4, heads=2, dim=64):
    """A cache's tensors that never leave the host: enough for what is refused before the GPU is looked for."""
    u8 = lambda *s: torch.zeros((pages, heads, *s), dtype=torch.uint8)
    i8 = lambda *s: torch.zeros((pages, heads, *s), dtype=torch.int8)
    return dict(keys=u8(64, dim // 2), key_scales=u8(dim // 32, 64), values=u8(16, dim // 8, 4, 4), value_scales=u8(dim // 32, 64),
                bounds=i8(2, dim), bound_scales=i8())


def test_tensors_of_a_cache_are_checked():
    with pytest.raises(RuntimeError):
        attention.KVCache(**on_cpu())  # right, but on the CPU
    with pytest.raises(RuntimeError):
        attention.KVCache.empty(4, 2, 64, device="cpu")
    with pytest.raises(AssertionError):
        attention.KVCache.empty(4, 2, 80, device="cpu")
    for name in on_cpu():
        for spoil in (lambda t: t.to(torch.int32), lambda t: t[:3], lambda t: torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype)[..., ::2]):
            parts = on_cpu()
            parts[name] = spoil(parts[name])
            with pytest.raises(AssertionError):
                attention.KVCache(**parts)


class Dims:
    """Stands for a cache where only its sizes are looked at."""
    (pages, heads, dim) = (4, 2, 64)
    _ref = None


@pytest.mark.parametrize("spoil", [dict(queries=torch.zeros((3, 3, 64))), dict(queries=torch.zeros((3, 4, 32))),
                                   dict(queries=torch.zeros((3, 4, 64), dtype=torch.float64)), dict(queries=torch.zeros((3, 4, 128))[..., ::2]),
                                   dict(queries=torch.zeros((2, 4, 64))), dict(table=torch.zeros((3, 4))),
                                   dict(table=torch.zeros((3, 8), dtype=torch.int32)[:, ::2]), dict(table=torch.zeros(3, dtype=torch.int32)),
                                   dict(lengths=torch.zeros(2, dtype=torch.int32)), dict(lengths=torch.zeros(3, dtype=torch.int64)),
                                   dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), dict(offsets=torch.zeros(3, dtype=torch.int32))])
def test_arguments_of_attention_are_checked(spoil):
    args = dict(queries=torch.zeros((3, 4, 64)), table=torch.zeros((3, 4), dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32),
                offsets=None)
    args.update(spoil)
    call = (args["queries"], Dims, args["table"], args["lengths"])
    for f in (lambda: attention.attend(*call, offsets=args["offsets"]),
              lambda: attention.select_blocks(*call, 2, offsets=args["offsets"]),
              lambda: attention.attend_selected(*call, 2, offsets=args["offsets"])):
        with pytest.raises(AssertionError):
            f()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        attention.attend(torch.zeros((3, 4, 64)), Dims, torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
