"""Attention over a key/value cache held in 4 bits (no counterpart in the reference; include/vlgpu.h has the
formats and formulas).

    cache = KVCache.empty(pages, heads, dim)                  # pages of 64 tokens, for any number of sequences
    cache.write(keys, values, table, starts)                  # new tokens behind the `starts` tokens a sequence has
    out = attend(queries, cache, table, starts + 1)           # over everything
    out, blocks = attend_selected(queries, cache, table, starts + 1, count=32)   # over the 32 best blocks of each token

table [sequences, blocks] int32 names the page of each block of 64 tokens of a sequence.  Rows of keys, values and
queries are tokens; offsets [sequences + 1] int32 says which rows are whose (None: one row a sequence).  Everything is
enqueued on torch's current stream; nothing is synchronised, and no length is read on the host.
"""
import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native as nv

PAGE = 64  # tokens
DIMS = (32, 64, 96, 128, 192, 256)


def _check_int32(t: Tensor, name: str, size: int):
    assert t.dtype == torch.int32, f"{name} must be int32"
    assert t.dim() == 1 and t.numel() == size and (size < 2 or t.stride(0) == 1), f"{name} must be a contiguous tensor of {size}"


def _tokens(rows: int, table: Tensor, lengths: Tensor, offsets: Optional[Tensor]) -> nv.Tokens:
    assert table.dtype == torch.int32 and table.dim() == 2, "table must be int32 [sequences, blocks]"
    (sequences, blocks) = table.size()
    assert blocks < 2 or table.stride(1) == 1, "rows of table must be contiguous"
    _check_int32(lengths, "lengths", sequences)
    if offsets is None:
        assert rows == sequences, f"without offsets every sequence has one row: {rows} rows, {sequences} sequences"
        nv.require_gpu(table, lengths)
    else:
        _check_int32(offsets, "offsets", sequences + 1)
        nv.require_gpu(table, lengths, offsets)
    return nv.Tokens(rows, sequences, blocks, table.stride(0) if sequences > 1 else blocks, table.data_ptr(), lengths.data_ptr(),
                     None if offsets is None else offsets.data_ptr())


def _check_rows(t: Tensor, name: str, dim: int) -> int:
    assert t.dim() == 3 and t.size(2) == dim, f"{name} must be [rows, heads, {dim}]"
    assert t.stride(2) == 1, f"the last dimension of {name} must be contiguous"
    assert t.dtype in nv.TYPES, f"{name} must be bfloat16, float16 or float32"
    return nv.TYPES[t.dtype]


class KVCache:
    """Keys and values of 4 bits in pages of 64 tokens, with the bounds of every page's keys, over tensors of the caller's (their
    shapes are those of KVCache.empty)."""

    def __init__(self, keys: Tensor, key_scales: Tensor, values: Tensor, value_scales: Tensor, bounds: Tensor, bound_scales: Tensor):
        assert keys.dim() == 4 and keys.size(2) == PAGE, "keys must be uint8 [pages, heads, 64, dim / 2]"
        (pages, heads, _, half) = keys.size()
        dim = 2 * half
        assert dim in DIMS, f"dim must be one of {DIMS}, got {dim}"
        scales = (pages, heads, dim // 32, PAGE)
        for (t, name, dtype, shape) in ((keys, "keys", torch.uint8, (pages, heads, PAGE, half)),
                                        (key_scales, "key_scales", torch.uint8, scales),
                                        (values, "values", torch.uint8, (pages, heads, PAGE // 4, dim // 8, 4, 4)),
                                        (value_scales, "value_scales", torch.uint8, scales),
                                        (bounds, "bounds", torch.int8, (pages, heads, 2, dim)),
                                        (bound_scales, "bound_scales", torch.int8, (pages, heads))):
            assert t.dtype == dtype and tuple(t.shape) == shape, f"{name} must be {dtype} {shape}"
            assert t.is_contiguous(), f"{name} must be contiguous"
        nv.require_gpu(keys, key_scales, values, value_scales, bounds, bound_scales)
        (self.keys, self.key_scales, self.values, self.value_scales) = (keys, key_scales, values, value_scales)
        (self.bounds, self.bound_scales) = (bounds, bound_scales)
        (self.pages, self.heads, self.dim) = (pages, heads, dim)
        self._native = nv.Cache(pages, heads, dim, *(t.data_ptr() for t in (keys, key_scales, values, value_scales, bounds, bound_scales)))
        self._ref = C.byref(self._native)

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, device="cuda") -> "KVCache":
        """A cache of `pages` pages; dim + dim / 16 bytes a token and head, and 2 dim + 1 a page and head."""
        assert dim in DIMS, f"dim must be one of {DIMS}, got {dim}"

        def part(*shape, dtype=torch.uint8):
            return torch.empty((pages, heads, *shape), dtype=dtype, device=device)

        return cls(part(PAGE, dim // 2), part(dim // 32, PAGE), part(PAGE // 4, dim // 8, 4, 4), part(dim // 32, PAGE),
                   part(2, dim, dtype=torch.int8), part(dtype=torch.int8))

    def write(self, keys: Tensor, values: Tensor, table: Tensor, starts: Tensor, offsets: Optional[Tensor] = None):
        """Quantise keys and values [rows, heads, dim] behind the `starts` [sequences] tokens that the sequences hold, and make
        the bounds of the blocks written into anew.  Writing again at an earlier place is allowed and takes back what was behind."""
        kind = _check_rows(keys, "keys", self.dim)
        assert _check_rows(values, "values", self.dim) == kind and values.size() == keys.size(), "keys and values differ in type or size"
        assert keys.size(1) == self.heads, f"keys have {keys.size(1)} heads, the cache {self.heads}"
        tokens = _tokens(keys.size(0), table, starts, offsets)
        nv.require_gpu(keys, values)
        nv.check(nv.lib().vl_cache_write(self._ref, C.byref(tokens), kind, keys.data_ptr(), keys.stride(0), keys.stride(1),
                                         values.data_ptr(), values.stride(0), values.stride(1), nv.stream()))

    def read(self, table: Tensor, starts: Tensor, rows: int, offsets: Optional[Tensor] = None,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
        """The keys and values [rows, heads, dim] that the cache holds from place `starts` of every sequence on: what write put
        there, rounded.  rows is the last of offsets, or the number of sequences."""
        assert dtype in nv.TYPES, "dtype must be bfloat16, float16 or float32"
        tokens = _tokens(rows, table, starts, offsets)
        keys = torch.empty((rows, self.heads, self.dim), dtype=dtype, device=self.keys.device)
        values = torch.empty_like(keys)
        nv.check(nv.lib().vl_cache_read(self._ref, C.byref(tokens), nv.TYPES[dtype], keys.data_ptr(), values.data_ptr(), nv.stream()))
        return (keys, values)

    def read_bounds(self, pages: Tensor) -> Tensor:
        """The largest and the smallest key of these pages in each dimension, rounded outwards: [*pages.shape, heads, 2, dim]."""
        assert pages.dtype == torch.int32, "pages must be int32"
        nv.require_gpu(pages)
        pages = pages.contiguous()
        out = torch.empty((*pages.shape, self.heads, 2, self.dim), dtype=torch.float32, device=pages.device)
        nv.check(nv.lib().vl_cache_read_bounds(self._ref, pages.data_ptr(), pages.numel(), out.data_ptr(), nv.stream()))
        return out


class _Call:
    """The checked arguments of a call with queries, as the library takes them."""

    def __init__(self, queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, offsets: Optional[Tensor],
                 scale: Optional[float] = None, causal: bool = True, output: bool = True, lse: bool = False):
        kind = _check_rows(queries, "queries", cache.dim)
        (rows, heads, dim) = queries.size()
        assert heads > 0 and heads % cache.heads == 0, f"{heads} heads of queries for {cache.heads} of the cache"
        self.tokens = _tokens(rows, table, lengths, offsets)
        nv.require_gpu(queries)
        self.out = torch.empty((rows, heads, dim), dtype=queries.dtype, device=queries.device) if output else None
        self.lse = torch.empty((rows, heads), dtype=torch.float32, device=queries.device) if lse else None
        self.native = nv.Queries(heads, queries.stride(0), queries.stride(1), queries.data_ptr(),
                                 self.out.data_ptr() if output else None, self.lse.data_ptr() if lse else None,
                                 dim ** -0.5 if scale is None else scale, kind, int(causal))
        self.args = (cache._ref, C.byref(self.tokens), C.byref(self.native))
        self.device = queries.device

    def workspace(self, need: int):
        """(pointer, bytes), kept with the call"""
        need = nv.check(need)
        if need == 0:
            return (None, 0)
        self.scratch = torch.empty(need, dtype=torch.uint8, device=self.device)
        return (self.scratch.data_ptr(), need)

    def blocks(self, cache: KVCache, count: int) -> Tensor:
        assert count >= 1, f"count: {count}"
        return torch.empty((self.tokens.rows, cache.heads, count), dtype=torch.int32, device=self.device)

    def result(self):
        return self.out if self.lse is None else (self.out, self.lse)


def attend(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None,
           scale: Optional[float] = None, causal: bool = True, return_lse: bool = False):
    """softmax(scale * queries keys^T) values over the `lengths` [sequences] tokens that the cache holds.  queries [rows, heads,
    dim], heads a multiple of the cache's; scale defaults to dim ** -0.5.  The rows of a sequence are its last tokens and see
    what stands before them and themselves, or with causal=False everything.  A row that sees nothing gives zeros.  With
    return_lse also the logarithms of the sums of exponentials [rows, heads], by which parts of an attention are joined."""
    call = _Call(queries, cache, table, lengths, offsets, scale, causal, lse=return_lse)
    lib = nv.lib()
    ws = call.workspace(lib.vl_attend_workspace_bytes(*call.args))
    nv.check(lib.vl_attend(*call.args, *ws, nv.stream()))
    return call.result()


def select_blocks(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, count: int,
                  offsets: Optional[Tensor] = None) -> Tensor:
    """For every row and head of the cache `count` blocks of its sequence, ascending: the row's own and those with the highest
    upper bound on a score in them, by queries and bounds of 8 bits; MAXINT where there are no more.  [rows, cache.heads, count]"""
    call = _Call(queries, cache, table, lengths, offsets, output=False)
    lib = nv.lib()
    blocks = call.blocks(cache, count)
    ws = call.workspace(lib.vl_select_blocks_workspace_bytes(*call.args, count))
    nv.check(lib.vl_select_blocks(*call.args, count, blocks.data_ptr(), *ws, nv.stream()))
    return blocks


def attend_blocks(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, blocks: Tensor,
                  offsets: Optional[Tensor] = None, scale: Optional[float] = None, return_lse: bool = False):
    """attend over the tokens of blocks [rows, cache.heads, count] alone, up to the row's own place."""
    call = _Call(queries, cache, table, lengths, offsets, scale, lse=return_lse)
    assert blocks.dtype == torch.int32 and blocks.is_contiguous(), "blocks must be contiguous int32"
    assert blocks.dim() == 3 and blocks.size(0) == queries.size(0) and blocks.size(1) == cache.heads and blocks.size(2) > 0, \
        "blocks must be [rows, cache.heads, count]"
    nv.require_gpu(blocks)
    lib = nv.lib()
    count = blocks.size(2)
    ws = call.workspace(lib.vl_attend_blocks_workspace_bytes(*call.args, count))
    nv.check(lib.vl_attend_blocks(*call.args, blocks.data_ptr(), count, *ws, nv.stream()))
    return call.result()


def attend_selected(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, count: int,
                    offsets: Optional[Tensor] = None, scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """(attend_blocks(...), blocks) with the blocks of select_blocks, in one call."""
    call = _Call(queries, cache, table, lengths, offsets, scale)
    lib = nv.lib()
    blocks = call.blocks(cache, count)
    ws = call.workspace(lib.vl_attend_selected_workspace_bytes(*call.args, count))
    nv.check(lib.vl_attend_selected(*call.args, count, blocks.data_ptr(), *ws, nv.stream()))
    return (call.out, blocks)
