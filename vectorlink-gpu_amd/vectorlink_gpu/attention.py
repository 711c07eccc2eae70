"""Attention over a key/value cache held in 4 or 8 bits (no counterpart in the reference; include/vlgpu.h has the
formats and formulas).

    cache = KVCache.empty(pages, heads, dim)                  # pages of 64 tokens, for any number of sequences
    cache.write(keys, values, table, starts)                  # new tokens behind the `starts` tokens a sequence has
    out = attend(queries, cache, table, starts + 1)           # over everything
    out, blocks = attend_selected(queries, cache, table, starts + 1, count=32)   # over the 32 best blocks of each token

    cache = KVCache8.empty(pages, heads, dim, weighted=True)  # twice the bytes, and weights of its tokens
    out = attend(queries, cache, table, lengths, accumulate=True)     # adds the weights that the queries give the tokens
    lengths = cache.evict(table, lengths, keep=4096, recent=256)      # the 4,096 that got most, and the latest, stay

table [sequences, blocks] int32 names the page of each block of 64 tokens of a sequence.  Rows of keys, values and
queries are tokens; offsets [sequences + 1] int32 says which rows are whose (None: one row a sequence).  Everything is
enqueued on torch's current stream; nothing is synchronised, and no length is read on the host.  There are no gradients: what
asks for one is refused.
"""
import ctypes as C
import struct
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _native as nv

PAGE = 64  # tokens
DIMS = (32, 64, 96, 128, 192, 256)
# A call's vl_tokens and vl_queries as bytes: a third of the time of a ctypes structure, which a single token's call notices
_TOKENS = struct.Struct("@qqqqPPP")
_QUERIES = struct.Struct("@qqqPPPdiiq")
assert _TOKENS.size == C.sizeof(nv.Tokens) and _QUERIES.size == C.sizeof(nv.Queries)


def _tokens(rows: int, table: Tensor, lengths: Tensor, offsets: Optional[Tensor]) -> bytes:
    assert table.dtype == torch.int32 and table.dim() == 2, "table must be int32 [sequences, blocks]"
    (sequences, blocks) = table.shape
    (stride, one) = table.stride()
    assert one == 1 or blocks < 2, "rows of table must be contiguous"
    assert lengths.dtype == torch.int32 and lengths.shape == (sequences,) and lengths.is_contiguous(), \
        f"lengths must be a contiguous int32 tensor of {sequences}"
    if offsets is None:
        assert rows == sequences, f"without offsets every sequence has one row: {rows} rows, {sequences} sequences"
        at = 0
    else:
        assert offsets.dtype == torch.int32 and offsets.shape == (sequences + 1,) and offsets.is_contiguous(), \
            f"offsets must be a contiguous int32 tensor of {sequences + 1}"
        at = offsets.data_ptr()
    return _TOKENS.pack(rows, sequences, blocks, stride if sequences > 1 else blocks, table.data_ptr(), lengths.data_ptr(), at)


def _check_rows(t: Tensor, name: str, dim: int) -> int:
    assert t.dim() == 3 and t.shape[2] == dim, f"{name} must be [rows, heads, {dim}]"
    assert t.stride(2) == 1, f"the last dimension of {name} must be contiguous"
    assert t.dtype in nv.TYPES, f"{name} must be bfloat16, float16 or float32"
    assert not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient, and there is none through a cache in few bits: call under no_grad"
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
        self.gpu = nv.require_one_gpu(keys, key_scales, values, value_scales, bounds, bound_scales)
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
        assert _check_rows(values, "values", self.dim) == kind and values.shape == keys.shape, "keys and values differ in type or size"
        assert keys.shape[1] == self.heads, f"keys have {keys.shape[1]} heads, the cache {self.heads}"
        tokens = _tokens(keys.shape[0], table, starts, offsets)
        gpu = nv.require_one_gpu(keys, values, table, starts, offsets)
        nv.check(nv.lib().vl_cache_write(self._ref, tokens, kind, keys.data_ptr(), keys.stride(0), keys.stride(1),
                                         values.data_ptr(), values.stride(0), values.stride(1), nv.stream_on(gpu, self.gpu)))

    def read(self, table: Tensor, starts: Tensor, rows: int, offsets: Optional[Tensor] = None,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
        """The keys and values [rows, heads, dim] that the cache holds from place `starts` of every sequence on: what write put
        there, rounded.  rows is the last of offsets, or the number of sequences."""
        assert dtype in nv.TYPES, "dtype must be bfloat16, float16 or float32"
        tokens = _tokens(rows, table, starts, offsets)
        gpu = nv.require_one_gpu(table, starts, offsets)
        keys = torch.empty((rows, self.heads, self.dim), dtype=dtype, device=self.keys.device)
        values = torch.empty_like(keys)
        nv.check(nv.lib().vl_cache_read(self._ref, tokens, nv.TYPES[dtype], keys.data_ptr(), values.data_ptr(), nv.stream_on(gpu, self.gpu)))
        return (keys, values)

    def read_bounds(self, pages: Tensor) -> Tensor:
        """The largest and the smallest key of these pages in each dimension, rounded outwards: [*pages.shape, heads, 2, dim]."""
        assert pages.dtype == torch.int32, "pages must be int32"
        gpu = nv.require_one_gpu(pages)
        pages = pages.contiguous()
        out = torch.empty((*pages.shape, self.heads, 2, self.dim), dtype=torch.float32, device=pages.device)
        nv.check(nv.lib().vl_cache_read_bounds(self._ref, pages.data_ptr(), pages.numel(), out.data_ptr(), nv.stream_on(gpu, self.gpu)))
        return out


class KVCache8:
    """Keys and values of 8 bits in pages of 64 tokens, with a power of two for each page and head, over tensors of the caller's (their
    shapes are those of KVCache8.empty).  weights and positions are there for a cache that tokens are evicted from, or None.  Tokens
    of a sequence differ from head to head once some have left; positions says which they are."""

    def __init__(self, keys: Tensor, values: Tensor, scales: Tensor, weights: Optional[Tensor] = None, positions: Optional[Tensor] = None):
        assert keys.dim() == 4 and keys.size(2) == PAGE, "keys must be uint8 [pages, heads, 64, dim]"
        (pages, heads, _, dim) = keys.size()
        assert dim in DIMS, f"dim must be one of {DIMS}, got {dim}"
        assert (weights is None) == (positions is None), "weights and positions are there together or not at all"
        for (t, name, dtype, shape) in ((keys, "keys", torch.uint8, (pages, heads, PAGE, dim)),
                                        (values, "values", torch.uint8, (pages, heads, PAGE // 4, dim, 4)),
                                        (scales, "scales", torch.uint8, (pages, heads, 4)),
                                        (weights, "weights", torch.float32, (pages, heads, PAGE)),
                                        (positions, "positions", torch.int32, (pages, heads, PAGE))):
            if t is None:
                continue
            assert t.dtype == dtype and tuple(t.shape) == shape, f"{name} must be {dtype} {shape}"
            assert t.is_contiguous(), f"{name} must be contiguous"
            assert not t.requires_grad, f"{name} requires a gradient, and the cache is written in place"
        self.gpu = nv.require_one_gpu(keys, values, scales, weights, positions)
        (self.keys, self.values, self.scales, self.weights, self.positions) = (keys, values, scales, weights, positions)
        (self.pages, self.heads, self.dim) = (pages, heads, dim)
        self._native = nv.Cache8(pages, heads, dim, *(0 if t is None else t.data_ptr() for t in (keys, values, scales, weights, positions)))
        self._ref = C.byref(self._native)

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, device="cuda", weighted: bool = False) -> "KVCache8":
        """A cache of `pages` pages; 2 dim bytes a token and head, 8 more if weighted, and 4 a page and head."""
        assert dim in DIMS, f"dim must be one of {DIMS}, got {dim}"

        def part(*shape, dtype=torch.uint8):
            return torch.empty((pages, heads, *shape), dtype=dtype, device=device)

        return cls(part(PAGE, dim), part(PAGE // 4, dim, 4), part(4), part(PAGE, dtype=torch.float32) if weighted else None,
                   part(PAGE, dtype=torch.int32) if weighted else None)

    def write(self, keys: Tensor, values: Tensor, table: Tensor, starts: Tensor, offsets: Optional[Tensor] = None,
              positions: Optional[Tensor] = None):
        """Round keys and values [rows, heads, dim] behind the `starts` [sequences] tokens that the sequences hold.  A page's power of
        two grows with its largest element, and what it holds is rounded to it again.  In a weighted cache the new tokens have weight 0
        and stand at positions [rows] of their texts (None: where they are written; say so once a sequence has had tokens evicted)."""
        kind = _check_rows(keys, "keys", self.dim)
        assert _check_rows(values, "values", self.dim) == kind and values.shape == keys.shape, "keys and values differ in type or size"
        assert keys.shape[1] == self.heads, f"keys have {keys.shape[1]} heads, the cache {self.heads}"
        at = 0
        if positions is not None:
            assert self.positions is not None, "the cache keeps no positions: weighted=True"
            assert positions.dtype == torch.int32 and positions.shape == keys.shape[:1] and positions.is_contiguous(), \
                f"positions must be a contiguous int32 tensor of {keys.shape[0]}"
            at = positions.data_ptr()
        tokens = _tokens(keys.shape[0], table, starts, offsets)
        gpu = nv.require_one_gpu(keys, values, table, starts, offsets, positions)
        nv.check(nv.lib().vl_cache8_write(self._ref, tokens, kind, keys.data_ptr(), keys.stride(0), keys.stride(1),
                                          values.data_ptr(), values.stride(0), values.stride(1), at, nv.stream_on(gpu, self.gpu)))

    def read(self, table: Tensor, starts: Tensor, rows: int, offsets: Optional[Tensor] = None,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
        """KVCache.read of this cache."""
        assert dtype in nv.TYPES, "dtype must be bfloat16, float16 or float32"
        tokens = _tokens(rows, table, starts, offsets)
        gpu = nv.require_one_gpu(table, starts, offsets)
        keys = torch.empty((rows, self.heads, self.dim), dtype=dtype, device=self.keys.device)
        values = torch.empty_like(keys)
        nv.check(nv.lib().vl_cache8_read(self._ref, tokens, nv.TYPES[dtype], keys.data_ptr(), values.data_ptr(), nv.stream_on(gpu, self.gpu)))
        return (keys, values)

    def evict(self, table: Tensor, lengths: Tensor, keep: int, recent: int = 0) -> Tensor:
        """Cut sequences of more than `keep` tokens down to that many, in each head those that count most: the `recent` latest positions,
        then the largest weights, of equal ones the earlier.  Tokens that stay move into the places of those that leave, so that a
        sequence's first places hold them, in no order that attention would depend on.  No page may stand twice in the table, and every
        block before the new length needs one: what would move to a place on no page is lost.  The lengths [sequences] that are left."""
        assert self.weights is not None, "the cache keeps no weights: weighted=True"
        assert 0 <= recent <= keep < 1 << 31, f"recent: {recent} of {keep} that stay"
        tokens = _tokens(table.shape[0], table, lengths, None)
        gpu = nv.require_one_gpu(table, lengths)
        left = torch.empty_like(lengths)
        lib = nv.lib()
        need = lib.vl_cache8_evict_workspace_bytes(self._ref, tokens, keep)
        ws = _workspace(need, table)
        nv.check(lib.vl_cache8_evict(self._ref, tokens, keep, recent, left.data_ptr(), nv.ptr(ws), need, nv.stream_on(gpu, self.gpu)))
        return left


def _queries(queries: Tensor, cache: Union[KVCache, KVCache8], scale: Optional[float], causal: bool, out: Optional[Tensor],
             lse: Optional[Tensor], form: Optional[str] = None) -> bytes:
    (row, head, _) = queries.stride()
    return _QUERIES.pack(queries.shape[1], row, head, queries.data_ptr(), 0 if out is None else out.data_ptr(),
                         0 if lse is None else lse.data_ptr(), cache.dim ** -0.5 if scale is None else scale,
                         nv.TYPES[queries.dtype], causal, 0 if form is None else nv.ATTEND_FORMS[form])


def _check_queries(queries: Tensor, cache: Union[KVCache, KVCache8]):
    _check_rows(queries, "queries", cache.dim)
    heads = queries.shape[1]
    assert heads > 0 and heads % cache.heads == 0, f"{heads} heads of queries for {cache.heads} of the cache"


def _require_bounds(cache: KVCache):
    assert not isinstance(cache, KVCache8), "blocks are chosen by bounds, and a cache in 8 bits has none"


def _workspace(need: int, beside: Tensor) -> Optional[Tensor]:
    return beside.new_empty(nv.check(need), dtype=torch.uint8) if need else None


def attend(queries: Tensor, cache: Union[KVCache, KVCache8], table: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None,
           scale: Optional[float] = None, causal: bool = True, return_lse: bool = False, form: Optional[str] = None,
           accumulate: bool = False):
    """softmax(scale * queries keys^T) values over the `lengths` [sequences] tokens that the cache holds.  queries [rows, heads,
    dim], heads a multiple of the cache's; scale defaults to dim ** -0.5.  The rows of a sequence are its last tokens and see
    what stands before them and themselves, or with causal=False everything.  A row that sees nothing gives zeros.  With
    return_lse also the logarithms of the sums of exponentials [rows, heads], by which parts of an attention are joined.
    form: the library chooses one by the sizes, "many" where enough rows of a sequence share its pages (over 8 bits, of 32 heads on 8,
    more than about 12); "few" or "many" ask for it.  Of bfloat16 "many" rounds the weights to bfloat16 as well, which makes the
    result's error 1.2 times that of its own rounding; "few" holds 16 bits of them, and takes longer for many rows.
    accumulate, for a weighted KVCache8 and a table in which no page stands twice: the softmax weights that a token gets from all
    rows and the queries that share its head are added to its weight."""
    assert form is None or form in nv.ATTEND_FORMS, f"unknown form {form!r}: expected one of {sorted(nv.ATTEND_FORMS)}"
    tokens = _tokens(queries.shape[0], table, lengths, offsets)
    _check_queries(queries, cache)
    gpu = nv.require_one_gpu(queries, table, lengths, offsets)
    out = queries.new_empty(queries.shape)
    lse = queries.new_empty(queries.shape[:2], dtype=torch.float32) if return_lse else None
    q = _queries(queries, cache, scale, causal, out, lse, form)
    lib = nv.lib()
    if isinstance(cache, KVCache8):
        assert not accumulate or cache.weights is not None, "the cache keeps no weights: weighted=True"
        need = lib.vl_attend8_workspace_bytes(cache._ref, tokens, q, accumulate)
        ws = _workspace(need, queries)
        nv.check(lib.vl_attend8(cache._ref, tokens, q, accumulate, nv.ptr(ws), need, nv.stream_on(gpu, cache.gpu)))
        return (out, lse) if return_lse else out
    assert not accumulate, "a cache in 4 bits keeps no weights"
    need = lib.vl_attend_workspace_bytes(cache._ref, tokens, q)
    ws = _workspace(need, queries)
    nv.check(lib.vl_attend(cache._ref, tokens, q, nv.ptr(ws), need, nv.stream_on(gpu, cache.gpu)))
    return (out, lse) if return_lse else out


def select_blocks(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, count: int,
                  offsets: Optional[Tensor] = None) -> Tensor:
    """For every row and head of the cache `count` blocks of its sequence, ascending: the row's own and those with the highest
    bound on a score in them, of queries rounded to 8 bits and keys' bounds of 8 bits; MAXINT where there are no more.  [rows, cache.heads, count]"""
    _require_bounds(cache)
    assert count >= 1, f"count: {count}"
    tokens = _tokens(queries.shape[0], table, lengths, offsets)
    _check_queries(queries, cache)
    gpu = nv.require_one_gpu(queries, table, lengths, offsets)
    blocks = table.new_empty((queries.shape[0], cache.heads, count))
    q = _queries(queries, cache, None, True, None, None)
    lib = nv.lib()
    need = lib.vl_select_blocks_workspace_bytes(cache._ref, tokens, q, count)
    ws = _workspace(need, queries)
    nv.check(lib.vl_select_blocks(cache._ref, tokens, q, count, blocks.data_ptr(), nv.ptr(ws), need, nv.stream_on(gpu, cache.gpu)))
    return blocks


def attend_blocks(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, blocks: Tensor,
                  offsets: Optional[Tensor] = None, scale: Optional[float] = None, return_lse: bool = False):
    """attend over the tokens of blocks [rows, cache.heads, count] alone, up to the row's own place."""
    _require_bounds(cache)
    tokens = _tokens(queries.shape[0], table, lengths, offsets)
    _check_queries(queries, cache)
    assert blocks.dtype == torch.int32 and blocks.is_contiguous(), "blocks must be contiguous int32"
    assert blocks.dim() == 3 and blocks.shape[:2] == (queries.shape[0], cache.heads) and blocks.shape[2] > 0, \
        "blocks must be [rows, cache.heads, count]"
    gpu = nv.require_one_gpu(queries, table, lengths, blocks, offsets)
    count = blocks.shape[2]
    out = queries.new_empty(queries.shape)
    lse = queries.new_empty(queries.shape[:2], dtype=torch.float32) if return_lse else None
    q = _queries(queries, cache, scale, True, out, lse)
    lib = nv.lib()
    need = lib.vl_attend_blocks_workspace_bytes(cache._ref, tokens, q, count)
    ws = _workspace(need, queries)
    nv.check(lib.vl_attend_blocks(cache._ref, tokens, q, blocks.data_ptr(), count, nv.ptr(ws), need, nv.stream_on(gpu, cache.gpu)))
    return (out, lse) if return_lse else out


def attend_selected(queries: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, count: int,
                    offsets: Optional[Tensor] = None, scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """(attend_blocks(...), blocks) with the blocks of select_blocks (of the negated queries where scale is negative), in one call."""
    _require_bounds(cache)
    assert count >= 1, f"count: {count}"
    tokens = _tokens(queries.shape[0], table, lengths, offsets)
    _check_queries(queries, cache)
    gpu = nv.require_one_gpu(queries, table, lengths, offsets)
    blocks = table.new_empty((queries.shape[0], cache.heads, count))
    out = queries.new_empty(queries.shape)
    q = _queries(queries, cache, scale, True, out, None)
    lib = nv.lib()
    need = lib.vl_attend_selected_workspace_bytes(cache._ref, tokens, q, count)
    ws = _workspace(need, queries)
    nv.check(lib.vl_attend_selected(cache._ref, tokens, q, count, blocks.data_ptr(), nv.ptr(ws), need, nv.stream_on(gpu, cache.gpu)))
    return (out, blocks)
