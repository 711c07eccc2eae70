"""Workloads of the operators on a key/value cache held in 4 bits, as a program that answers with a language model calls them.

A case is a dict of plain values.  `op` says what one pass is:
  write   new keys and values of every sequence are quantised into the cache, then read back with the bounds of their blocks
  attend  softmax attention of new tokens over everything that the cache holds of their sequences
  sparse  for every new token and key/value head the `count` blocks with the best scores (from 8-bit bounds of each block's
          keys), and softmax attention over those alone

The cache holds pages of 64 tokens.  A group of 32 dimensions of one token is 32 codes of 4 bits (sign, two bits of exponent,
one of mantissa: 0 0.5 1 1.5 2 3 4 6) and a power of two, held as its exponent + 127.  Of every page and head it also holds, in
8 bits with one power of two, the largest and the smallest key in each dimension.
  keys          uint8 [pages, heads, 64, dim / 2]            two dimensions a byte, the even one in the low bits
  values        uint8 [pages, heads, 16, dim / 8, 4, 4]      token / 4, dim / 8, token % 4, four bytes of two dimensions
  key_scales, value_scales  uint8 [pages, heads, dim / 32, 64]
  bounds        int8 [pages, heads, 2, dim]                  largest, smallest
  bound_scales  int8 [pages, heads]                          exponent
A table [sequences, blocks] names the page of each block of 64 tokens of a sequence.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE = 64
EMPTY = 2147483647  # the empty id
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LEAST = -124        # the smallest exponent of a group's scale
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(op, **kw):
    """longest: tokens that the longest sequence has with the new ones; shortest: the same of the shortest (the others lie between);
    rows: new tokens a sequence (ragged: from that many down to one); empty: sequences without a token."""
    c = dict(op=op, dtype="bf16", batch=1, heads=8, group=4, dim=128, longest=1024, shortest=1024, rows=1, ragged=False, empty=0,
             count=0, causal=True)
    c.update(kw)
    return c


def listed():
    return [
        # one step of a batch of answers: a token each, launches and host work
        dict(_case("write", batch=64, longest=8_192, shortest=500), name="write-64x1"),
        # a few prompts of odd lengths that go on in the middle of a block, float32 rows of 96
        dict(_case("write", dtype="f32", batch=5, heads=3, group=5, dim=96, longest=1_701, shortest=303, rows=1_333, ragged=True),
             name="write-odd"),
        # a long prompt read in at once
        dict(_case("write", longest=32_768, shortest=32_768, rows=32_768), name="write-32768"),
        # one answer at a time on a short context: latency
        dict(_case("attend", longest=1_000, shortest=1_000), name="attend-1"),
        # a batch of answers of all lengths, one not begun yet; half precision, 7 query heads a key head, rows of 64
        dict(_case("attend", dtype="f16", batch=37, heads=2, group=7, dim=64, longest=4_099, shortest=1, empty=1),
             name="attend-37-odd"),
        # a batch of answers on ordinary contexts
        dict(_case("attend", batch=64, longest=8_192, shortest=4_096), name="attend-64"),
        # a few answers on very long contexts: what the memory gives
        dict(_case("attend", batch=4, longest=131_072, shortest=131_072), name="attend-4-long"),
        # five proposed tokens each, checked at once, in float32 with rows of 256
        dict(_case("attend", dtype="f32", batch=3, heads=4, group=2, dim=256, longest=2_050, shortest=777, rows=5),
             name="attend-3x5"),
        # a piece of a long prompt against what was read before: matrix products
        dict(_case("attend", longest=16_384, shortest=16_384, rows=2_048), name="attend-2048"),
        # one answer on a very long context, 32 blocks of it
        dict(_case("sparse", longest=131_072, shortest=131_072, count=32), name="sparse-1"),
        # a batch of answers on long contexts of all lengths
        dict(_case("sparse", batch=32, longest=32_768, shortest=9_999, count=32), name="sparse-32"),
        # pieces of prompts: every token with a choice of its own, half precision, rows of 96
        dict(_case("sparse", dtype="f16", batch=3, heads=4, group=6, dim=96, longest=9_001, shortest=2_500, rows=600, ragged=True,
                   count=16), name="sparse-600"),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "attend", "sparse"))
    (heads, group, dim) = (rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16)), rng.choice((32, 64, 96, 128, 128, 192, 256)))
    dtype = rng.choices(("bf16", "f16", "f32"), (3, 1, 1))[0]
    values = heads * dim  # a token's
    if op == "write":
        batch = _spread(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _spread(rng, 2, max(3, 24_000_000 // (values * batch)))
        longest = rows + rng.choice((0, 1, rng.randint(0, 2_000)))
        return _case(op, dtype=dtype, batch=batch, heads=heads, group=group, dim=dim, rows=rows, ragged=rows > 1,
                     longest=longest, shortest=max(rows, longest // 2))
    if op == "sparse":
        rows = 1 if rng.random() < 0.6 else _spread(rng, 2, 512)
        batch = _spread(rng, 1, 32 if rows == 1 else 3)
        count = rng.choice((4, 8, 16, 17, 32))
        rows = min(rows, max(1, (1 << 29) // (values * batch * count * PAGE)))
        longest = max(rows, min((1 << 30) // (batch * values), _spread(rng, 200, 131_072)))
        return _case(op, dtype=dtype, batch=batch, heads=heads, group=group, dim=dim, rows=rows, ragged=rows > 1,
                     longest=longest, shortest=max(rows, int(longest * rng.random())), count=count)
    kind = rng.choices(("one", "few", "many"), (3, 1, 2))[0]
    if kind == "many":
        batch = _spread(rng, 1, 4)
        room = 2_048 * 15_360 * 32 * 128 // (batch * group * values)  # rows times tokens
        rows = _spread(rng, 64, min(2_048, math.isqrt(room)))
        longest = max(rows, min(room // rows, _spread(rng, rows, 16_384)))
    else:
        rows = 1 if kind == "one" else rng.randint(2, 9)
        batch = _spread(rng, 1, 64)
        longest = max(rows, min(131_072, 4 * 131_072 * 1_024 // (batch * values), _spread(rng, 100, 131_072)))
    return _case(op, dtype=dtype, batch=batch, heads=heads, group=group, dim=dim, rows=rows, ragged=rows > 1, longest=longest,
                 shortest=max(rows, int(longest * rng.random())), empty=int(rows == 1 and batch > 2 and rng.random() < 0.3),
                 causal=rng.random() < 0.8)


def _even(first, last, n):
    """n whole numbers from first to last in even steps."""
    return [first + (last - first) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(tokens of each sequence, the new ones among them)"""
    n = case["batch"] - case["empty"]
    lengths = [0] * case["empty"] + _even(case["longest"], case["shortest"], n)
    return lengths, _even(case["rows"], 1 if case["ragged"] else case["rows"], case["batch"])


def _exponent(x):
    """floor(log2 x), for x = 0 far below any that counts."""
    return torch.where(x > 0, torch.frexp(x).exponent - 1, -1000)


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """(codes uint8 [..., dim], scales uint8 [..., dim / 32]) of x [..., dim] in 32 bits: every group's scale is the power of two that
    brings its largest magnitude into [4, 8); codes are the nearest ones, of two as near the even one, 6 where it is passed."""
    g = x.unflatten(-1, (-1, 32))
    e = (_exponent(g.abs().amax(-1)) - 2).clamp(min=LEAST)
    a = (g * _power(-e)[..., None]).abs()
    a = torch.where(a < 2.0, torch.round(a * 2) * 0.5, torch.where(a < 4.0, torch.round(a), torch.round(a * 0.5) * 2)).clamp(max=6.0)
    code = torch.where(a < 2.0, a * 2, torch.where(a < 4.0, a + 2, a * 0.5 + 4)).to(torch.uint8)
    code = code | ((g < 0).to(torch.uint8) << 3)
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _bytes(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values_of(packed, scales):
    """The values in 32 bits: packed [..., dim / 2], scales [..., dim / 32]"""
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).to(torch.int32)
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=packed.device)
    return (grid[code].unflatten(-1, (-1, 32)) * _power(scales.to(torch.int32) - 127)[..., None]).flatten(-2)


def _keys(cache, *at):
    """Keys of the blocks that the index names, [..., 64, dim]"""
    return _values_of(cache["keys"][at], cache["key_scales"][at].transpose(-1, -2))


def _values(cache, *at):
    v = cache["values"][at].transpose(-3, -2).flatten(-2)  # [..., 16, 4, dim / 8, 4] -> dim / 2
    return _values_of(v.flatten(-3, -2), cache["value_scales"][at].transpose(-1, -2))


def _bounds_of(keys, seen):
    """(bounds int8 [..., 2, dim], exponent int8 [...]) of the keys [..., 64, dim] of a block, where `seen` [..., 64] says which count."""
    hi = keys.masked_fill(~seen[..., None], -math.inf).amax(-2)
    lo = keys.masked_fill(~seen[..., None], math.inf).amin(-2)
    (hi, lo) = (torch.where(hi < lo, 0.0, hi), torch.where(hi < lo, 0.0, lo))
    e = (_exponent(torch.maximum(hi.abs(), lo.abs()).amax(-1)) - 6).clamp(min=-126)
    s = _power(-e)[..., None]
    return torch.stack((torch.ceil(hi * s), torch.floor(lo * s)), -2).to(torch.int8), e.to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    (batch, heads, group, dim) = (case["batch"], case["heads"], case["group"], case["dim"])
    (lengths, new) = _lengths(case)
    turn = torch.randperm(batch, generator=gen, device=DEV).tolist()
    (lengths, new) = ([lengths[i] for i in turn], [new[i] for i in turn])
    blocks = max(1, -(-case["longest"] // PAGE))
    pages = batch * blocks + 3
    length = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    names = torch.randperm(pages, generator=gen, device=DEV)[:batch * blocks].view(batch, blocks)
    seen = (length[:, None] - PAGE * torch.arange(blocks, device=DEV)).clamp(0, PAGE)
    table = torch.where(seen > 0, names, EMPTY).to(torch.int32)
    held = torch.zeros(pages, dtype=torch.int64, device=DEV)
    held[names] = seen
    # keys of a page have a subject in common, and some dimensions are larger than others everywhere
    wide = torch.exp(0.5 * torch.randn((heads, 1, dim), generator=gen, device=DEV))
    subject = torch.randn((pages, heads, 1, dim), generator=gen, device=DEV)
    x = torch.randn((pages, heads, PAGE, dim), generator=gen, device=DEV).add_(subject).mul_(wide)
    (code, scale) = _quantised(x)
    keys = _bytes(code)
    key_scales = scale.transpose(-1, -2).contiguous()
    cache = dict(keys=keys, key_scales=key_scales)
    (cache["bounds"], cache["bound_scales"]) = _bounds_of(_values_of(keys, scale), torch.arange(PAGE, device=DEV) < held[:, None, None])
    (code, scale) = _quantised(x.normal_(generator=gen))
    cache["values"] = _bytes(code).view(pages, heads, 16, 4, dim // 8, 4).transpose(-3, -2).contiguous()
    cache["value_scales"] = scale.transpose(-1, -2).contiguous()
    # what the layer's one projection gives: queries, keys and values of a token side by side
    rows = sum(new)
    heads_q = heads * group
    mixed = torch.randn((rows, heads_q + 2 * heads, dim), generator=gen, device=DEV)
    about = subject[torch.randint(0, pages, (rows,), generator=gen, device=DEV), :, 0]  # what the token asks about
    mixed[:, :heads_q] += 0.7 * about.repeat_interleave(group, dim=1)
    mixed[:, heads_q:heads_q + heads] *= wide[:, 0]
    mixed = mixed.to(TYPES[case["dtype"]])
    offsets = torch.tensor([sum(new[:i]) for i in range(batch + 1)], dtype=torch.int32, device=DEV)
    state = dict(case=case, tensors=cache, table=table, lengths=length, queries=mixed[:, :heads_q],
                 new_keys=mixed[:, heads_q:heads_q + heads], new_values=mixed[:, heads_q + heads:],
                 offsets=None if case["rows"] == 1 else offsets)
    if case["op"] == "write":
        # the table of the blocks that are written into: their bounds change
        starts = length - torch.tensor(new, dtype=torch.int32, device=DEV)
        widest = max((n - 1) // PAGE - (n - m) // PAGE + 1 for n, m in zip(lengths, new))
        block = starts[:, None] // PAGE + torch.arange(widest, device=DEV)
        inside = block * PAGE < length[:, None]
        touched = torch.where(inside, table.gather(1, block.clamp(max=blocks - 1).long()), EMPTY)
        state.update(starts=starts, touched=touched.to(torch.int32))
    if own:  # the handle over the same tensors
        sys.path.insert(0, os.path.join(os.getcwd(), "vectorlink-gpu_amd"))
        from vectorlink_gpu.attention import KVCache

        state["cache"] = KVCache(**cache)
    return state


def _rows(state):
    """(sequence, place among its new tokens) of every row"""
    rows = state["queries"].size(0)
    at = torch.arange(rows, device=DEV)
    if state["offsets"] is None:
        return at, torch.zeros_like(at)
    b = torch.searchsorted(state["offsets"], at, right=True) - 1
    return b, at - state["offsets"][b]


def _positions(state):
    """The place of every row's token in its sequence"""
    (b, t) = _rows(state)
    new = 1 if state["offsets"] is None else (state["offsets"][1:] - state["offsets"][:-1])[b]
    return state["lengths"][b] - new + t


def _softmax(scores, mask, values):
    """Rows of the mask that hold nothing give zeros."""
    scores = torch.where(mask, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(total > 0, total, 1.0)


def _padded(state, x):
    """x [rows, heads, group, n] as [sequences, heads, tokens * group, n], and the way back"""
    (b, t) = _rows(state)
    case = state["case"]
    out = torch.zeros((case["batch"], case["rows"], *x.shape[1:]), dtype=x.dtype, device=DEV)
    out[b, t] = x
    return out.transpose(1, 2).flatten(2, 3), lambda y: y.unflatten(2, (case["rows"], -1)).transpose(1, 2)[b, t]


def _grouped(state):
    return state["queries"].float().unflatten(1, (state["case"]["heads"], -1))


def _plain_attend(state):
    (case, cache) = (state["case"], state["tensors"])
    at = state["table"].long().clamp(max=cache["keys"].size(0) - 1)
    k = _keys(cache, at).transpose(1, 2).flatten(2, 3)      # [sequences, heads, tokens, dim]
    v = _values(cache, at).transpose(1, 2).flatten(2, 3)
    (q, back) = _padded(state, _grouped(state))
    last = state["lengths"].long()[:, None].expand(-1, case["rows"]) - 1
    if case["causal"] and state["offsets"] is not None:
        new = state["offsets"][1:] - state["offsets"][:-1]
        last = last - new[:, None] + 1 + torch.arange(case["rows"], device=DEV)
    last = last.repeat_interleave(case["group"], dim=1)
    mask = torch.arange(k.size(2), device=DEV) <= last[:, None, :, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) * (case["dim"] ** -0.5)
    return back(_softmax(scores, mask, v)).flatten(1, 2).to(state["queries"].dtype)


def _plain_select(state):
    """Scores are whole numbers times a power of two, so they are the same in any order of the sums.  A token's own block is
    always among the chosen ones."""
    (case, cache) = (state["case"], state["tensors"])
    q = _grouped(state)
    e = _exponent(q.abs().amax((-1, -2))) - 6
    q = torch.round(q * _power(-e.clamp(min=-100))[..., None, None]).clamp(-127, 127)
    (q, back) = _padded(state, torch.cat((q.clamp(min=0), q.clamp(max=0)), -1))
    at = state["table"].long().clamp(max=cache["keys"].size(0) - 1)
    bounds = cache["bounds"][at].float().flatten(-2).transpose(1, 2)     # [sequences, heads, blocks, 2 dim]
    power = _power(cache["bound_scales"][at]).transpose(1, 2)
    scores = back(torch.matmul(q, bounds.transpose(-1, -2))).amax(-2)     # [rows, heads, blocks]
    (b, _) = _rows(state)
    scores = scores * power[b]
    block = torch.arange(at.size(1), device=DEV)
    mine = (_positions(state) // PAGE)[:, None, None]
    scores = torch.where(block == mine, math.inf, torch.where(block < mine, scores, -math.inf))
    (best, ids) = torch.sort(scores, dim=-1, descending=True, stable=True)
    ids = torch.where(best > -math.inf, ids, EMPTY)[..., :case["count"]]
    ids = torch.nn.functional.pad(ids, (0, case["count"] - ids.size(-1)), value=EMPTY)
    return torch.sort(ids, dim=-1).values.to(torch.int32)


def _plain_sparse(state):
    (case, cache) = (state["case"], state["tensors"])
    ids = _plain_select(state)
    (b, _) = _rows(state)
    real = ids != EMPTY
    block = torch.where(real, ids, 0).long()
    at = state["table"][b[:, None, None], block].long().clamp(max=cache["keys"].size(0) - 1)
    head = torch.arange(case["heads"], device=DEV)[None, :, None]
    k = _keys(cache, at, head).flatten(2, 3)        # [rows, heads, count * 64, dim]
    v = _values(cache, at, head).flatten(2, 3)
    token = block[..., None] * PAGE + torch.arange(PAGE, device=DEV)
    mask = ((token <= _positions(state)[:, None, None, None]) & real[..., None]).flatten(2)[:, :, None]
    scores = torch.matmul(_grouped(state), k.transpose(-1, -2)) * (case["dim"] ** -0.5)
    return dict(blocks=ids, out=_softmax(scores, mask, v).flatten(1, 2).to(state["queries"].dtype))


def _plain_write(state):
    (case, cache) = (state["case"], state["tensors"])
    (b, _) = _rows(state)
    place = _positions(state).long()
    page = state["table"][b, place // PAGE].long()[:, None]
    token = (place % PAGE)[:, None]
    head = torch.arange(case["heads"], device=DEV)
    (code, scale) = _quantised(state["new_keys"].float())
    cache["keys"][page, head, token] = _bytes(code)
    cache["key_scales"][page, head, :, token] = scale
    (code, scale) = _quantised(state["new_values"].float())
    cache["values"][page, head, token // 4, :, token % 4] = _bytes(code).unflatten(-1, (-1, 4))
    cache["value_scales"][page, head, :, token] = scale
    # the bounds of all blocks that the new tokens lie in
    real = state["touched"] != EMPTY
    touched = state["touched"].long().clamp(max=cache["keys"].size(0) - 1)
    first = state["starts"][:, None] // PAGE + torch.arange(touched.size(1), device=DEV)
    held = state["lengths"][:, None] - PAGE * first
    (bounds, power) = _bounds_of(_keys(cache, touched), torch.arange(PAGE, device=DEV) < held[..., None, None])
    cache["bounds"][touched[real]] = bounds[real]
    cache["bound_scales"][touched[real]] = power[real]
    # and all of it as the values it stands for
    dtype = state["new_keys"].dtype
    k = _values_of(cache["keys"][page, head, token], cache["key_scales"][page, head, :, token])
    v = _values_of(cache["values"][page, head, token // 4, :, token % 4].flatten(-2), cache["value_scales"][page, head, :, token])
    bounds = cache["bounds"][touched].float() * _power(cache["bound_scales"][touched])[..., None, None]
    return dict(keys=k.to(dtype), values=v.to(dtype), bounds=torch.where(real[..., None, None, None], bounds, 0.0))


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"write": _plain_write, "attend": _plain_attend, "sparse": _plain_sparse}[op](state)
    from vectorlink_gpu.attention import attend, attend_selected

    (cache, table, offsets) = (state["cache"], state["table"], state["offsets"])
    if op == "attend":
        return attend(state["queries"], cache, table, state["lengths"], offsets=offsets, causal=case["causal"])
    if op == "sparse":
        (out, blocks) = attend_selected(state["queries"], cache, table, state["lengths"], case["count"], offsets=offsets)
        return dict(blocks=blocks, out=out)
    cache.write(state["new_keys"], state["new_values"], table, state["starts"], offsets=offsets)
    (k, v) = cache.read(table, state["starts"], state["new_keys"].size(0), offsets=offsets, dtype=state["new_keys"].dtype)
    return dict(keys=k, values=v, bounds=cache.read_bounds(state["touched"]))


def work(case):
    """Inputs read once, outputs written once; of a cache what the path has to look at: all that attention sees, or the bounds of
    all blocks and the chosen blocks (each once, however many tokens choose it)."""
    (lengths, new) = _lengths(case)
    (heads, group, dim) = (case["heads"], case["group"], case["dim"])
    rows = sum(new)
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    token = heads * (dim + dim // 16)  # bytes of a token in the cache: codes and scales of key and value
    ends = 2.0 * size * rows * heads * group * dim
    if case["op"] == "write":
        blocks = sum(-(-n // PAGE) - (n - m) // PAGE for n, m in zip(lengths, new))
        before = sum((n - m) % PAGE for n, m in zip(lengths, new))  # keys that the first block holds already
        return dict(bytes=4.0 * size * rows * heads * dim + 2.0 * rows * token + 0.5 * before * token
                    + blocks * heads * (2 * dim * 5 + 1), flops=8.0 * rows * heads * dim)
    if case["op"] == "attend":
        # of a sequence's new tokens, each sees what stands before it and itself
        pairs = sum(m * n - (m * (m - 1) / 2 if case["causal"] else 0) for n, m in zip(lengths, new) if n)
        return dict(bytes=ends + sum(lengths) * token, flops=4.0 * pairs * heads * group * dim)
    count = case["count"]
    some = sum(min(n, m * count * PAGE) for n, m in zip(lengths, new))
    pairs = sum(m * min(n, count * PAGE) for n, m in zip(lengths, new))
    blocks = sum(-(-n // PAGE) for n in lengths)
    scored = sum(m * -(-n // PAGE) for n, m in zip(lengths, new))
    return dict(bytes=ends + some * token + blocks * heads * (2 * dim + 1) + 4.0 * rows * heads * count,
                flops=4.0 * pairs * heads * group * dim + 2.0 * scored * heads * group * dim)


def _stands_for(byte, scale):
    """Values of codes in 64 bits from the bits' meaning: byte [n, dim / 2], scale [n, dim / 32]"""
    code = torch.zeros((byte.size(0), byte.size(1) * 2), dtype=torch.float64, device=byte.device)
    for half in (0, 1):
        c = (byte >> (4 * half)) & 15
        (up, odd) = ((c >> 1) & 3, c & 1)
        mag = torch.where(up == 0, odd * 0.5, (1 + 0.5 * odd.double()) * torch.exp2(up.double() - 1))
        code[:, half::2] = torch.where(c >= 8, -mag, mag)
    return code * torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)


def _binade(top, below, least):
    """2^(floor(log2 top) + below) in 64 bits, at least 2^least"""
    return torch.exp2((torch.frexp(top).exponent - 1 + below).masked_fill(top == 0, least).clamp(min=least).double())


def _rounded(x):
    """x [n, dim] in 64 bits as the cache holds it: nearest point of the grid of its group."""
    out = torch.zeros_like(x)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    for g in range(0, x.size(1), 32):
        part = x[:, g:g + 32]
        power = _binade(part.abs().amax(1), -2, LEAST)
        a = part.abs() / power[:, None]
        at = torch.searchsorted((grid[1:] + grid[:-1]) / 2, a.contiguous())            # a tie stays below
        tie = (at < 7) & (a == ((grid[1:] + grid[:-1]) / 2)[at.clamp(max=6)])
        at = torch.where(tie & (at % 2 == 1), at + 1, at)                              # and goes to the even code
        out[:, g:g + 32] = torch.sign(part) * grid[at] * power[:, None]
    return out


def _held(state, b, head, blocks):
    """(keys, values) of these blocks of a sequence, [blocks * 64, dim] in 64 bits"""
    t = state["tensors"]
    page = state["table"][b, blocks].long()
    k = t["keys"][page, head].flatten(0, 1)
    v = t["values"][page, head].permute(0, 1, 3, 2, 4).flatten(3).flatten(0, 2)
    return (_stands_for(k, t["key_scales"][page, head].permute(0, 2, 1).flatten(0, 1)),
            _stands_for(v, t["value_scales"][page, head].permute(0, 2, 1).flatten(0, 1)))


def exact(case, seed):
    """The definitions in 64 bits, a sequence and a head at a time."""
    state = prepare(case, seed)
    rows = state["queries"].size(0)
    offsets = list(range(rows + 1)) if state["offsets"] is None else state["offsets"].tolist()
    lengths = state["lengths"].tolist()
    (heads, group, dim, count) = (case["heads"], case["group"], case["dim"], case["count"])
    if case["op"] == "write":
        new = [_rounded(state[x].double().flatten(0, 1)).view(rows, heads, dim) for x in ("new_keys", "new_values")]
        bounds = torch.zeros((*state["touched"].shape, heads, 2, dim), dtype=torch.float64, device=DEV)
        starts = state["starts"].tolist()
        for b in range(case["batch"]):
            k = new[0][offsets[b]:offsets[b + 1]].transpose(0, 1)
            if starts[b] % PAGE:  # what the first block holds already
                block = torch.tensor([starts[b] // PAGE], device=DEV)
                before = torch.stack([_held(state, b, h, block)[0] for h in range(heads)])
                k = torch.cat((before[:, :starts[b] % PAGE], k), dim=1)
            for i, part in enumerate(k.split(PAGE, dim=1)):
                power = _binade(part.abs().amax((1, 2)), -6, -126)[:, None]
                bounds[b, i, :, 0] = torch.ceil(part.amax(1) / power) * power
                bounds[b, i, :, 1] = torch.floor(part.amin(1) / power) * power
        return dict(keys=new[0], values=new[1], bounds=bounds)
    out = torch.zeros((rows, heads * group, dim), dtype=torch.float64, device=DEV)
    chosen = torch.full((rows, heads, count), EMPTY, dtype=torch.int64, device=DEV) if count else None
    for b in range(case["batch"]):
        (first, end, n) = (offsets[b], offsets[b + 1], lengths[b])
        if n == 0:
            continue
        last = torch.full((end - first,), n - 1, device=DEV)
        if case["causal"]:
            last = n - (end - first) + torch.arange(end - first, device=DEV)
        blocks = torch.arange(-(-n // PAGE), device=DEV)
        token = torch.arange(blocks.numel() * PAGE, device=DEV)
        for h in range(heads):
            (k, v) = _held(state, b, h, blocks)
            seen = token[None] <= last[:, None]
            q = state["queries"][first:end, h * group:(h + 1) * group].double()
            if count:
                page = state["table"][b, blocks].long()
                edge = state["tensors"]["bounds"][page, h].double() * torch.exp2(state["tensors"]["bound_scales"][page, h].double())[:, None, None]
                unit = _binade(q.abs().amax((1, 2)), -6, -100)[:, None, None]
                w = torch.clamp(torch.round(q / unit), -127, 127)
                score = torch.matmul(w.clamp(min=0), edge[:, 0].T.contiguous()) + torch.matmul(w.clamp(max=0), edge[:, 1].T.contiguous())
                score = score.amax(1)
                score = torch.where(blocks == (last // PAGE)[:, None], math.inf, torch.where(blocks < (last // PAGE)[:, None], score, -math.inf))
                best = torch.sort(score, dim=1, descending=True, stable=True)
                ids = torch.where(best.values[:, :count] > -math.inf, best.indices[:, :count], EMPTY)
                chosen[first:end, h, :ids.size(1)] = torch.sort(ids, dim=1).values
                takes = torch.zeros((end - first, blocks.numel() + 1), dtype=torch.bool, device=DEV)
                takes.scatter_(1, ids.clamp(max=blocks.numel()), True)
                seen &= takes[:, :-1].repeat_interleave(PAGE, dim=1)
            for g in range(group):
                s = torch.matmul(q[:, g], k.T.contiguous()) / math.sqrt(dim)
                s = torch.softmax(s.masked_fill_(~seen, -math.inf), dim=1)
                out[first:end, h * group + g] = torch.matmul(s, v)
    return dict(blocks=chosen.to(torch.int32), out=out) if count else out
