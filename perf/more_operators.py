"""Workloads of the operators on a key/value cache held in 8 bits and cut down by what its tokens were looked at, as a program
that answers with a language model calls them.

A case is a dict of plain values.  `op` says what one pass is:
  write   new keys and values of every sequence are rounded into the cache, then read back
  attend  softmax attention of new tokens over everything that the cache holds of their sequences
  weigh   the same, and every token of the cache is added the weights that it got from all of the pass's rows and queries
  evict   of every sequence and head the `keep` tokens that count most stay: the `recent` latest, then those of the largest
          accumulated weight

The cache holds pages of 64 tokens.  A key or value is dim codes of 8 bits (e4m3: sign, four bits of exponent, three of
mantissa, largest 448, no infinity) times a power of two that all 64 tokens of a page and head share, one for keys and one for
values, held as its exponent + 127.
  keys       uint8 [pages, heads, 64, dim]
  values     uint8 [pages, heads, 16, dim, 4]    token / 4, dim, token % 4
  scales     uint8 [pages, heads, 4]             of keys, of values; whether a token is not finite; 0
  weights    float32 [pages, heads, 64]          accumulated weight of each token
  positions  int32 [pages, heads, 64]            where each token stood in its text
A table [sequences, blocks] names the page of each block of 64 tokens of a sequence.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE = 64
EMPTY = 2147483647  # a block without a page
LEAST = -117        # the smallest exponent of a page's scale
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = torch.float8_e4m3fn


def _case(op, **kw):
    """longest: tokens that the longest sequence has with the new ones; shortest: the same of the shortest (the others lie between);
    rows: new tokens a sequence (ragged: from that many down to one); empty: sequences without a token."""
    c = dict(op=op, dtype="bf16", batch=1, heads=8, group=4, dim=128, longest=1024, shortest=1024, rows=1, ragged=False, empty=0,
             causal=True, keep=0, recent=0)
    c.update(kw)
    return c


def listed():
    return [
        # one step of a batch of answers: a token each, launches and host work
        dict(_case("write", batch=64, longest=8_192, shortest=500), name="write-64x1"),
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
        # a piece of a long prompt against what was read before: matrix products
        dict(_case("attend", longest=16_384, shortest=16_384, rows=2_048), name="attend-2048"),
        # a batch of answers whose weights are kept, for the next eviction
        dict(_case("weigh", batch=32, longest=16_384, shortest=8_192), name="weigh-32"),
        # the last pieces of prompts, which say what of the prompts will be asked for: half precision, rows of 96
        dict(_case("weigh", dtype="f16", batch=3, heads=4, group=6, dim=96, longest=9_001, shortest=2_500, rows=600, ragged=True),
             name="weigh-600-odd"),
        # a batch of answers is a page over its budget: each head gives 64 tokens up
        dict(_case("evict", batch=64, longest=4_160, shortest=4_160, keep=4_096, recent=256), name="evict-64"),
        # a long prompt is cut down to an eighth
        dict(_case("evict", longest=131_072, shortest=131_072, keep=16_384, recent=512), name="evict-prompt"),
        # some sequences over an odd budget and some under it, rows of 96
        dict(_case("evict", batch=5, heads=3, dim=96, longest=3_001, shortest=700, keep=1_111, recent=33), name="evict-odd"),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "attend", "attend", "weigh", "weigh", "evict", "evict"))
    (heads, group, dim) = (rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16)), rng.choice((32, 64, 96, 128, 128, 192, 256)))
    dtype = rng.choices(("bf16", "f16", "f32"), (3, 1, 1))[0]
    values = heads * dim  # a token's
    if op == "write":
        batch = _spread(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _spread(rng, 2, max(3, 24_000_000 // (values * batch)))
        longest = rows + rng.choice((0, 1, rng.randint(0, 2_000)))
        return _case(op, dtype=dtype, batch=batch, heads=heads, group=group, dim=dim, rows=rows, ragged=rows > 1,
                     longest=longest, shortest=max(rows, longest // 2))
    if op == "evict":
        batch = _spread(rng, 1, 64)
        longest = _spread(rng, 70, min(131_072, 131_072 * 1_024 // (batch * values)))
        keep = _spread(rng, 1, longest)
        return _case(op, batch=batch, heads=heads, group=group, dim=dim, longest=longest, shortest=int(longest * rng.random()),
                     keep=keep, recent=int(keep * rng.choice((0.0, 0.05, 0.3, 1.0))))
    kind = rng.choices(("one", "few", "many"), (3, 1, 2))[0]
    if kind == "many":
        batch = _spread(rng, 1, 4)
        room = 2_048 * 15_360 * 32 * 128 // (batch * group * values) // (4 if op == "weigh" else 1)  # rows times tokens
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


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _least_exponent(top):
    """The smallest e, LEAST at least, with top <= 448 * 2^e"""
    (part, e) = torch.frexp(top)  # part in [0.5, 1)
    return torch.where(top > 0, e - 9 + (part > 0.875).to(e.dtype), LEAST).clamp(min=LEAST)


def _coded(x, e):
    """Codes of x in 32 bits over 2^e: the nearest ones, of two as near the even one."""
    return (x * _power(-e)).to(CODES).view(torch.uint8)


def _decoded(code, byte):
    """Values in 32 bits: code [..., n], byte [...] the exponent + 127"""
    return code.view(CODES).float() * _power(byte.to(torch.int32) - 127)[..., None]


def _by_token(values):
    """[..., 16, dim, 4] -> [..., 64, dim]"""
    return values.transpose(-1, -2).flatten(-3, -2)


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
    # keys of a page have a subject in common, and some dimensions are larger than others everywhere
    wide = torch.exp(0.5 * torch.randn((heads, 1, dim), generator=gen, device=DEV))
    subject = torch.randn((pages, heads, 1, dim), generator=gen, device=DEV)
    scales = torch.zeros((pages, heads, 4), dtype=torch.uint8, device=DEV)
    x = torch.randn((pages, heads, PAGE, dim), generator=gen, device=DEV).add_(subject).mul_(wide)
    e = _least_exponent(x.abs().amax((-1, -2)))
    keys = _coded(x, e[..., None, None])
    scales[..., 0] = (e + 127).to(torch.uint8)
    x.normal_(generator=gen)
    e = _least_exponent(x.abs().amax((-1, -2)))
    values = _coded(x, e[..., None, None]).unflatten(2, (16, 4)).transpose(-1, -2).contiguous()
    scales[..., 1] = (e + 127).to(torch.uint8)
    del x
    cache = dict(keys=keys, values=values, scales=scales)
    if case["op"] != "attend":
        # most tokens are hardly looked at, a tenth not once
        w = torch.exp(2 * torch.randn((pages, heads, PAGE), generator=gen, device=DEV))
        cache["weights"] = torch.where(torch.rand(w.shape, generator=gen, device=DEV) < 0.1, 0.0, w)
        cache["positions"] = torch.zeros((pages, heads, PAGE), dtype=torch.int32, device=DEV)
        place = (PAGE * torch.arange(blocks, device=DEV)[:, None] + torch.arange(PAGE, device=DEV)).expand(batch, heads, blocks, PAGE)
        if case["op"] == "evict" and case["longest"] - case["keep"] <= PAGE:
            # earlier evictions have left what stayed in another order; what came since stands behind it
            old = torch.rand((batch, heads, case["keep"]), generator=gen, device=DEV).argsort(-1)
            place = place.flatten(2).clone()
            place[..., :case["keep"]] = old
            place = place.unflatten(2, (blocks, PAGE))
        cache["positions"][names] = place.transpose(1, 2).to(torch.int32)
    state = dict(case=case, tensors=cache, table=table, lengths=length)
    if case["op"] == "evict":
        state.update(weights=cache["weights"].clone(), positions=cache["positions"].clone())
    else:
        # what the layer's one projection gives: queries, keys and values of a token side by side
        rows = sum(new)
        heads_q = heads * group
        mixed = torch.randn((rows, heads_q + 2 * heads, dim), generator=gen, device=DEV)
        about = subject[torch.randint(0, pages, (rows,), generator=gen, device=DEV), :, 0]  # what the token asks about
        mixed[:, :heads_q] += 0.7 * about.repeat_interleave(group, dim=1)
        mixed[:, heads_q:heads_q + heads] *= wide[:, 0]
        mixed = mixed.to(TYPES[case["dtype"]])
        offsets = torch.tensor([sum(new[:i]) for i in range(batch + 1)], dtype=torch.int32, device=DEV)
        state.update(queries=mixed[:, :heads_q], new_keys=mixed[:, heads_q:heads_q + heads], new_values=mixed[:, heads_q + heads:],
                     offsets=None if case["rows"] == 1 else offsets)
        if case["op"] == "write":
            starts = length - torch.tensor(new, dtype=torch.int32, device=DEV)
            widest = max((n - 1) // PAGE - (n - m) // PAGE + 1 for n, m in zip(lengths, new))
            state.update(starts=starts, widest=widest)
    if own:  # the handle over the same tensors
        sys.path.insert(0, os.path.join(os.getcwd(), "vectorlink-gpu_amd"))
        from vectorlink_gpu.attention import KVCache8

        state["cache"] = KVCache8(**cache)
    return state


def _rows(state):
    """(sequence, place among its new tokens) of every row"""
    rows = state["queries"].size(0)
    at = torch.arange(rows, device=DEV)
    if state["offsets"] is None:
        return at, torch.zeros_like(at)
    b = torch.searchsorted(state["offsets"], at, right=True) - 1
    return b, at - state["offsets"][b]


def _padded(state, x):
    """x [rows, heads, group, n] as [sequences, heads, tokens * group, n], and the way back"""
    (b, t) = _rows(state)
    case = state["case"]
    out = torch.zeros((case["batch"], case["rows"], *x.shape[1:]), dtype=x.dtype, device=DEV)
    out[b, t] = x
    return out.transpose(1, 2).flatten(2, 3), lambda y: y.unflatten(2, (case["rows"], -1)).transpose(1, 2)[b, t]


def _plain_attend(state):
    """softmax(q k^T / sqrt(dim)) v; rows that see nothing give zeros.  Of `weigh` every token's weight grows by the sum of its
    column of the softmax, over the rows and the queries that share its head."""
    (case, cache) = (state["case"], state["tensors"])
    at = state["table"].long().clamp(max=cache["keys"].size(0) - 1)
    k = _decoded(cache["keys"][at], cache["scales"][at][..., :1]).transpose(1, 2).flatten(2, 3)  # [sequences, heads, tokens, dim]
    (q, back) = _padded(state, state["queries"].float().unflatten(1, (case["heads"], -1)))
    last = state["lengths"].long()[:, None].expand(-1, case["rows"]) - 1
    new = 1 if state["offsets"] is None else (state["offsets"][1:] - state["offsets"][:-1])[:, None]
    if case["causal"]:
        last = last - new + 1 + torch.arange(case["rows"], device=DEV)
    last = torch.where(torch.arange(case["rows"], device=DEV) < new, last, -1)  # rows that are there for the padding
    last = last.repeat_interleave(case["group"], dim=1)
    mask = torch.arange(k.size(2), device=DEV) <= last[:, None, :, None]
    scores = torch.where(mask, torch.matmul(q, k.transpose(-1, -2)) * (case["dim"] ** -0.5), -math.inf)
    del k
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    del scores
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    v = _decoded(_by_token(cache["values"][at]), cache["scales"][at][..., 1:2]).transpose(1, 2).flatten(2, 3)
    out = back(torch.matmul(p, v)).flatten(1, 2).to(state["queries"].dtype)
    if case["op"] == "attend":
        return out
    added = p.sum(2).unflatten(2, (-1, PAGE)).transpose(1, 2)  # [sequences, blocks, heads, 64]
    real = state["table"] != EMPTY
    cache["weights"][at[real]] = cache["weights"][at[real]] + added[real]
    return dict(out=out, weights=cache["weights"])


def _plain_write(state):
    """Every block that is written into gets the smallest power of two for its new tokens, its old one at least if it holds tokens
    already, which are then rounded to the new one; new tokens are rounded over it."""
    (case, cache) = (state["case"], state["tensors"])
    (batch, heads) = (case["batch"], case["heads"])
    pages = cache["keys"].size(0)
    (b, t) = _rows(state)
    place = state["starts"][b] + t
    nth = place // PAGE - state["starts"][b] // PAGE                  # block among those that the sequence writes into
    block = state["starts"][:, None] // PAGE + torch.arange(state["widest"], device=DEV)
    inside = block * PAGE < state["lengths"][:, None]
    touched = torch.where(inside, state["table"].gather(1, block.clamp(max=state["table"].size(1) - 1).long()), EMPTY).long()
    real = touched < pages
    touched = touched.clamp(max=pages - 1)
    before = (state["starts"][:, None] - PAGE * block).clamp(0, PAGE)  # tokens that a block holds already
    mixed = (torch.arange(PAGE, device=DEV) < before[..., None])[:, :, None, :, None]
    got = {}
    for (which, name, rows) in ((0, "keys", state["new_keys"].float()), (1, "values", state["new_values"].float())):
        flat = (b * state["widest"] + nth).long()[:, None].expand(-1, heads)
        top = torch.zeros((batch * state["widest"], heads), device=DEV).scatter_reduce(0, flat, rows.abs().amax(-1), "amax").unflatten(0, (batch, -1))
        was = cache["scales"][touched][..., which].to(torch.int32) - 127
        e = torch.where(before[..., None] > 0, torch.maximum(was, _least_exponent(top)), _least_exponent(top))
        held = cache[name][touched[real]]
        old = _by_token(held) if which else held
        again = _coded(_decoded(old, (was[real] + 127)[..., None].expand(-1, -1, PAGE)), e[real][..., None, None])
        old = torch.where(mixed[real], again, old)
        cache[name][touched[real]] = old.unflatten(2, (16, 4)).transpose(-1, -2) if which else old
        cache["scales"][..., which][touched[real]] = (e[real] + 127).to(torch.uint8)
        page = touched[b, nth][:, None]
        (head, token) = (torch.arange(heads, device=DEV), (place % PAGE)[:, None])
        code = _coded(rows, e[b, nth][..., None])
        if which:
            cache[name][page, head, token // 4, :, token % 4] = code
        else:
            cache[name][page, head, token] = code
        got[name] = _decoded(code, e[b, nth] + 127).to(state["new_keys"].dtype)
    cache["weights"][page, head, token] = 0.0
    cache["positions"][page, head, token] = place[:, None].expand(-1, heads).to(torch.int32)
    return dict(keys=got["keys"], values=got["values"], weights=cache["weights"], positions=cache["positions"])


def _plain_evict(state):
    """Tokens are ranked: the latest `recent` positions before all others, then by weight, of equal ones the earlier place.  The best
    `keep` stay; those of them that stand behind the first `keep` places move, in their order, to the places there that got free.  What
    stands behind the first `keep` places is left as it is, also on the page where they end, whose power may have grown."""
    (case, cache) = (state["case"], state["tensors"])
    (keep, batch, heads) = (case["keep"], case["batch"], case["heads"])
    cache["weights"].copy_(state["weights"])  # as another part of the program left them
    cache["positions"].copy_(state["positions"])
    at = state["table"].long().clamp(max=cache["keys"].size(0) - 1)
    weights = cache["weights"][at].transpose(1, 2).flatten(2)  # [sequences, heads, places]
    positions = cache["positions"][at].transpose(1, 2).flatten(2).long()
    place = torch.arange(weights.size(2), device=DEV)
    held = (place < state["lengths"][:, None, None]).expand_as(weights)
    newest = torch.where(held, positions, -1).amax(-1, keepdim=True)
    rank = torch.where(positions > newest - case["recent"], math.inf, weights)
    order = torch.sort(torch.where(held, rank, -math.inf), dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(held).scatter(2, order[..., :keep], True) & held
    free = (held & ~stays & (place < keep)).nonzero()          # by sequence, head and place: as many as there are to move
    moves = (stays & (place >= keep)).nonzero()
    ((b, h, to), (_, _, source)) = (free.unbind(1), moves.unbind(1))
    (page, token) = (at[b, to // PAGE], to % PAGE)
    (page0, token0) = (at[b, source // PAGE], source % PAGE)
    unit = page * heads + h
    stands = torch.full((cache["keys"].size(0),), PAGE, device=DEV)  # tokens of a page before the first `keep` places end
    if keep < weights.size(2):
        stands[at[:, keep // PAGE]] = keep % PAGE
    token_of = {"keys": torch.arange(PAGE, device=DEV)[:, None], "values": torch.arange(PAGE, device=DEV).view(16, 1, 4)}
    for (which, name) in ((0, "keys"), (1, "values")):
        x = cache[name][page0, h, token0] if which == 0 else cache[name][page0, h, token0 // 4, :, token0 % 4]
        x = _decoded(x, cache["scales"][page0, h, which])
        was = cache["scales"][..., which].flatten().to(torch.int32) - 127
        e = was.scatter_reduce(0, unit, _least_exponent(x.abs().amax(-1)), "amax")  # of every page and head
        grown = (e > was).nonzero()[:, 0]
        flat = cache[name].flatten(0, 1)
        old = flat[grown]
        again = _coded(_decoded(old.flatten(1), was[grown] + 127), e[grown][:, None]).view_as(old)
        flat[grown] = torch.where(token_of[name] < stands[grown // heads].view(-1, *[1] * (old.dim() - 1)), again, old)
        cache["scales"][..., which] = (e + 127).view(-1, heads).to(torch.uint8)
        if which:
            cache[name][page, h, token // 4, :, token % 4] = _coded(x, e[unit][:, None])
        else:
            cache[name][page, h, token] = _coded(x, e[unit][:, None])
    cache["weights"][page, h, token] = cache["weights"][page0, h, token0]
    cache["positions"][page, h, token] = cache["positions"][page0, h, token0]
    return _after_eviction(state, state["lengths"].clamp(max=keep))


def _after_eviction(state, lengths):
    t = state["tensors"]
    return dict(lengths=lengths, keys=t["keys"].view(CODES), values=t["values"].view(CODES), scales=t["scales"], weights=t["weights"],
                positions=t["positions"])


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"write": _plain_write, "attend": _plain_attend, "weigh": _plain_attend, "evict": _plain_evict}[op](state)
    from vectorlink_gpu.attention import attend

    (cache, table, lengths) = (state["cache"], state["table"], state["lengths"])
    if op == "attend":
        return attend(state["queries"], cache, table, lengths, offsets=state["offsets"], causal=case["causal"])
    if op == "weigh":
        out = attend(state["queries"], cache, table, lengths, offsets=state["offsets"], causal=case["causal"], accumulate=True)
        return dict(out=out, weights=cache.weights)
    if op == "write":
        cache.write(state["new_keys"], state["new_values"], table, state["starts"], offsets=state["offsets"])
        (k, v) = cache.read(table, state["starts"], state["new_keys"].size(0), offsets=state["offsets"], dtype=state["new_keys"].dtype)
        return dict(keys=k, values=v, weights=cache.weights, positions=cache.positions)
    cache.weights.copy_(state["weights"])
    cache.positions.copy_(state["positions"])
    return _after_eviction(state, cache.evict(table, lengths, case["keep"], recent=case["recent"]))


def work(case):
    """Inputs read once, outputs written once: of a cache what attention sees; of an eviction all weights and positions, and the
    tokens that move, as many as weights that do not depend on the place leave to move."""
    (lengths, new) = _lengths(case)
    (heads, group, dim) = (case["heads"], case["group"], case["dim"])
    rows = sum(new)
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    token = heads * 2 * dim  # bytes of a token in the cache
    if case["op"] == "write":
        return dict(bytes=4.0 * size * rows * heads * dim + 2.0 * rows * token + 8.0 * rows * heads, flops=8.0 * rows * heads * dim)
    if case["op"] == "evict":
        (keep, recent) = (case["keep"], case["recent"])
        moved = 0.0
        for n in lengths:
            if n > keep:
                late = min(recent, n - keep)  # of those behind the budget, the ones that stay whatever their weight
                moved += late + (n - keep - late) * (keep - recent) / max(1, n - recent)
        return dict(bytes=2.0 * moved * (token + 8 * heads) + 16.0 * sum(lengths) * heads, flops=4.0 * sum(lengths) * heads)
    # of a sequence's new tokens, each sees what stands before it and itself
    pairs = sum(m * n - (m * (m - 1) / 2 if case["causal"] else 0) for n, m in zip(lengths, new) if n)
    weights = 8.0 * sum(lengths) * heads if case["op"] == "weigh" else 0.0
    return dict(bytes=2.0 * size * rows * heads * group * dim + sum(lengths) * token + weights, flops=4.0 * pairs * heads * group * dim)


def _stands_for(code):
    """Values of codes in 64 bits from the bits' meaning"""
    c = code.long()
    (up, part) = ((c >> 3) & 15, (c & 7).double())
    mag = torch.where(up == 0, part * 2.0 ** -9, (8 + part) * torch.exp2(up.double() - 10))
    return torch.where(c >= 128, -mag, mag)


def _nearest(x, e):
    """x in 64 bits over 2^e as the nearest value of the code, of two as near the one with an even last bit"""
    a = x.abs() * torch.exp2(-e.double())
    step = torch.exp2((torch.frexp(a).exponent - 4).clamp(min=-9).double())
    return torch.sign(x) * torch.round(a / step) * step


def _fitting(top):
    """The smallest exponent, LEAST at least, whose 448-fold is not below top, in 64 bits"""
    e = torch.full_like(top, LEAST, dtype=torch.int64)
    wanted = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448) - 1e-9).long()
    wanted = torch.where(top > 448 * torch.exp2(wanted.double()), wanted + 1, wanted)
    return torch.maximum(e, wanted)


def _held(state, b, head, which):
    """The keys (0) or values (1) of all blocks of a sequence, [blocks * 64, dim] in 64 bits"""
    t = state["tensors"]
    page = state["table"][b].long().clamp(max=t["keys"].size(0) - 1)
    x = t["values"][page, head].transpose(-1, -2).flatten(1, 2) if which else t["keys"][page, head]
    return (_stands_for(x) * torch.exp2(t["scales"][page, head, which].double() - 127)[:, None, None]).flatten(0, 1)


def exact(case, seed):
    """The definitions in 64 bits, a sequence and a head at a time."""
    state = prepare(case, seed)
    tensors = state["tensors"]
    lengths = state["lengths"].tolist()
    (heads, group, dim, batch) = (case["heads"], case["group"], case["dim"], case["batch"])
    if case["op"] == "evict":
        return _exact_evict(state, lengths)
    rows = state["queries"].size(0)
    offsets = list(range(rows + 1)) if state["offsets"] is None else state["offsets"].tolist()
    if case["op"] == "write":
        got = {}
        starts = state["starts"].tolist()
        for (which, name) in ((0, "keys"), (1, "values")):
            new = state["new_" + name].double()
            got[name] = torch.zeros_like(new)
            for b in range(batch):
                (place, first) = (starts[b], offsets[b])
                while first < offsets[b + 1]:
                    n = min(PAGE - place % PAGE, offsets[b + 1] - first)
                    part = new[first:first + n]
                    e = _fitting(part.abs().amax((0, 2)))
                    if place % PAGE:
                        page = int(state["table"][b, place // PAGE])
                        e = torch.maximum(e, tensors["scales"][page, :, which].long() - 127)
                    got[name][first:first + n] = _nearest(part, e[:, None]) * torch.exp2(e.double())[:, None]
                    (place, first) = (place + n, first + n)
        weights = tensors["weights"].double()
        positions = tensors["positions"].long()
        for b in range(batch):
            place = torch.arange(starts[b], starts[b] + offsets[b + 1] - offsets[b], device=DEV)
            page = state["table"][b, place // PAGE].long()
            weights[page, :, place % PAGE] = 0.0
            positions[page, :, place % PAGE] = place[:, None]
        return dict(keys=got["keys"], values=got["values"], weights=weights, positions=positions.to(torch.int32))
    out = torch.zeros((rows, heads * group, dim), dtype=torch.float64, device=DEV)
    weights = tensors["weights"].double() if case["op"] == "weigh" else None
    for b in range(batch):
        (first, end, n) = (offsets[b], offsets[b + 1], lengths[b])
        if n == 0:
            continue
        last = torch.full((end - first,), n - 1, device=DEV)
        if case["causal"]:
            last = n - (end - first) + torch.arange(end - first, device=DEV)
        hidden = torch.arange(n, device=DEV)[None] > last[:, None]
        place = torch.arange(n, device=DEV)
        page = state["table"][b, place // PAGE].long()
        for h in range(heads):
            (k, v) = (_held(state, b, h, which)[:n] for which in (0, 1))
            k = k.T.contiguous()
            for g in range(h * group, (h + 1) * group):
                s = torch.matmul(state["queries"][first:end, g].double(), k) / math.sqrt(dim)
                s = torch.softmax(s.masked_fill_(hidden, -math.inf), dim=1)
                out[first:end, g] = torch.matmul(s, v)
                if weights is not None:
                    weights[page, h, place % PAGE] += s.sum(0)
    return out if weights is None else dict(out=out, weights=weights)


def _exact_evict(state, lengths):
    (case, t) = (state["case"], state["tensors"])
    (keep, recent) = (case["keep"], case["recent"])
    token_values = t["values"].transpose(-1, -2).flatten(2, 3)
    codes = [_stands_for(t["keys"]), _stands_for(token_values)]
    exponent = t["scales"].long() - 127
    (weights, positions) = (t["weights"].double(), t["positions"].long())
    for b, n in enumerate(lengths):
        if n <= keep:
            continue
        place = torch.arange(n, device=DEV)
        page = state["table"][b, place // PAGE].long()
        for h in range(case["heads"]):
            (w, p) = (weights[page, h, place % PAGE], positions[page, h, place % PAGE])
            late = p > p.max() - recent
            # the best first: late ones, then large weights, then early places
            order = torch.sort(w, descending=True, stable=True).indices
            order = order[torch.sort((~late[order]).long(), stable=True).indices]
            stays = torch.zeros(n, dtype=torch.bool, device=DEV)
            stays[order[:keep]] = True
            to = place[:keep][~stays[:keep]]
            source = place[keep:][stays[keep:]]
            (page1, page0) = (page[to], page[source])
            for which in (0, 1):
                x = codes[which][page0, h, source % PAGE] * torch.exp2(exponent[page0, h, which].double())[:, None]
                need = _fitting(x.abs().amax(1))
                e = exponent[:, h, which].scatter_reduce(0, page1, need, "amax")
                grown = (e > exponent[:, h, which]).nonzero()[:, 0]
                was = torch.exp2(exponent[grown, h, which].double())[:, None, None]
                before = codes[which][page[keep // PAGE], h, keep % PAGE:].clone()
                codes[which][grown, h] = _nearest(codes[which][grown, h] * was, e[grown][:, None, None])
                codes[which][page[keep // PAGE], h, keep % PAGE:] = before  # behind what stays nothing changes
                exponent[:, h, which] = e
                codes[which][page1, h, to % PAGE] = _nearest(x, e[page1][:, None])
            weights[page1, h, to % PAGE] = w[source]
            positions[page1, h, to % PAGE] = p[source]
    scales = t["scales"].long()
    scales[..., :2] = exponent[..., :2] + 127
    return dict(lengths=state["lengths"].clamp(max=keep), keys=codes[0], values=codes[1].unflatten(2, (16, 4)).transpose(-1, -2),
                scales=scales.to(torch.uint8), weights=weights, positions=positions.to(torch.int32))
