"""Definitions of the cache in 4 bits and of attention over it in 64 bits, a sequence and a head at a time (include/vlgpu.h)."""
import math

import torch

PAGE = 64
MAXINT = 2147483647
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def rounded(x):
    """x [..., dim] as the cache holds it; a row with an element that is not finite is NaN."""
    x = x.detach().cpu().double()
    out = torch.empty_like(x)
    for g in range(0, x.size(-1), 32):
        part = x[..., g:g + 32]
        top = torch.where(part.isfinite(), part, 0.0).abs().amax(-1, keepdim=True)
        e = torch.where(top > 0, torch.frexp(top).exponent - 1, -1000) - 2
        power = torch.exp2(e.clamp(min=-124).double())
        a = part.abs() / power
        # distance to every point of the grid; the even code of two as near comes first
        order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
        near = (a[..., None] - GRID[order]).abs()
        out[..., g:g + 32] = torch.sign(part) * GRID[order][near.argmin(-1)] * power
    out[~x.isfinite().all(-1)] = math.nan
    return out


def values_of(packed, scales):
    """packed uint8 [n, dim / 2], scales uint8 [n, dim / 32] -> [n, dim] in 64 bits"""
    (packed, scales) = (packed.cpu().long(), scales.cpu().long())
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    v = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    power = torch.where(scales == 255, math.nan, torch.exp2((scales - 127).double()))
    return v * power.repeat_interleave(32, dim=-1)


def unpacked(cache, page, h):
    """(keys, values) [64, dim] of a page"""
    v = cache.values[page, h].transpose(1, 2).flatten(2).flatten(0, 1)
    return (values_of(cache.keys[page, h], cache.key_scales[page, h].T), values_of(v, cache.value_scales[page, h].T))


def bounds_of(keys, values):
    """(hi, lo, exponent) of a page's tokens [n, dim]; exponent 127: no bounds"""
    if not (keys.isfinite().all() and values.isfinite().all()):
        return None, None, 127
    (hi, lo) = (keys.amax(0), keys.amin(0))
    top = float(torch.maximum(hi.abs(), lo.abs()).max())
    e = max(math.frexp(top)[1] - 1 - 6, -126) if top else -126
    return torch.ceil(hi * 2.0 ** -e), torch.floor(lo * 2.0 ** -e), e


class Held:
    """What a cache holds of the sequences of a table, in 64 bits."""

    def __init__(self, cache, table, lengths):
        (self.k, self.v) = ({}, {})
        self.lengths = [min(max(int(n), 0), table.size(1) * PAGE) for n in lengths]
        table = table.cpu()
        for b, n in enumerate(self.lengths):
            for h in range(cache.heads):
                ks, vs = [], []
                for i in range(-(-n // PAGE)):
                    page = int(table[b, i])
                    if 0 <= page < cache.pages:
                        (k, v) = unpacked(cache, page, h)
                    else:
                        k = v = torch.full((PAGE, cache.dim), -math.inf, dtype=torch.float64)  # takes no part
                    ks.append(k)
                    vs.append(v)
                self.k[b, h] = torch.cat(ks)[:n] if n else torch.zeros((0, cache.dim), dtype=torch.float64)
                self.v[b, h] = torch.cat(vs)[:n] if n else torch.zeros((0, cache.dim), dtype=torch.float64)


def attention(queries, cache, table, lengths, offsets=None, scale=None, causal=True, blocks=None):
    """(out, lse, slack): slack bounds what 32-bit sums and exponentials may be off by, in units of 2^-24, per row and head; and the
    sum of weighted magnitudes, which errors of the weights scale with."""
    q = queries.detach().cpu().double()
    (rows, heads, dim) = q.shape
    group = heads // cache.heads
    scale = dim ** -0.5 if scale is None else scale
    lengths = lengths.cpu().tolist()
    offsets = list(range(rows + 1)) if offsets is None else offsets.cpu().tolist()
    held = Held(cache, table, lengths)
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    slack = torch.zeros((rows, heads), dtype=torch.float64)
    size = torch.zeros((rows, heads, dim), dtype=torch.float64)
    for b in range(table.size(0)):
        n = held.lengths[b]
        for row in range(offsets[b], offsets[b + 1]):
            sees = n
            if causal or blocks is not None:
                sees = min(max(lengths[b] - (offsets[b + 1] - offsets[b]) + row - offsets[b] + 1, 0), n)
            for h in range(cache.heads):
                (k, v) = (held.k[b, h][:sees], held.v[b, h][:sees])
                at = torch.arange(sees)
                if blocks is not None:
                    at = torch.cat([torch.arange(int(x) * PAGE, min(int(x) * PAGE + PAGE, sees))
                                    for x in blocks[row, h].tolist() if 0 <= x < table.size(1) and x * PAGE < sees] + [at[:0]])
                at = at[~torch.isneginf(k[at, 0])]
                (k, v) = (k[at], v[at])
                if not len(at):
                    continue
                for g in range(h * group, (h + 1) * group):
                    s = k @ q[row, g] * scale
                    spoilt = bool(s.isnan().any() or v.isnan().any())
                    p = torch.softmax(s, 0)
                    out[row, g] = math.nan if spoilt else p @ v
                    lse[row, g] = math.nan if spoilt else torch.logsumexp(s, 0)
                    slack[row, g] = (dim + 8) * float((k.abs() @ q[row, g].abs()).max()) * abs(scale) + 4 * float(s.abs().max()) + len(at) / 16 + 16
                    size[row, g] = p @ v.abs()
    return out, lse, slack, size


def check_attention(got, want, dtype):
    """Tolerances: the weights are rounded to 8, 16 or 24 bits (relative 2^-9, 2^-16, 2^-24 with a cut before the last part),
    scores and exponentials are off by slack * 2^-24 at most, and the result is rounded once to its type."""
    (out, _, slack, size) = want
    weight = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}[dtype]
    last = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), out.isnan())
    # the error of a weight counts twice: in the sum of values and in the sum that it is divided by
    room = 2 * (weight + slack[..., None] * 2.0 ** -24) * size + 1.01 * last * out.abs() + 2.0 ** -24
    bad = ((got - out).abs() > room) & ~out.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - out).abs() / room).nan_to_num().max()):.2f} times the bound"


def selection(queries, cache, table, lengths, count, offsets=None):
    q = queries.detach().cpu().double()
    (rows, heads, dim) = q.shape
    group = heads // cache.heads
    lengths = lengths.cpu().tolist()
    offsets = list(range(rows + 1)) if offsets is None else offsets.cpu().tolist()
    table = table.cpu()
    out = torch.full((rows, cache.heads, count), MAXINT, dtype=torch.int32)
    for b in range(table.size(0)):
        if cache.pages and table.size(1):
            pages = table[b].long().clamp(0, cache.pages - 1).to(cache.bounds.device)
            (edge, power) = (cache.bounds[pages].cpu().double(), cache.bound_scales[pages].cpu().long())  # of its blocks
        for row in range(offsets[b], offsets[b + 1]):
            place = lengths[b] - (offsets[b + 1] - offsets[b]) + row - offsets[b]
            if place < 0 or table.size(1) == 0:
                continue
            own = min(place, table.size(1) * PAGE - 1) // PAGE
            for h in range(cache.heads):
                u = q[row, h * group:(h + 1) * group]
                top = float(u.abs().max()) if bool(u.isfinite().all()) else 0.0
                e = max(math.frexp(top)[1] - 1 - 6, -100) if top else 0
                u = torch.clamp(torch.round(u * 2.0 ** -e), -127, 127) if top else torch.zeros_like(u)
                scores = []
                for i in range(own + 1):
                    page = int(table[b, i])
                    if i == own:
                        scores.append((3, 0.0))
                    elif not 0 <= page < cache.pages:
                        continue
                    elif int(power[i, h]) == 127:
                        scores.append((2, 0.0))
                    else:
                        s = u.clamp(min=0) @ edge[i, h, 0] + u.clamp(max=0) @ edge[i, h, 1]
                        scores.append((1, float(s.max()) * 2.0 ** int(power[i, h])))
                    scores[-1] = (*scores[-1], -i)
                best = sorted(-s[2] for s in sorted(scores, reverse=True)[:count])
                out[row, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out
