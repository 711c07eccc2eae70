"""Definitions of the cache in 8 bits, of the weights that attention gives its tokens and of eviction in 64 bits (include/vlgpu.h)."""
import math

import torch

PAGE = 64
EPS = 2.0 ** -24


def exponent(top):
    """The least e, -117 to 119, with top <= 448 * 2^e"""
    if top == 0:
        return -117
    (part, e) = math.frexp(top)
    return min(max(e - 9 + (part > 0.875), -117), 119)


def nearest(x):
    """x in 64 bits as the nearest code's value, of two as near the even one, magnitudes over 448 as 448; NaN stays"""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2((torch.frexp(a).exponent - 4).clamp(min=-9).double())
    return torch.sign(x) * torch.round(a / step) * step


def decoded(code):
    c = code.cpu().long()
    (up, part) = (c >> 3 & 15, (c & 7).double())
    mag = torch.where(up == 0, part * 2.0 ** -9, (8 + part) * torch.exp2(up.double() - 10))
    mag = torch.where((c & 127) == 127, math.nan, mag)
    return torch.where(c >= 128, -mag, mag)


def by_token(values):
    """[..., 16, dim, 4] -> [..., 64, dim]"""
    return values.transpose(-1, -2).flatten(-3, -2)


class Model:
    """A cache as numbers: per kind codes' values [pages, heads, 64, dim] in 64 bits and exponents [pages, heads]."""

    def __init__(self, cache):
        (self.pages, self.heads, self.dim) = (cache.pages, cache.heads, cache.dim)
        self.codes = [decoded(cache.keys), decoded(by_token(cache.values))]
        scales = cache.scales.cpu().long()
        self.e = [(scales[..., i] - 127).clamp(-117, 119) for i in (0, 1)]
        self.marked = scales[..., 2] != 0
        self.weights = cache.weights.cpu().double() if cache.weights is not None else None
        self.positions = cache.positions.cpu().long() if cache.positions is not None else None

    def values_of(self, which, page, h):
        return self.codes[which][page, h] * 2.0 ** int(self.e[which][page, h])

    def raise_to(self, which, page, h, e, tokens):
        """Rounds the first tokens of a page to a larger power."""
        was = int(self.e[which][page, h])
        if e > was:
            part = self.codes[which][page, h, :tokens]
            self.codes[which][page, h, :tokens] = torch.where(part.isnan(), part, nearest(part * 2.0 ** (was - e)))
            self.e[which][page, h] = e

    def write(self, rows, table, starts, offsets, positions=None):
        table = table.cpu()
        rows = [r.detach().cpu().double() for r in rows]
        for b in range(table.size(0)):
            (place, row) = (min(max(int(starts[b]), 0), table.size(1) * PAGE), offsets[b])
            while row < offsets[b + 1]:
                n = min(PAGE - place % PAGE, offsets[b + 1] - row)
                page = int(table[b, place // PAGE]) if place // PAGE < table.size(1) else -1
                if 0 <= page < self.pages:
                    (j, stop) = (place % PAGE, place % PAGE + n)
                    for h in range(self.heads):
                        self.marked[page, h] = bool(self.marked[page, h]) if j else False
                        for which in (0, 1):
                            x = rows[which][row:row + n, h]
                            bad = ~x.isfinite().all(-1)
                            e = exponent(float(x[~bad].abs().max()) if bool((~bad).any()) else 0.0)
                            if j:
                                e = max(e, int(self.e[which][page, h]))
                                self.raise_to(which, page, h, e, j)
                            self.e[which][page, h] = e
                            new = nearest(x * 2.0 ** -e)
                            new[bad] = math.nan
                            self.codes[which][page, h, j:stop] = new
                            if bool(bad.any()):
                                self.marked[page, h] = True
                    if self.weights is not None:
                        self.weights[page, :, j:stop] = 0
                        at = torch.arange(place, place + n) if positions is None else positions[row:row + n].cpu().long()
                        self.positions[page, :, j:stop] = at
                (place, row) = (place + n, row + n)

    def pages_of(self, table, b, n):
        return [int(p) if 0 <= int(p) < self.pages else -1 for p in table[b, :-(-n // PAGE)].tolist()]

    def evict(self, table, lengths, keep, recent):
        table = table.cpu()
        left = []
        for b, n in enumerate(lengths.cpu().tolist()):
            n = min(max(n, 0), table.size(1) * PAGE)
            if n <= keep:
                left.append(n)
                continue
            pages = self.pages_of(table, b, n)
            there = [i for i in range(n) if pages[i // PAGE] >= 0]
            kept = min(keep, len(there))
            left.append(kept)
            for h in range(self.heads):
                at = {i: (pages[i // PAGE], h, i % PAGE) for i in there}
                newest = max((int(self.positions[at[i]]) for i in there), default=0)

                def rank(i):
                    w = float(self.weights[at[i]])
                    late = int(self.positions[at[i]]) > newest - recent
                    return (not late, w != w, 0.0 if late or w != w else -w, i)

                stay = set(sorted(there, key=rank)[:kept])
                holes = [i for i in range(kept) if i not in stay]
                movers = sorted(i for i in stay if i >= kept)
                assert len(holes) == len(movers)
                moved = {}
                for to, source in zip(holes, movers):
                    if to in at:
                        moved.setdefault(to // PAGE, []).append((to, at[source]))
                image = [[self.values_of(which, p, h) for _, (p, _, _) in sum(moved.values(), [])] for which in (0, 1)]
                image = [iter(x) for x in image]
                for block, pairs in moved.items():
                    page = pages[block]
                    for which in (0, 1):
                        rows = [next(image[which])[token] for _, (_, _, token) in pairs]
                        need = [exponent(float(x.abs().max())) for x in rows if not bool(x.isnan().any())]
                        e = max(need + [int(self.e[which][page, h])])
                        self.raise_to(which, page, h, e, min(kept - block * PAGE, PAGE))
                        for (to, _), x in zip(pairs, rows):
                            spoilt = bool(x.isnan().any())
                            self.codes[which][page, h, to % PAGE] = math.nan if spoilt else nearest(x * 2.0 ** -e)
                            if spoilt:
                                self.marked[page, h] = True
                    for to, source in pairs:
                        self.weights[page, h, to % PAGE] = self.weights[source]
                        self.positions[page, h, to % PAGE] = self.positions[source]
        return left

    def check(self, cache):
        """Every code, power, weight and position of the cache is the model's."""
        other = Model(cache)
        for which in (0, 1):
            assert torch.equal(self.e[which], other.e[which]), ("keys", "values")[which]
            (a, b) = (self.codes[which], other.codes[which])
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()), ("keys", "values")[which]
        assert bool((other.marked | ~self.marked).all()), "a page whose token is not finite is not marked"
        if self.weights is not None:
            assert torch.equal(self.weights.nan_to_num(-7.0, 1e30, -1e30), other.weights.nan_to_num(-7.0, 1e30, -1e30))
            assert torch.equal(self.positions, other.positions)


def attention(queries, cache, table, lengths, offsets=None, scale=None, causal=True, model=None):
    """(out, lse, slack, size) as attention_reference.attention has them, and the weights that the tokens get [pages, heads, 64] with
    what their sums may be off by."""
    model = Model(cache) if model is None else model
    q = queries.detach().cpu().double()
    (rows, heads, dim) = q.shape
    group = heads // model.heads
    scale = dim ** -0.5 if scale is None else scale
    table = table.cpu()
    lengths = lengths.cpu().tolist()
    offsets = list(range(rows + 1)) if offsets is None else offsets.cpu().tolist()
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    slack = torch.zeros((rows, heads), dtype=torch.float64)
    size = torch.zeros((rows, heads, dim), dtype=torch.float64)
    added = torch.zeros((model.pages, model.heads, PAGE), dtype=torch.float64)
    room = torch.zeros_like(added)
    for b in range(table.size(0)):
        n = min(max(lengths[b], 0), table.size(1) * PAGE)
        pages = model.pages_of(table, b, n)
        places = torch.tensor([i for i in range(n) if pages[i // PAGE] >= 0], dtype=torch.long)
        page = torch.tensor([pages[int(i) // PAGE] for i in places], dtype=torch.long)
        count = offsets[b + 1] - offsets[b]
        for h in range(model.heads):
            (k, v) = (model.codes[w][page, h, places % PAGE] * torch.exp2(model.e[w][page, h].double())[:, None] for w in (0, 1))
            for row in range(offsets[b], offsets[b + 1]):
                sees = min(max(lengths[b] - count + row - offsets[b] + 1, 0), n) if causal else n
                m = int((places < sees).sum())
                if not m:
                    continue
                for g in range(h * group, (h + 1) * group):
                    s = k[:m] @ q[row, g] * scale
                    spoilt = bool(s.isnan().any() or v[:m].isnan().any() or not s.isfinite().all())
                    p = torch.softmax(s, 0)
                    out[row, g] = math.nan if spoilt else p @ v[:m]
                    lse[row, g] = math.nan if spoilt else torch.logsumexp(s, 0)
                    if spoilt:
                        continue
                    off = (dim + 8) * float((k[:m].abs() @ q[row, g].abs()).max()) * abs(scale) + 4 * float(s.abs().max()) + m / 16 + 16
                    slack[row, g] = off
                    size[row, g] = p @ v[:m].abs()
                    added[page[:m], h, places[:m] % PAGE] += p
                    # a score off by its slack, the row's sum as much, and a rounding for every row that is added
                    room[page[:m], h, places[:m] % PAGE] += p * (2 * off + 4 + count * group) * EPS
    return (out, lse, slack, size), added, room


def check_output(got, want, dtype, many):
    """A weight is rounded to as many bits as its bfloat16 parts hold: one part is off by 2^-8 of it, a part cut off and one rounded by
    2^-16, three by 2^-24 (of bfloat16 the form for many rows takes one, for few rows two).  Scores, exponentials and sums are off by
    slack * 2^-24, in the sum of values and in the sum that it is divided by; the result is rounded once, by half a step."""
    (out, _, slack, size) = want
    weight = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8 if many and dtype == torch.bfloat16 else 2.0 ** -16
    last = torch.finfo(dtype).eps / 2
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), out.isnan())
    least = torch.finfo(dtype).smallest_normal * last  # half a step of a result below the normal ones
    room = (weight + 2 * slack[..., None] * EPS) * size * (1 + last) + last * out.abs() + least
    bad = ((got - out).abs() > room) & ~out.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - out).abs() / room).nan_to_num().max()):.2f} times the bound"


def check_weights(got, before, added, room):
    """got: weights after a call that found `before`; one more rounding where the sum is added to what was there."""
    want = before.double().cpu() + added
    got = got.double().cpu()
    bad = (got - want).abs() > room + EPS * want.abs() + 2.0 ** -120
    assert not bad.any(), f"{int(bad.sum())} weights off, worst {float((got - want).abs().max())}"
