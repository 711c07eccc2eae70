"""Eviction's definition in 64 bits for long sequences: attention8_reference.Model.evict over whole heads at a time."""
import math

import torch

from attention8_reference import PAGE, nearest


def exponents(top):
    """attention8_reference.exponent of every number"""
    (part, e) = torch.frexp(top)
    return torch.where(top == 0, -117, (e - 9 + (part > 0.875)).clamp(-117, 119))


def evict(model, table, lengths, keep, recent):
    """Model.evict; the lengths that are left"""
    table = table.cpu()
    left = []
    for b, n in enumerate(lengths.cpu().tolist()):
        n = min(max(n, 0), table.size(1) * PAGE)
        if n <= keep:
            left.append(n)
            continue
        blocks = -(-n // PAGE)
        pages = table[b, :blocks].long()
        paged = (pages >= 0) & (pages < model.pages)
        pages = pages.clamp(0, max(model.pages - 1, 0))
        place = torch.arange(n)
        there = paged[place // PAGE]
        kept = min(keep, int(there.sum()))
        left.append(kept)
        if not kept:
            continue
        for h in range(model.heads):
            (w, p) = (t[pages, h].flatten()[:n] for t in (model.weights, model.positions))
            late = p > p[there].max() - recent
            # late ones first, as they stand; then by weight with NaN last, of equal ones the earlier place; what is on no page behind all
            group = torch.where(~there, 3, torch.where(late, 0, torch.where(w.isnan(), 2, 1)))
            order = torch.sort(torch.where(group == 1, -w, 0.0), stable=True).indices
            order = order[torch.sort(group[order], stable=True).indices]
            stay = torch.zeros(n, dtype=torch.bool)
            stay[order[:kept]] = True
            (holes, movers) = (place[:kept][~stay[:kept]], place[kept:][stay[kept:]])
            assert len(holes) == len(movers)
            real = there[holes]
            (holes, movers) = (holes[real], movers[real])
            (to, source) = ((pages[holes // PAGE], h, holes % PAGE), (pages[movers // PAGE], h, movers % PAGE))
            rows = [model.codes[k][source] * torch.exp2(model.e[k][source[0], h].double())[:, None] for k in (0, 1)]
            (weights, positions) = (model.weights[source], model.positions[source])
            for k in (0, 1):
                spoilt = rows[k].isnan().any(-1)
                need = torch.where(spoilt, -117, exponents(rows[k].abs().nan_to_num().amax(-1)).long())
                e = model.e[k][:, h].clone().scatter_reduce(0, to[0], need, "amax")
                for page in torch.unique(to[0][e[to[0]] > model.e[k][to[0], h]]).tolist():
                    block = int(holes[to[0] == page][0]) // PAGE
                    model.raise_to(k, page, h, int(e[page]), min(kept - block * PAGE, PAGE))
                new = nearest(rows[k] * torch.exp2(-e[to[0]].double())[:, None])
                new[spoilt] = math.nan
                model.codes[k][to] = new
                model.marked[to[0][spoilt], h] = True
            model.weights[to] = weights
            model.positions[to] = positions
    return left
