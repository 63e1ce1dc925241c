"""The router from its definition, in 64 bits on the CPU (score kept in fp32 where it is compared)."""
from __future__ import annotations

import torch


def scores(logits, score):
    l = logits.double()
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    empty = torch.isneginf(l).all(-1, keepdim=True)
    return torch.softmax(l.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)


def _rank(c):
    """Positions by falling value, NaN first, lowest position first among equals."""
    return torch.sort(c, dim=-1, descending=True, stable=True).indices


def choose(logits, k, r, bias=None):
    T, E = logits.shape
    c = logits.double()
    if bias is not None or (r.groups > 1 and r.group_score == "top2"):
        c = scores(logits, r.score).float()
        c = (c if bias is None else c + bias).double()
    size = E // r.groups
    out = []
    for row in c:
        keep = torch.ones(E, dtype=torch.bool)
        if r.groups > 1:
            best = torch.sort(row.view(r.groups, size), dim=-1, descending=True).values
            two = r.group_score == "top2" and size > 1
            rank = (best[:, 0].float() + best[:, 1].float()).double() if two else best[:, 0]
            keep = torch.zeros(r.groups, dtype=torch.bool)
            keep[_rank(rank)[:r.top_groups]] = True
            keep = keep.repeat_interleave(size)
        order = _rank(row)
        out.append(order[keep[order]][:k])
    return torch.stack(out) if out else torch.empty(0, k, dtype=torch.int64)


def shares(logits, ids, r):
    """The weights before the scale (differentiable in the logits), 64 bits."""
    l = logits.double()
    none = torch.isneginf(l.detach().gather(1, ids)).all(-1, keepdim=True)
    if not r.renormalize:
        if r.score == "sigmoid":
            return torch.sigmoid(l).gather(1, ids)
        empty = torch.isneginf(l.detach()).all(-1, keepdim=True)
        return torch.softmax(l.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0).gather(1, ids)
    chosen = l.gather(1, ids).masked_fill(none, 0.0)
    if r.score == "sigmoid":
        part = torch.nn.functional.logsigmoid(chosen)
        return torch.softmax(part, -1).masked_fill(none, 0.0)
    return torch.softmax(chosen, -1).masked_fill(none, 0.0)
