"""Routing to experts and combining in 64 bits, token by token, for the tests."""
import math

import torch


def _ranked(values, among):
    """Indices of `among` by falling value, the lowest first among equals."""
    return sorted(among, key=lambda i: (-values[i], i))


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, tokens=None):
    """-> weights f64 [T, k], experts, rows, offsets, positions, as lists would have them"""
    x = logits.cpu().double()
    total, n = x.shape
    live = total if tokens is None else min(max(int(tokens), 0), total)
    b = None if bias is None else bias.cpu().double().tolist()
    size = n // groups
    weights, experts = torch.zeros((total, k), dtype=torch.float64), torch.full((total, k), -1, dtype=torch.int32)
    of_expert = [[] for _ in range(n)]
    largest = float(torch.finfo(torch.float32).max)
    for t in range(live):
        v = [-math.inf if math.isnan(l) else min(l, largest) for l in x[t].tolist()]
        if score == "softmax":
            top = max(v)
            e = [0.0 if top == -math.inf else math.exp(l - top) for l in v]
            s = [i / sum(e) if sum(e) else 0.0 for i in e]
        else:
            s = [0.0 if l < -700 else 1 / (1 + math.exp(-l)) for l in v]
        c = [s[i] + (b[i] if b else 0.0) for i in range(n)]
        c = [-math.inf if v[i] == -math.inf or math.isnan(c[i]) else min(c[i], largest) for i in range(n)]
        choice = c if b else v
        best = [sum(sorted((choice if group_top == 1 else c)[g * size:(g + 1) * size])[-group_top:]) for g in range(groups)]
        kept = _ranked(best, range(groups))[:top_groups]
        picked = _ranked(choice, [i for i in range(n) if i // size in kept])[:k]
        w = torch.tensor([0.0 if choice[i] == -math.inf else s[i] for i in picked], dtype=torch.float64)
        weights[t] = (w / (w.sum() + 1e-20) if renormalize else w) * scale
        experts[t] = torch.tensor(picked, dtype=torch.int32)
        for j, e in enumerate(picked):
            of_expert[e].append((t, j))
    rows, positions = torch.full((total * k,), -1, dtype=torch.int32), torch.full((total, k), -1, dtype=torch.int32)
    offsets, at = [0], 0
    for pairs in of_expert:
        for t, j in pairs:
            rows[at], positions[t, j] = t, at
            at += 1
        offsets.append(at)
    return weights, experts, rows, torch.tensor(offsets, dtype=torch.int32), positions


def combine(x, weights, positions, residual=None):
    """-> (y f64, sum of the magnitudes of its terms)"""
    x, weights, positions = x.cpu().double(), weights.cpu().double(), positions.cpu().long()
    there = (positions >= 0) & (positions < x.shape[0]) & (weights != 0)
    terms = x[positions.clamp(0, x.shape[0] - 1)]
    terms = torch.where(there.unsqueeze(2), terms * weights.unsqueeze(2), torch.zeros_like(terms))
    y, size = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        y, size = y + residual.cpu().double(), size + residual.cpu().double().abs()
    return y, size
