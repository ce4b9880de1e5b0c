"""Plain 64-bit forms of the int4 products and of the experts' router, from their definitions."""
from __future__ import annotations

import torch


def pack(values: torch.Tensor) -> torch.Tensor:
    """Codes of whole numbers [rows, k], a byte at a time."""
    rows, k = values.shape
    nb = (k + 31) // 32
    full = torch.zeros(rows, nb * 32, dtype=torch.long, device=values.device)
    full[:, :k] = values.long()
    out = torch.zeros(rows, nb * 16, dtype=torch.long, device=values.device)
    for b in range(4):
        out[:, b::4] = full[:, b::8] + 16 * full[:, b + 4::8]
    return out.to(torch.uint8)


def weight(values: torch.Tensor, scales: torch.Tensor, zeros, group: int) -> torch.Tensor:
    """w [..., k] in 64 bits."""
    col = torch.arange(values.shape[-1], device=values.device) // group
    z = zeros.double()[..., col] if zeros is not None else 8.0
    return (values.double() - z) * scales.double()[..., col]


def reach(values: torch.Tensor, scales: torch.Tensor, zeros, group: int) -> torch.Tensor:
    """s (q + z): the magnitudes of the terms where x meets q and z apart."""
    col = torch.arange(values.shape[-1], device=values.device) // group
    z = zeros.double()[..., col] if zeros is not None else 8.0
    return (values.double() + z) * scales.double()[..., col].abs()


def random_weight(g: torch.Generator, shape, k: int, group: int, dtype, zeros: bool, device, whole: bool = False):
    """(values [*shape, k], scales, zeros): any values, zeros up to 16, scales of a layer, or `whole`: powers of two."""
    groups = (k + group - 1) // group
    values = torch.randint(0, 16, (*shape, k), generator=g, device=device, dtype=torch.uint8)
    if whole:
        scales = torch.exp2(torch.randint(-1, 2, (*shape, groups), generator=g, device=device).float())
    else:
        scales = 0.01 * torch.exp(0.5 * torch.randn(*shape, groups, generator=g, device=device))
    z = torch.randint(0, 17, (*shape, groups), generator=g, device=device, dtype=torch.uint8) if zeros else None
    return values, scales.to(dtype), z


def scores_of(logits: torch.Tensor, scores: str) -> torch.Tensor:
    """Scores in 64 bits; zero in rows that are -inf throughout."""
    l = logits.double()
    if scores == "sigmoid":
        return torch.sigmoid(l)
    empty = (l == float("-inf")).all(dim=1, keepdim=True)
    return torch.where(empty, torch.zeros_like(l), torch.softmax(torch.where(empty, torch.zeros_like(l), l), dim=1))


def route(logits, top, scores="softmax", bias=None, normalize=True, scale=1.0):
    """(ids, weights) a token and an expert at a time."""
    l = logits.cpu()
    score = scores_of(l, scores)
    key = l.double() if bias is None else score + bias.cpu().double()
    key = torch.where((l == float("-inf")) | torch.isnan(l) | torch.isnan(key), torch.full_like(key, float("-inf")), key)
    ids = torch.full((l.shape[0], top), -1, dtype=torch.int32)
    for t in range(l.shape[0]):
        order = sorted(range(l.shape[1]), key=lambda e: (-float(key[t, e]), e))
        chosen = [e for e in order if float(key[t, e]) > float("-inf")][:top]
        ids[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return ids.to(logits.device), shares_of(logits, ids.to(logits.device), scores, normalize) * scale


def shares_of(logits, ids, scores, normalize):
    """Shares of the chosen experts, differentiable, in 64 bits."""
    there = ids >= 0
    l = logits.double()
    if ids.shape[1] == 0:
        return torch.zeros(ids.shape, dtype=torch.float64, device=l.device)
    if normalize and scores == "softmax":  # the quotient of two softmaxes, without their common sum
        chosen = torch.where(there, l.gather(1, ids.clamp(min=0).long()), torch.full((), float("-inf"), dtype=torch.float64, device=l.device))
        top = chosen.amax(dim=1, keepdim=True)
        e = torch.where(there, torch.exp(chosen - torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)), torch.zeros_like(chosen))
        total = e.sum(dim=1, keepdim=True)
        return e / torch.where(total == 0, torch.ones_like(total), total)
    mine = torch.where(there, scores_of(logits, scores).gather(1, ids.clamp(min=0).long()), torch.zeros((), dtype=torch.float64, device=l.device))
    if not normalize:
        return mine
    total = mine.sum(dim=1, keepdim=True)
    return mine / torch.where(total == 0, torch.ones_like(total), total)


def balance(logits, ids, scores):
    """(loss, counts), differentiable by the logits, in 64 bits."""
    experts = logits.shape[1]
    counts = torch.stack([(ids == e).sum() for e in range(experts)])
    live = torch.where((logits > float("-inf")).any(dim=1) | torch.isnan(logits).any(dim=1))[0]
    if live.numel() == 0 or int(counts.sum()) == 0:
        return logits.double().nan_to_num(0, 0, 0).sum() * 0, counts.int()
    p = scores_of(logits[live], scores)
    p = p / p.sum(dim=1, keepdim=True)
    return experts * (counts.double() / counts.sum() * p.mean(dim=0)).sum(), counts.int()
