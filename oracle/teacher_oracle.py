"""Definitions of the frozen-teacher operators in float64 on the CPU (test infrastructure): 4-bit storage and its products,
top logits, distillation.  Written from the formulas, row by row where that is the plainest."""
from __future__ import annotations

import math

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx4_round(x: torch.Tensor):
    """the values [rows, cols] float64 that x's 4-bit form stands for, and the scale codes [rows, ceil(cols / 32)]"""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -cols % 32)).reshape(rows, -1, 32)
    big = b.abs().amax(-1)
    whole = torch.isfinite(big)
    e = torch.frexp(torch.where(whole, big, torch.ones_like(big))).exponent.double() - 1  # floor(log2 big)
    e = torch.where(big == 0, torch.full_like(e, -200.0), e)
    code = (e - 2 + 127).clamp(min=0.0)
    unit = torch.exp2(code - 127).unsqueeze(-1)
    a = (b / unit).abs()
    levels = torch.tensor(LEVELS, dtype=torch.float64)
    at = torch.searchsorted(levels, a.contiguous(), right=True) - 1   # the level at or below
    at = at.clamp(0, 7)
    up = (at + 1).clamp(max=7)
    lo, hi = a - levels[at], levels[up] - a
    take = (hi < lo) | ((hi == lo) & (up % 2 == 0))                    # nearest, ties to the even code
    v = torch.copysign(levels[torch.where(take & (up > at), up, at)], b) * unit
    v = torch.where(whole.unsqueeze(-1), v, torch.full_like(v, math.nan))
    code = torch.where(whole, code, torch.full_like(code, 255.0))
    return v.reshape(rows, -1)[:, :cols], code.to(torch.uint8)


def mx4_pack(x: torch.Tensor):
    """(codes uint8 [G, rows, 128], scales uint8 [G, rows, 8]) of x, from mx4_round's values"""
    rows, cols = x.shape
    pad = -cols % 256
    v, code = mx4_round(torch.nn.functional.pad(x, (0, pad)))
    s = torch.exp2(code.double() - 127).repeat_interleave(32, 1)
    lv = torch.tensor(LEVELS, dtype=torch.float64)
    n = torch.where(v.isnan(), torch.zeros_like(v), v / s)
    c = torch.searchsorted(lv, n.abs().contiguous()).to(torch.uint8)
    c = c + 8 * (torch.signbit(n) & ~v.isnan()).to(torch.uint8)
    two = c.reshape(rows, -1, 2)
    codes = (two[..., 0] + 16 * two[..., 1]).reshape(rows, -1, 128).transpose(0, 1).contiguous()
    return codes, code.reshape(rows, -1, 8).transpose(0, 1).contiguous()


def top_logits(x: torch.Tensor, k: int, temperature: float):
    """x [rows, C]: values, indices [rows, k], rest [rows]; NaN above all numbers, ties to the lowest index"""
    x = x.double()
    order = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
    nan_first = x.isnan().double()
    values, indices, rest = [], [], []
    for r in range(x.shape[0]):
        by = sorted(range(x.shape[1]), key=lambda c: (-float(nan_first[r, c]), -float(order[r, c]), c))
        indices.append(by[:k])
        values.append([float(x[r, c]) for c in by[:k]])
        others = x[r, by[k:]] / temperature
        rest.append(float(torch.logsumexp(others, 0)) if others.numel() else -math.inf)
    t = torch.tensor
    return t(values, dtype=torch.float64).view(-1, k), t(indices).view(-1, k), t(rest, dtype=torch.float64)


def distill(z, values, indices, rest, mask, temperature: float):
    """rows of logits z [rows, C]: (loss [rows], gradient [rows, C] of each row's loss, counts [rows]) in float64"""
    z, values, T = z.double(), values.double(), temperature
    rows, C = z.shape
    loss, grad, counts = torch.zeros(rows, dtype=torch.float64), torch.zeros_like(z), torch.zeros(rows, dtype=torch.bool)
    for r in range(rows):
        entries = [(int(c), float(v) / T) for c, v in zip(indices[r], values[r]) if int(c) >= 0]
        logs = [v for _, v in entries] + ([float(rest[r])] if rest is not None else [])
        if not logs or all(v == -math.inf for v in logs) or (mask is not None and not bool(mask[r])):
            continue
        counts[r] = True
        if any(c >= C for c, _ in entries):
            loss[r], grad[r] = math.nan, math.nan
            continue
        L = torch.logsumexp(torch.tensor(logs, dtype=torch.float64), 0)
        a = z[r] / T
        Z = torch.logsumexp(a, 0)
        nothing = bool(Z == -math.inf)
        q = torch.zeros_like(a) if nothing else torch.exp(a - Z)
        logq = torch.full_like(a, -math.inf) if nothing else a - Z
        listed = torch.zeros(C, dtype=torch.bool)
        share = torch.zeros(C, dtype=torch.float64)
        total = 0.0
        for c, v in entries:
            p = math.exp(v - L)
            listed[c] = True
            share[c] += p
            if p != 0.0:
                total += p * ((v - float(L)) - float(logq[c]))
        g = q - share
        qr = q[~listed].sum()
        lq_r = torch.logsumexp(logq[~listed], 0) if (~listed).any() else torch.tensor(-math.inf, dtype=torch.float64)
        pr = math.exp(float(rest[r]) - L) if rest is not None else 0.0
        if pr != 0.0:
            total += pr * ((float(rest[r]) - float(L)) - float(lq_r))
        if (~listed).any():
            rj = torch.exp(logq[~listed] - lq_r) if float(lq_r) > -math.inf or bool(lq_r.isnan()) else torch.zeros_like(q[~listed])
            g[~listed] = rj * (qr - pr)
        loss[r], grad[r] = T * T * total, T * g
    return loss, grad, counts
