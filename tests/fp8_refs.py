"""Rows in 8-bit floating point, the products of such rows and the router of experts, in 64 bits on the CPU or the GPU: what the kernels are
held to.  Written from the definitions, without the framework's code."""
import math

import torch

RUN = 128


def held(x):
    """``(codes, exponents)`` of the rows of ``x``: the numbers the codes stand for (64 bits, NaN where x is not finite) and the scales' exponents."""
    x = x.double()
    K = x.shape[1]
    runs = -(-K // RUN)
    codes, exps = torch.empty_like(x), torch.empty((x.shape[0], runs), dtype=torch.long, device=x.device)
    for b in range(runs):
        v = x[:, b * RUN:(b + 1) * RUN]
        fine = torch.isfinite(v)
        top = torch.where(fine, v.abs(), 0.0).amax(1)
        e = torch.full_like(top, -127.0)
        for k in range(-127, 121):                       # the least exponent that reaches the largest magnitude
            e = torch.where(top > 448.0 * 2.0 ** k, k + 1.0, e)
        e = torch.where(top == 0, 0.0, e)
        scaled = torch.ldexp(torch.where(fine, v, 0.0), -e[:, None].long())
        _, p = torch.frexp(scaled)                        # |scaled| in [2**(p-1), 2**p): codes are 2**(p-4) apart, 2**-9 below 2**-6
        step = torch.ldexp(torch.ones_like(scaled), torch.clamp(p - 4, min=-9).long())
        codes[:, b * RUN:(b + 1) * RUN] = torch.where(fine, torch.round(scaled / step) * step, math.nan)
        exps[:, b] = e.long()
    return codes, exps


def values(x):
    """The numbers that the rows of ``x`` are held as."""
    codes, exps = held(x)
    return torch.ldexp(codes, exps.repeat_interleave(RUN, 1)[:, :x.shape[1]])


def read(codes, scales, columns, group_rows):
    """What the framework's codes and scales stand for (64 bits): ``(codes, exponents)`` of all rows."""
    rows = codes.shape[0]
    r = torch.arange(rows, device=codes.device)
    g, i = r // group_rows, r % group_rows
    runs = -(-columns // RUN)
    b = torch.arange(runs, device=codes.device)
    byte = scales[g[:, None], (i // 128)[:, None], (b // 4)[None], (i % 32 * 16 + i // 32 % 4 * 4)[:, None] + (b % 4)[None]]
    return codes[:, :columns].float().double(), byte.long() - 127


def numbers(codes, scales, columns, group_rows):
    c, e = read(codes, scales, columns, group_rows)
    return torch.ldexp(c, e.repeat_interleave(RUN, 1)[:, :columns])


def gelu_new(y):
    return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))


ACTS = {"none": lambda y: y, "relu": torch.relu, "gelu_new": gelu_new, "tanh": torch.tanh}


def unit(kind, g, u, w, limit):
    if kind == "bounded":
        g = torch.clamp(g, max=limit)
        u = torch.clamp(u, -limit, limit)
        return w * g * torch.sigmoid(1.702 * g) * (u + 1.0)
    return w * g * torch.sigmoid(w * g) * w * u


def route(logits, live, top, score="sigmoid", correction=None, groups=1, keep=1, two=False, renormalize=False, eps=0.0, factor=1.0, n_real=None):
    """Choices (lists of lists, -1: nobody, -2: no tensors) and weights, token by token."""
    E = logits.shape[1]
    n_real = E if n_real is None else n_real
    sel, weight = [], []
    for z, on in zip(logits.double().tolist(), live):
        if not on:
            sel.append([-1] * top)
            weight.append([0.0] * top)
            continue
        if score == "sigmoid":
            s = [v if v != v else 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in z]
        else:
            m = max(v for v in z if v == v)
            x = [math.exp(v - m) if v == v else math.nan for v in z]
            s = [v / sum(y for y in x if y == y) for v in x]
        by = [a + (float(correction[e]) if correction is not None else 0.0) for e, a in enumerate(s)]
        fair = [e for e in range(E) if by[e] == by[e] and by[e] > -math.inf]
        if keep < groups:
            per = E // groups
            judged = []
            for g in range(groups):
                c = sorted((by[e] for e in fair if e // per == g), reverse=True)
                if c:
                    judged.append((-(c[0] + c[1]) if two and len(c) > 1 else -c[0], g))
            kept = {g for _, g in sorted(judged)[:keep]}
            fair = [e for e in fair if e // per in kept]
        chosen = sorted(fair, key=lambda e: (-by[e], e))[:top]
        total = sum(s[e] for e in chosen) + eps if renormalize else 1.0
        weight.append([s[e] / total * factor for e in chosen] + [0.0] * (top - len(chosen)))
        sel.append([e if e < n_real else -2 for e in chosen] + [-1] * (top - len(chosen)))
    return sel, weight


def plan(sel, n_experts, tile_rows):
    """``(sorted slots, tiles)`` of the choices of all slots."""
    order, tiles = [], []
    for e in range(n_experts):
        mine = [i for i, x in enumerate(sel) if x == e]
        tiles += [(e, len(order) + a, min(tile_rows, len(mine) - a)) for a in range(0, len(mine), tile_rows)]
        order += mine
    return order, tiles
