"""Trees, definitions in 64 bits and error bounds of the tests of drafted trees, accounts and eviction.

Error bound of an attention output against the definition, element by element, with A = sum_j p_j |v_j| of the row and
n keys:
  u |o|             the output's one rounding, u = eps / 2 of its type
  2 s A             probabilities in two parts of a 16-bit type, off by at most s = 2^-17 (bf16) or 2^-20 (fp16) of
                    themselves, in the sum too; whole in fp32 where the kernel has no matrix products (s covers it)
  4 d A             scores off by d move each probability by a factor within e^(+-d), and the sum;
                    d = (D + 24) 2^-24 M, M = the row's largest sum_d |q_d k_d| scale: the fp32 sums of D products and
                    a few operations on the score.  A softcap of at most 64 may add 2^-16 (a few steps of the cap
                    itself), a larger one nothing
  (n + 64) 2^-23 A  fp32 sums over the keys, the exponential's and the scales' last bits
Bound of a key's weight: every probability p in it is off by p (4 d + (n + 64 + |c|) 2^-23), c = the constant of its
row's softmax in log2 units (rounded once, and the score beside it), and a sum of R positive terms in any order by
(R + 8) 2^-24 of itself.
"""
from __future__ import annotations

import math
import random

import torch

from masked_cases import half_step

PAIR = {torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -20, torch.float32: 2.0 ** -24}


def tree(rng, nodes, chain=0.4):
    """Parents of a tree, row 0 its root."""
    return [-1] + [r - 1 if rng.random() < chain else rng.randrange(r) for r in range(1, nodes)]


def lines(parents):
    """Ancestors (and itself) of every node [n, n], and its depth; a parent that is no earlier row makes a root."""
    n = len(parents)
    above, depth = torch.zeros(n, n, dtype=torch.bool), torch.zeros(n, dtype=torch.long)
    for r, p in enumerate(parents):
        if 0 <= p < r:
            above[r] = above[p]
            depth[r] = depth[p] + 1
        above[r, r] = True
    return above, depth


def tree_seen(parents, past, window=-1):
    above, depth = lines(parents)
    n = len(parents)
    seen = torch.cat([torch.ones(n, past, dtype=torch.bool), above], 1)
    if window > 0:
        place = torch.cat([torch.arange(past), past + depth])
        seen &= place > (past + depth)[:, None] - window
    return seen


def causal_seen(new, past, window=-1, causal=1):
    pos, j = torch.arange(new)[:, None] + past, torch.arange(past + new)
    seen = j <= pos if causal else torch.ones(new, past + new, dtype=torch.bool)
    return seen & (j > pos - window) if window > 0 else seen


def attention64(st, seen, *, scale=0.0, softcap=0.0, sink=None, observed=0):
    """(outputs, bounds) [tokens, H * D] under seen[b] [new, total], and per sequence the weights [KV, total] of the
    rows that count with their bounds."""
    H, KV, D, bs, dev = st["H"], st["KV"], st["D"], st["block"], st["q"].device
    scale, u, s = scale or D ** -0.5, half_step(st["dtype"]), PAIR[st["dtype"]]
    out = torch.zeros(sum(st["new"]), H, D, dtype=torch.float64, device=dev)
    tol, weights, t0 = torch.zeros_like(out), [], 0
    for b, n in enumerate(st["new"]):
        total = st["total"][b]
        w, wt = torch.zeros(2, KV, total, dtype=torch.float64, device=dev)
        weights.append((w, wt))
        if n == 0:
            continue
        vis = seen[b].to(dev)
        p = torch.arange(total, device=dev)
        at = st["bt"][b].long()[p // bs], p % bs
        q = st["q"][t0:t0 + n].double().view(n, H, D)
        dead = ~vis.any(0)
        counts = torch.arange(n, device=dev) >= (n - observed if observed else 0)
        for h in range(H):
            kh = h * KV // H
            k, v = (st[x][at[0], at[1], kh].masked_fill(dead[:, None], 0.0) for x in ("kd", "vd"))
            x, M = q[:, h] @ k.T * scale, q[:, h].abs() @ k.abs().T * abs(scale)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            x = x.masked_fill(~vis, -torch.inf)
            top = x.amax(1, keepdim=True)
            if sink is not None:
                top = torch.maximum(top, sink[h].double())
            e = torch.exp(x - top)
            den = e.sum(1, keepdim=True) + (0.0 if sink is None else torch.exp(sink[h].double() - top))
            pr = e / den
            d = (D + 24) * 2.0 ** -24 * M.masked_fill(~vis, 0.0).amax(1, keepdim=True)
            if 0.0 < softcap <= 64.0:
                d = d + 2.0 ** -16
            vz = v.nan_to_num(0.0, 0.0, 0.0)
            o, A = pr @ vz, pr @ vz.abs()
            bad = ~torch.isfinite(v)
            for j in bad.any(1).nonzero().flatten().tolist():
                o[vis[:, j]] += torch.where(bad[j], v[j], 0.0) * pr[vis[:, j], j:j + 1]
            out[t0:t0 + n, h] = o
            tol[t0:t0 + n, h] = u * o.abs() + A * (2 * s + 4 * d + (total + 64) * 2.0 ** -23) * 1.01
            const = (top + torch.log(den)).abs() / math.log(2.0)
            w[kh] += pr[counts].sum(0)
            wt[kh] += (pr * (4 * d + (total + 64 + const) * 2.0 ** -23))[counts].sum(0) * 1.01
        wt += w * (int(counts.sum()) * H // KV + 8) * 2.0 ** -24 + 1e-30
        t0 += n
    tol = tol + torch.finfo(st["dtype"]).smallest_normal * half_step(st["dtype"]) * 2
    return out.view(-1, H * D), tol.view(-1, H * D), weights


def accepted(parents, tokens, targets):
    """The accepted path of one tree."""
    path = [0] if parents else []
    while path:
        child = next((r for r in range(path[-1] + 1, len(parents))
                      if parents[r] == path[-1] and tokens[r] == targets[path[-1]]), None)
        if child is None:
            break
        path.append(child)
    return path


def staying(weights, budget, sinks, recent):
    """Positions of one head's keys that stay, by their weights."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    rank = lambda j: (0, 0.0, j) if math.isnan(weights[j]) else (1, -weights[j], j)  # noqa: E731
    heavy = sorted(range(sinks, n - recent), key=rank)[:budget - sinks - recent]
    return [*range(sinks), *sorted(heavy), *range(n - recent, n)]


def trees(st, chain=0.4, seed=0):
    rng = random.Random(seed)
    return [tree(rng, n, chain) if n else [] for n in st["new"]]


def packed(parents, device="cuda", pad=0):
    return torch.tensor(sum(parents, []) + [-1] * pad, dtype=torch.int32, device=device)
