"""Batches, definitions in 64 bits and error bounds of masked, shared-prefix and multi-axis tests.

Error bound of an attention output against the definition, element by element.  With A = sum_j p_j
|v_j| / sum_j p_j of its row, u = eps / 2 of the output type and n keys:
  u |o|            the output's rounding
  u A              the probabilities' rounding to the same type for the second product
  4 d A            scores off by d each move every probability by a factor within e^(+-d), the sum too;
                   d = (D + 16) 2^-24 M, M = the row's largest sum_d |q_d k_d| scale + |bias|: the fp32
                   sums of D products and a few operations on the score (softcap: at most 2^-21 cap more)
  (n + 64) 2^-23 A fp32 sums over the keys, the exponential's and the scales' last bits
"""
from __future__ import annotations

import numpy as np
import torch


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make_batch(new, past, *, H, KV, D, block, dtype, seed=0, shared=None, group_cum=None, spare=2,
               pad_tokens=0, device="cuda", cache_dtype=None, scales="PER_TENSOR", std=1.0):
    """Paged batch on `device`.  Pages the sequences do not use, and the rows behind a sequence's last
    key in its last page, are NaN (codes: random).  group_cum / shared: a group's sequences name the
    same pages for their shared keys (whole pages)."""
    g = torch.Generator().manual_seed(seed)
    total = [p + n for p, n in zip(past, new)]
    max_blocks = max(-(-t // block) for t in total) + spare
    used, table = 0, []
    group_cum = list(group_cum or [])
    for b, t in enumerate(total):
        need = -(-t // block)
        row = []
        gi = next((i for i in range(len(group_cum) - 1) if group_cum[i] <= b < group_cum[i + 1]), None)
        if gi is not None and b > group_cum[gi]:
            row = table[group_cum[gi]][:shared[gi] // block]
        row = row + list(range(used, used + need - len(row)))
        used = max([used] + [x + 1 for x in row])
        table.append(row)
    nb = used + 3
    order = torch.randperm(nb, generator=g)
    bt = torch.full((len(new), max_blocks), -1, dtype=torch.int64)
    for b, row in enumerate(table):
        if row:
            bt[b, :len(row)] = order[torch.tensor(row)]
    T = sum(new)
    rnd = lambda *s: torch.randn(*s, generator=g) * std  # noqa: E731
    st = dict(H=H, KV=KV, D=D, block=block, dtype=dtype, new=new, past=past, total=total,
              q=rnd(T + pad_tokens, H * D).to(dtype).to(device),
              cum=torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=device),
              past_t=torch.tensor(past, dtype=torch.int32, device=device),
              bt=bt.to(torch.int32).to(device), k_scale=None, v_scale=None, quant="NONE")
    if cache_dtype is None:
        kc, vc = torch.full((nb, block, KV, D), float("nan")), torch.full((nb, block, KV, D), float("nan"))
        for b, t in enumerate(total):
            p = torch.arange(t)
            kc[bt[b, p // block], p % block] = rnd(t, KV, D)
            vc[bt[b, p // block], p % block] = rnd(t, KV, D)
        st["kc"], st["vc"] = kc.to(dtype).to(device), vc.to(dtype).to(device)
        st["kd"], st["vd"] = st["kc"].double(), st["vc"].double()
    elif cache_dtype == torch.float8_e4m3fn:
        for s in "kv":
            codes = rnd(nb, block, KV, D).to(torch.float8_e4m3fn)
            sc = torch.rand(nb, KV, generator=g) + 0.5
            st[s + "c"], st[s + "_scale"] = codes.to(device), sc.to(device)
            st[s + "d"] = st[s + "c"].double() * st[s + "_scale"].double()[:, None, :, None]
    else:
        st["quant"] = scales
        for s in "kv":
            sc = (torch.rand(KV, D, generator=g) if scales == "PER_CHANNEL" else torch.rand(1, generator=g)) * 0.2 + 0.1
            st[s + "_scale"] = sc.to(device)
            if cache_dtype == torch.int8:
                codes = torch.randint(-20, 21, (nb, block, KV, D), generator=g, dtype=torch.int8)
                vals = codes.double()
            else:
                codes = torch.randint(0, 256, (nb, block, KV, (D + 1) // 2), generator=g).to(torch.uint8)
                vals = torch.stack([(codes & 15).double() - 8, (codes >> 4).double() - 8], -1).flatten(-2)[..., :D]
            st[s + "c"] = codes.to(device)
            st[s + "d"] = vals.to(device) * st[s + "_scale"].double()
    return st


def ranges(st, b, *, window=-1, causal=1, prefix=None, starts=None):
    """[first, end) of the keys that the rows of sequence b see."""
    t0 = sum(st["new"][:b])
    pos = torch.arange(st["new"][b]) + st["past"][b]
    hi = pos + 1 if causal else torch.full_like(pos, st["total"][b])
    if prefix is not None and causal:
        hi = torch.clamp(hi, min=int(prefix[b]))
    hi = torch.clamp(hi, max=st["total"][b])
    lo = torch.zeros_like(pos)
    if window > 0:
        lo = torch.maximum(lo, pos - window + 1)
    if starts is not None:
        lo = torch.maximum(lo, torch.as_tensor(starts)[t0:t0 + st["new"][b]].long())
    return pos, lo, hi


def attention64(st, *, scale=0.0, softcap=0.0, window=-1, causal=1, sink=None, slopes=None,
                prefix=None, starts=None):
    """(definition, error bound) of the packed output rows [sum(new), H * D] in 64 bits."""
    H, KV, D, bs, dev = st["H"], st["KV"], st["D"], st["block"], st["q"].device
    scale = scale or D ** -0.5
    T = sum(st["new"])
    out = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    u, t0 = half_step(st["dtype"]), 0
    for b, n in enumerate(st["new"]):
        pos, lo, hi = (x.to(dev)[:, None] for x in ranges(st, b, window=window, causal=causal, prefix=prefix, starts=starts))
        p = torch.arange(st["total"][b], device=dev)
        at = st["bt"][b].long()[p // bs], p % bs
        seen = (p >= lo) & (p < hi)
        dist = (pos - p).abs().double()
        q = st["q"][t0:t0 + n].double().view(n, H, D)
        for kh in range(KV if n else 0):
            k, v = st["kd"][at[0], at[1], kh], st["vd"][at[0], at[1], kh]
            # keys that no row sees take no part, whatever they hold
            dead = ~seen.any(0)
            k, v = k.masked_fill(dead[:, None], 0.0), v.masked_fill(dead[:, None], 0.0)
            for h in range(kh * H // KV, (kh + 1) * H // KV):
                x = q[:, h] @ k.T * scale
                M = (q[:, h].abs() @ k.abs().T * abs(scale))
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                    M = M + 8 * softcap  # 2^-21 cap = 8 cap 2^-24
                if slopes is not None:
                    x = x - float(slopes[h]) * dist
                    M = M + abs(float(slopes[h])) * dist
                x = x.masked_fill(~seen, -torch.inf)
                M = M.masked_fill(~seen, 0.0).nan_to_num(0.0).amax(1, keepdim=True) if st["total"][b] else 0.0
                top = x.amax(1, keepdim=True)
                if sink is not None:
                    top = torch.maximum(top, sink[h].double().expand_as(top))
                top = torch.where(top == -torch.inf, 0.0, top)
                e = torch.exp(x - top)
                den = e.sum(1, keepdim=True)
                if sink is not None:
                    den = den + torch.exp(sink[h].double() - top)
                w = torch.where(den == 0, 0.0, e / den)
                # weights of exactly zero take no part, whatever the value
                vz = v.nan_to_num(0.0, 0.0, 0.0)
                o = w @ vz
                bad = ~torch.isfinite(v)
                if bad.any():
                    for j in bad.any(1).nonzero().flatten().tolist():
                        rows = seen[:, j]
                        o[rows] = o[rows] + torch.where(bad[j], v[j], 0.0) * w[rows, j:j + 1]
                A = w @ vz.abs()
                d = (D + 16) * 2.0 ** -24 * M
                out[t0:t0 + n, h] = o
                tol[t0:t0 + n, h] = u * o.abs() + A * (u + 4 * d + (p.numel() + 64) * 2.0 ** -23) * 1.01 + 1e-30
        t0 += n
    # values below the smallest normal of the output type round to its steps
    tol = tol + torch.finfo(st["dtype"]).smallest_normal * half_step(st["dtype"]) * 2
    return out.view(T, H * D), tol.view(T, H * D)


def check(got, want, tol):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN places differ"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), "infinities differ"
    over = ((got - want).abs() / tol)[fin]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"error is {worst:.3g} of its bound"
    return worst
