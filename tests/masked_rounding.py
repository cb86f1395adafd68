"""Calls and error bounds of tests of rounding: pa_masked_attention and pa_shared_prefix_attention,
whose outputs stay within what 32-bit arithmetic with one rounding leaves, whatever the softcap.

Error bound against the definition in 64 bits, element by element, with A = sum_j p_j |v_j| / sum_j p_j of the
row and n keys (nothing in it grows with the softcap):
  u |o|             the output's one rounding, u = eps / 2 of its type
  2 s A             probabilities in two parts of that type, off by at most s = 2^-17 (bf16: half a step of eight
                    bits, twice) or 2^-20 (fp16: a step of ten bits, twice) of themselves, in the sum too
  4 d A             scores off by d move each probability by a factor within e^(+-d), and the sum;
                    d = (D + 24) 2^-24 M, M = the row's largest sum_d |q_d k_d| scale + |bias|: the fp32 sums of
                    D products and a few operations on the score, each within a step of what it yields.  A
                    softcap of at most 64 may add 2^-16 (a few steps of the cap itself), a larger one nothing
  (n + 64) 2^-23 A  fp32 sums over the keys, the exponential's and the scales' last bits
"""
from __future__ import annotations

import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import half_step, ranges

BF16, F16 = torch.bfloat16, torch.float16
PAIR = {BF16: 2.0 ** -17, F16: 2.0 ** -20}


def narrow64(st, *, softcap=0.0, window=-1, causal=1, slopes=None, prefix=None, starts=None):
    """(definition, bound) as above, for batches whose visible keys and values are finite."""
    H, KV, D, bs, dev = st["H"], st["KV"], st["D"], st["block"], st["q"].device
    u, s, t0 = half_step(st["dtype"]), PAIR[st["dtype"]], 0
    out = torch.zeros(sum(st["new"]), H, D, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    for b, n in enumerate(st["new"]):
        pos, lo, hi = (x.to(dev)[:, None] for x in ranges(st, b, window=window, causal=causal, prefix=prefix, starts=starts))
        p = torch.arange(st["total"][b], device=dev)
        at = st["bt"][b].long()[p // bs], p % bs
        seen = (p >= lo) & (p < hi)
        dist = (pos - p).abs().double()
        q = st["q"][t0:t0 + n].double().view(n, H, D)
        for h in range(H if n else 0):
            k, v = (st[x][at[0], at[1], h * KV // H].nan_to_num(0.0) for x in ("kd", "vd"))
            x, M = q[:, h] @ k.T * D ** -0.5, q[:, h].abs() @ k.abs().T * D ** -0.5
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x, M = x - float(slopes[h]) * dist, M + float(slopes[h]) * dist
            w = torch.softmax(x.masked_fill(~seen, -torch.inf), 1).nan_to_num(0.0)
            d = (D + 24) * 2.0 ** -24 * M.masked_fill(~seen, 0.0).amax(1, keepdim=True)
            if 0.0 < softcap <= 64.0:
                d = d + 2.0 ** -16
            o, A = w @ v, w @ v.abs()
            out[t0:t0 + n, h] = o
            tol[t0:t0 + n, h] = u * o.abs() + A * (2 * s + 4 * d + (p.numel() + 64) * 2.0 ** -23) * 1.01
        t0 += n
    tol = tol + torch.finfo(st["dtype"]).smallest_normal * half_step(st["dtype"]) * 2
    return out.view(-1, H * D), tol.view(-1, H * D)


def run(st, *, slopes=None, prefix=None, starts=None, window=-1, group_cum=None, shared=None, **kw):
    i32 = lambda x: None if x is None else torch.tensor(list(x), dtype=torch.int32, device="cuda")  # noqa: E731
    args = [st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"]]
    call = ep.masked_attention
    if shared is not None:
        call, args = ep.shared_prefix_attention, args + [i32(group_cum), i32(shared)]
    return call(*args, num_heads=st["H"], distance_slopes=None if slopes is None else torch.tensor(slopes, device="cuda"),
                prefix_lens=i32(prefix), document_starts=i32(starts), local_window_size=window,
                max_query_len=max(st["new"]), max_context_len=max(st["total"]), **kw)


def slopes_of(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


BATCHES = {"decode": ([1] * 6, [0, 1, 40, 63, 200, 900]), "few": ([2, 0, 5, 1], [9, 100, 31, 700]),
           "prompts": ([33, 1, 200, 65], [0, 0, 30, 333])}
