"""Operators beside paged attention that are measured: masks and distance biases over the pages, a
prefix shared by a group of sequences, and rotary positions of several axes on the way into the pages.

  masked   attention over a paged cache whose rows see the keys of their document, of their prefix or
           of their past, with a bias that falls with the distance (per-head slopes)
  shared   attention of groups of sequences that hold the same prefix in the same pages
  append   RMSNorm (optional) and rotary positions of three axes (time, height, width) on queries and
           keys, and the new keys and values into their pages

Where `own` is false, run() computes them from elementary torch operations in 32 bits on padded
batches; where it is true it makes the library's calls.  A case holds sizes and options only.
`layout` seeds the ragged lengths (so work() can count them); the seed of prepare() makes the tensors
and the order of the pages.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEVICE = "cuda"


# ---------------------------------------------------------------------------------------- cases

def _masked(name=None, **kw):
    # seqs sequences of new_min..new_max tokens after past_min..past_max cached ones; slopes: the
    # distance bias; prefix_min..prefix_max leading keys that every row sees (0: causal alone);
    # doc_min..doc_max tokens to a document (0: one document).
    c = dict(op="masked", dtype="bf16", heads=32, kv=8, head=128, block=16, seqs=1, new_min=1,
             new_max=1, past_min=0, past_max=0, slopes=False, prefix_min=0, prefix_max=0, doc_min=0,
             doc_max=0, window=-1, softcap=0.0, sink=False, layout=1)
    c.update(kw)
    return c if name is None else dict(name=name, **c)


def _shared(name=None, **kw):
    # groups of seqs sequences each: shared_min..shared_max keys (their whole pages) held once for the
    # group, then past_min..past_max cached keys and new_min..new_max new tokens of each one's own.
    c = dict(op="shared", dtype="bf16", heads=32, kv=8, head=128, block=16, groups=1, seqs=8,
             new_min=1, new_max=1, shared_min=0, shared_max=0, past_min=0, past_max=0, softcap=0.0,
             sink=False, layout=1)
    c.update(kw)
    return c if name is None else dict(name=name, **c)


def _append(name=None, **kw):
    # sections: frequencies of the time, height and width axis; interleaved_axes: the axes take
    # turns over the frequencies instead of one section after the other.
    c = dict(op="append", dtype="bf16", heads=32, kv=8, head=128, block=16, seqs=1, new_min=1,
             new_max=1, past_min=0, past_max=0, s0=16, s1=24, s2=24, interleaved_axes=False,
             norm=False, theta=1000000.0, layout=1)
    c.update(kw)
    return c if name is None else dict(name=name, **c)


def listed():
    return [
        # The next token of one user's chat with a picture in it: launch latency is all of it.
        _append("append_one_token", past_min=700, past_max=700),
        # A loaded server's step, QK-normalised heads with a short rotated part.
        _append("append_step_64", dtype="f16", heads=24, kv=4, head=256, block=256, seqs=64,
                past_min=100, past_max=6000, s0=8, s1=12, s2=12, interleaved_axes=True, norm=True),
        # Prompts with images and video frames: thousands of tokens, every row rotated.
        _append("append_prompts", seqs=6, new_min=301, new_max=2500, interleaved_axes=True,
                norm=True, layout=4),
        # One token of a small model with distance biases after a short text.
        _masked("slopes_one_token", dtype="f16", heads=8, kv=2, head=64, past_min=128,
                past_max=128, slopes=True),
        # A loaded server's step of a model with distance biases.
        _masked("slopes_step_64", seqs=64, past_min=511, past_max=8190, slopes=True, layout=3),
        # Many short documents packed into each row of a batch that is scored or embedded.
        _masked("documents_packed", dtype="f16", heads=64, kv=8, head=64, seqs=4, new_min=1001,
                new_max=2500, doc_min=20, doc_max=700, layout=5),
        # Image tokens and the question seen from both sides, the answer causal; one kv head.
        _masked("prefix_prompts", heads=8, kv=1, head=256, block=32, seqs=8, new_min=290,
                new_max=1100, prefix_min=256, prefix_max=900, softcap=50.0, layout=6),
        # A long text's first pass with distance biases.
        _masked("slopes_prompt_8k", new_min=8191, new_max=8191, slopes=True),
        # A few samples of one short question.
        _shared("samples_of_300", seqs=4, shared_min=300, shared_max=300, past_min=1, past_max=40),
        # Many samples of one long prompt, as in best-of-n search and rollouts.
        _shared("samples_64_of_8k", seqs=64, shared_min=8190, shared_max=8190, past_min=1,
                past_max=500, layout=3),
        # Three system prompts, each with the requests that begin with it; sinks, head 64.
        _shared("system_prompts", dtype="f16", heads=64, kv=8, head=64, block=32, groups=3, seqs=16,
                shared_min=700, shared_max=5000, past_min=10, past_max=900, sink=True, layout=4),
        # Drafted tokens of several continuations checked at once against a long document.
        _shared("drafts_over_document", heads=28, kv=4, seqs=12, new_min=3, new_max=9,
                shared_min=30001, shared_max=30001, past_min=0, past_max=200, layout=5),
    ]


HEADS = ((32, 8, 128), (28, 4, 128), (8, 2, 64), (64, 8, 64), (24, 8, 96), (8, 1, 256), (24, 4, 256))


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST_BYTES, MOST_FLOPS, MOST_SCORES = 1.2e9, 5.0e11, 2.2e9


def _scores(case):
    """Scores of the padded plain form."""
    s = _lengths(case)
    if case["op"] == "append":
        return 0
    return (len(s["new"]) * max(s["new"]) * case["heads"] *
            max(p + n for p, n in zip(s["past"], s["new"])))


def _draw_once(rng):
    op = rng.choices(("masked", "shared", "append"), (0.5, 0.3, 0.2))[0]
    heads, kv, head = rng.choice(HEADS)
    base = dict(dtype=rng.choice(("bf16", "f16")), heads=heads, kv=kv, head=head,
                block=rng.choice((16, 16, 32, 64, 256)), layout=rng.randrange(1 << 20))
    if op == "append":
        half = rng.choice((head // 2, head // 4)) // 8 * 8
        s1 = rng.randrange(1, half // 3 + 1)
        s2 = rng.randrange(1, half // 3 + 1)
        most = _logint(rng, 1, 3000)
        return _append(**base, seqs=_logint(rng, 1, 64), new_min=max(1, most // 3), new_max=most,
                       past_max=_logint(rng, 1, 4000), s0=half - s1 - s2, s1=s1, s2=s2,
                       interleaved_axes=rng.random() < 0.5,
                       norm=head in (64, 128, 256) and rng.random() < 0.5)
    if op == "shared":
        shared = _logint(rng, 64, 32000)
        most = 1 if rng.random() < 0.6 else _logint(rng, 2, 40)
        return _shared(**base, groups=rng.choice((1, 1, 2, 5)), seqs=_logint(rng, 2, 64),
                       new_min=max(1, most // 2), new_max=most, shared_min=max(1, shared // 2),
                       shared_max=shared, past_max=_logint(rng, 1, 2000),
                       softcap=rng.choice((0.0, 0.0, 0.0, 30.0)), sink=rng.random() < 0.25)
    forms = dict(slopes=rng.random() < 0.5, softcap=rng.choice((0.0, 0.0, 0.0, 50.0)),
                 sink=rng.random() < 0.2, window=rng.choice((-1, -1, -1, _logint(rng, 16, 2000))))
    if rng.random() < 0.45:  # a step of a token or a few
        longest = _logint(rng, 20, 16000)
        return _masked(**base, **forms, seqs=_logint(rng, 1, 64), new_max=rng.choice((1, 1, 1, 3)),
                       past_min=longest // 4, past_max=longest,
                       prefix_max=rng.choice((0, longest // 2)),
                       doc_min=5, doc_max=rng.choice((0, longest)))
    longest = _logint(rng, 17, 6000)
    docs = rng.random() < 0.4
    pre = 0 if docs and rng.random() < 0.7 else rng.choice((0, longest // 2))
    return _masked(**base, **forms, seqs=_logint(rng, 1, 12), new_min=max(1, longest // 3),
                   new_max=longest, past_max=rng.choice((0, _logint(rng, 1, 4000))),
                   prefix_min=pre // 2, prefix_max=pre, doc_min=5,
                   doc_max=_logint(rng, 10, longest) if docs else 0)


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and _scores(case) <= MOST_SCORES:
            return case


# -------------------------------------------------------------------------------------- lengths

def _between(rng, lo, hi):
    return rng.randint(min(lo, hi), hi)


def _lengths(case):
    """New tokens, cached keys (a shared prefix among them), prefixes and document starts."""
    rng = random.Random(case["layout"])
    out = dict(new=[], past=[], prefix=[], starts=[], shared=[], group_cum=[0])
    for _ in range(case.get("groups", 1)):
        shared = _between(rng, case["shared_min"], case["shared_max"]) if case["op"] == "shared" else 0
        shared -= shared % case["block"]  # whole pages are what sequences hold together
        out["shared"].append(shared)
        for _ in range(case["seqs"]):
            new = _between(rng, case["new_min"], case["new_max"])
            past = shared + _between(rng, case["past_min"], case["past_max"])
            out["new"].append(new)
            out["past"].append(past)
            if case["op"] == "masked":
                out["prefix"].append(min(_between(rng, case["prefix_min"], case["prefix_max"]),
                                         past + new))
                start, starts = 0, []
                while len(starts) < past + new:
                    n = (_between(rng, case["doc_min"], case["doc_max"]) if case["doc_max"]
                         else past + new)
                    starts += [start] * n
                    start += n
                out["starts"].append(starts[past:past + new])
        out["group_cum"].append(len(out["new"]))
    return out


def _ranges(case, s):
    """[first, end) of the keys that every packed token sees."""
    lo, hi = [], []
    for b, (new, past) in enumerate(zip(s["new"], s["past"])):
        for i in range(new):
            pos = past + i
            first, end = 0, pos + 1
            if case["op"] == "masked":
                first, end = s["starts"][b][i], max(end, s["prefix"][b])
                if case["window"] > 0:
                    first = max(first, pos - case["window"] + 1)
            lo.append(first)
            hi.append(min(end, past + new))
    return lo, hi


def work(case):
    s = _lengths(case)
    tokens = sum(s["new"])
    H, KV, D = case["heads"], case["kv"], case["head"]
    if case["op"] == "append":
        half = case["s0"] + case["s1"] + case["s2"]
        moved = 2 * (H + 2 * KV) * D * 2  # rows in, rows out
        return {"bytes": float(tokens * (moved + 3 * 8 + 2 * half * 2)),
                "flops": float(tokens * (H + KV) * (6 * half + (4 * D if case["norm"] else 0)))}
    lo, hi = _ranges(case, s)
    pairs = sum(max(0, h - l) for l, h in zip(lo, hi))
    # keys that some row sees, each once; a group's prefix once for the group
    keys, t = sum(s["shared"]), 0
    for b, new in enumerate(s["new"]):
        seen_lo, seen_hi = min(lo[t:t + new]), max(hi[t:t + new])
        if case["op"] == "shared":
            seen_lo = s["shared"][b // case["seqs"]]
        keys += max(0, seen_hi - seen_lo)
        t += new
    return {"bytes": float(keys * KV * D * 2 * 2 + 2 * tokens * H * D * 2),
            "flops": float(4 * pairs * H * D)}


# ------------------------------------------------------------------------------------ preparing

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    s = _lengths(case)
    H, KV, D, bs = case["heads"], case["kv"], case["head"], case["block"]
    dt = DTYPES[case["dtype"]]
    T, B = sum(s["new"]), len(s["new"])
    total = [p + n for p, n in zip(s["past"], s["new"])]
    max_blocks = max(-(-t // bs) for t in total) + 1

    def normal(*shape, std=1.0):
        x = torch.empty(shape, dtype=dt, device=DEVICE)
        return x.normal_(0.0, std, generator=g)

    # Pages: a group's sequences hold their shared keys in the same pages.
    seqs = case["seqs"]
    need, table = 0, []
    for gi, shared in enumerate(s["shared"]):
        common = shared // bs
        first = list(range(need, need + common))
        need += common
        for b in range(gi * seqs, (gi + 1) * seqs):
            mine = -(-total[b] // bs) - common
            table.append(first + list(range(need, need + mine)))
            need += mine
    num_blocks = need + 3
    order = torch.randperm(num_blocks, device=DEVICE, generator=g).to(torch.int32)
    index = torch.tensor([row + [0] * (max_blocks - len(row)) for row in table], device=DEVICE)
    st = dict(case=case, tokens=T,
              key_cache=normal(num_blocks, bs, KV, D), value_cache=normal(num_blocks, bs, KV, D),
              cum=_i32([0] + torch.tensor(s["new"]).cumsum(0).tolist()), past=_i32(s["past"]),
              block_table=order[index].contiguous(), max_query_len=max(s["new"]),
              max_context_len=max(total), query=normal(T, H * D))
    # where the plain form finds the packed tokens in a padded batch
    nmax = max(s["new"])
    inside = torch.arange(nmax, device=DEVICE)[None, :] < _i32(s["new"])[:, None]
    st["rows"] = inside.flatten().nonzero().flatten()
    if case["op"] == "append":
        half = case["s0"] + case["s1"] + case["s2"]
        st["key"], st["value"] = normal(T, KV * D), normal(T, KV * D)
        # time, height and width: a patch grid after each sequence's text
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(s["past"], s["new"])])
        side = 1 + int(math.isqrt(max(s["new"])))
        st["positions"] = torch.stack([pos, pos % side + pos // 7, pos // side + pos // 5]).to(DEVICE)
        angle = (torch.arange(max(total) * 2 + 8, dtype=torch.float64, device=DEVICE)[:, None] *
                 case["theta"] ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half))
        st["cos"], st["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        st["q_norm"] = st["k_norm"] = None
        if case["norm"]:
            st["q_norm"], st["k_norm"] = 1 + normal(D, std=0.1), 1 + normal(D, std=0.1)
        st["q_out"] = torch.empty_like(st["query"])
        return st
    # scores of a trained model spread wider than one
    st["query"] *= 1.5
    st["output"] = torch.empty_like(st["query"])
    st["sink"] = normal(H) if case["sink"] else None
    if case["op"] == "shared":
        st["group_cum"], st["shared"] = _i32(s["group_cum"]), _i32(s["shared"])
        st["max_shared"] = max(s["shared"])
        st["max_own"] = max(t - s["shared"][b // seqs] for b, t in enumerate(total))
        return st
    st["slopes"] = st["prefix"] = st["starts"] = None
    if case["slopes"]:  # 2^(-8 (h + 1) / heads)
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEVICE) / H).float()
    if case["prefix_max"]:
        st["prefix"] = _i32(s["prefix"])
    if case["doc_max"]:
        st["starts"] = _i32(sum(s["starts"], []))
    return st


# ------------------------------------------------------------------------------------ plain form

def _axis_of(case, half):
    """Axis of every frequency."""
    i = torch.arange(half, device=DEVICE)
    if not case["interleaved_axes"]:
        return (i >= case["s0"]).long() + (i >= case["s0"] + case["s1"]).long()
    s = torch.tensor([0, case["s1"], case["s2"]], device=DEVICE)
    a = i % 3
    return torch.where(i < 3 * s[a], a, 0)


def _token_places(st):
    """Sequence and position of every packed token."""
    cum, t = st["cum"].long(), torch.arange(st["tokens"], device=DEVICE)
    b = torch.searchsorted(cum, t, right=True) - 1
    return b, st["past"].long()[b] + t - cum[b]


def _plain_append(st):
    case = st["case"]
    H, KV, D, bs = case["heads"], case["kv"], case["head"], case["block"]
    dt, T = st["query"].dtype, st["tokens"]
    half = st["cos"].shape[1]
    at = st["positions"][_axis_of(case, half)].T  # [T, half]
    f = torch.arange(half, device=DEVICE)
    cos, sin = st["cos"][at, f].float()[:, None], st["sin"][at, f].float()[:, None]

    def turn(rows, heads, weight):
        x = rows.view(T, heads, D).float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(dt)

    b, pos = _token_places(st)
    block, off = st["block_table"].long()[b, pos // bs], pos % bs
    st["key_cache"][block, off] = turn(st["key"], KV, st["k_norm"])
    st["value_cache"][block, off] = st["value"].view(T, KV, D)
    st["q_out"].copy_(turn(st["query"], H, st["q_norm"]).view(T, H * D))
    return st["q_out"], st["key_cache"], st["value_cache"]


def _pages(st, table, first, keys):
    """Keys and values [N, KV, keys, D] of the positions first[n] + 0 .. keys - 1, in 32 bits."""
    bs = st["case"]["block"]
    pos = (first[:, None] + torch.arange(keys, device=DEVICE)).clamp(max=table.shape[1] * bs - 1)
    block, off = table.long().gather(1, pos // bs), pos % bs
    return (st["key_cache"][block, off].float().transpose(1, 2),
            st["value_cache"][block, off].float().transpose(1, 2))


def _score(case, q, k):
    x = q @ k.transpose(-1, -2) / math.sqrt(case["head"])
    return case["softcap"] * torch.tanh(x / case["softcap"]) if case["softcap"] else x


def _padded_queries(st, n, rows, per):
    """Queries [n, KV, per * g, D] of packed tokens that stand at `rows` of n x per places."""
    H, KV, D = st["case"]["heads"], st["case"]["kv"], st["case"]["head"]
    q = torch.zeros(n * per, H * D, device=DEVICE)
    q[rows] = st["query"].float()
    return q.view(n, per, KV, H // KV, D).transpose(1, 2).reshape(n, KV, per * (H // KV), D)


def _packed(st, x, rows, n, per):
    H, KV, D = st["case"]["heads"], st["case"]["kv"], st["case"]["head"]
    width = x.shape[-1]
    x = x.view(n, KV, per, H // KV, width).transpose(1, 2).reshape(n * per, H, width)
    return x[rows]


def _softmax_parts(x, v):
    """Largest score, sum of the weights and weighted values; rows of no key weigh nothing."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    return torch.cat([m, p.sum(-1, keepdim=True), p @ v], -1)


def _joined(st, parts):
    """Rows of several key ranges (and the sink) joined: [T, H, 2 + D] each."""
    m = torch.stack([p[..., 0] for p in parts])
    if st["sink"] is not None:
        sink = st["sink"].float().expand(m.shape[1:])
        m = torch.cat([m, sink[None]])
    top = m.amax(0)
    w = [torch.exp(p[..., 0] - top) for p in parts]
    den = sum(p[..., 1] * f for p, f in zip(parts, w))
    if st["sink"] is not None:
        den = den + torch.exp(sink - top)
    out = sum(p[..., 2:] * f[..., None] for p, f in zip(parts, w))
    out = torch.where(den[..., None] > 0, out / den[..., None], 0.0)
    st["output"].copy_(out.reshape(st["output"].shape))
    return st["output"]


def _plain_masked(st):
    case = st["case"]
    H, KV, g = case["heads"], case["kv"], case["heads"] // case["kv"]
    B, per, keys = len(st["past"]), st["max_query_len"], st["max_context_len"]
    past, new = st["past"].long(), st["cum"].long().diff()
    zero = torch.zeros_like(past)
    k, v = _pages(st, st["block_table"], zero, keys)
    j = torch.arange(keys, device=DEVICE)
    pos = past[:, None] + torch.arange(per, device=DEVICE)  # [B, per]
    end = pos + 1
    if st["prefix"] is not None:
        end = torch.maximum(end, st["prefix"].long()[:, None])
    end = torch.minimum(end, (past + new)[:, None])
    first = torch.zeros_like(pos)
    if st["starts"] is not None:
        first = first.flatten().index_put((st["rows"],), st["starts"].long()).view(B, per)
    if case["window"] > 0:
        first = torch.maximum(first, pos - case["window"] + 1)
    seen = (j >= first[..., None]) & (j < end[..., None])  # [B, per, keys]
    x = _score(case, _padded_queries(st, B, st["rows"], per), k).view(B, KV, per, g, keys)
    if st["slopes"] is not None:
        far = (pos[..., None] - j).abs().float()[:, None, :, None]
        x = x - st["slopes"].view(1, KV, 1, g, 1) * far
    x = torch.where(seen[:, None, :, None], x, -math.inf).view(B, KV, per * g, keys)
    v = torch.where((j < (past + new)[:, None])[:, None, :, None], v, 0.0)
    return _joined(st, [_packed(st, _softmax_parts(x, v), st["rows"], B, per)])


def _plain_shared(st):
    """The prefix once for every group's rows, the own keys for every sequence, and their join."""
    case = st["case"]
    g, seqs, G = case["heads"] // case["kv"], case["seqs"], case["groups"]
    B, per = len(st["past"]), st["max_query_len"]
    past, new, shared = st["past"].long(), st["cum"].long().diff(), st["shared"].long()
    mine = shared.repeat_interleave(seqs)  # first own key of every sequence
    # prefix: a group's rows are its sequences' padded rows, one after another
    keys = max(1, st["max_shared"])
    k, v = _pages(st, st["block_table"][::seqs], torch.zeros_like(shared), keys)
    j = torch.arange(keys, device=DEVICE)
    seen = j < shared[:, None]
    x = _score(case, _padded_queries(st, G, st["rows"], seqs * per), k)
    x = torch.where(seen[:, None, None], x, -math.inf)
    prefix = _packed(st, _softmax_parts(x, v), st["rows"], G, seqs * per)
    # own keys
    keys = st["max_own"]
    k, v = _pages(st, st["block_table"], mine, keys)
    j = torch.arange(keys, device=DEVICE)
    pos = past[:, None] + torch.arange(per, device=DEVICE) - mine[:, None]
    seen = (j <= pos[..., None]) & (j < (past + new - mine)[:, None, None])
    x = _score(case, _padded_queries(st, B, st["rows"], per), k).view(B, -1, per, g, keys)
    x = torch.where(seen[:, None, :, None], x, -math.inf).view(B, -1, per * g, keys)
    v = torch.where((j < (past + new - mine)[:, None])[:, None, :, None], v, 0.0)
    own_keys = _packed(st, _softmax_parts(x, v), st["rows"], B, per)
    return _joined(st, [prefix, own_keys])


# ------------------------------------------------------------------------------------------ runs

def _library():
    place = str(Path(__file__).resolve().parent.parent / "onnxruntime-ep-mlx_amd")
    if place not in sys.path:
        sys.path.insert(0, place)
    import onnxruntime_ep_mlx_amd as ep
    return ep


def _own(st):
    ep, case = _library(), st["case"]
    if case["op"] == "append":
        q = ep.multi_axis_rotary_append(
            st["query"], st["key"], st["value"], st["key_cache"], st["value_cache"], st["cum"],
            st["past"], st["block_table"], st["positions"], st["cos"], st["sin"],
            num_heads=case["heads"], axis_sections=(case["s0"], case["s1"], case["s2"]),
            axes_interleaved=case["interleaved_axes"], q_norm_weight=st["q_norm"],
            k_norm_weight=st["k_norm"], qk_norm_epsilon=1e-6, slots_distinct=True,
            q_out=st["q_out"])
        return q, st["key_cache"], st["value_cache"]
    args = (st["query"], st["key_cache"], st["value_cache"], st["cum"], st["past"], st["block_table"])
    kw = dict(num_heads=case["heads"], softcap=case["softcap"], head_sink=st["sink"],
              max_query_len=st["max_query_len"], max_context_len=st["max_context_len"],
              out=st["output"])
    if case["op"] == "shared":
        return ep.shared_prefix_attention(*args, st["group_cum"], st["shared"],
                                          max_prefix_len=st["max_shared"], **kw)
    return ep.masked_attention(*args, distance_slopes=st["slopes"], prefix_lens=st["prefix"],
                               document_starts=st["starts"], local_window_size=case["window"], **kw)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return (_plain_append if op == "append" else _plain_shared if op == "shared" else _plain_masked)(state)


# ----------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """From the definitions, in 64 bits, one sequence at a time."""
    st = prepare(case, seed)
    s = _lengths(case)
    H, KV, D, bs = case["heads"], case["kv"], case["head"], case["block"]
    kc, vc = st["key_cache"].double(), st["value_cache"].double()
    flat_k, flat_v = kc.view(-1, KV, D), vc.view(-1, KV, D)

    def slots(b, lo, hi):
        p = torch.arange(lo, hi, device=DEVICE)
        return st["block_table"][b].long()[p // bs] * bs + p % bs

    starts_at = [0]
    for n in s["new"]:
        starts_at.append(starts_at[-1] + n)
    if case["op"] == "append":
        half = case["s0"] + case["s1"] + case["s2"]
        sizes = (case["s0"], case["s1"], case["s2"])
        axes = [(0 if i < sizes[0] else 1 if i < sizes[0] + sizes[1] else 2) for i in range(half)]
        if case["interleaved_axes"]:
            axes = [i % 3 if i % 3 and i < 3 * sizes[i % 3] else 0 for i in range(half)]
        ids = torch.stack([st["positions"][a] for a in axes], 1)
        c = torch.stack([st["cos"][ids[:, i], i] for i in range(half)], 1).double()
        z = torch.complex(c, torch.stack([st["sin"][ids[:, i], i] for i in range(half)], 1).double())

        def turned(x, n, w):
            x = x.double().view(-1, n, D)
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
            y = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z[:, None]
            return torch.cat([y.real, y.imag, x[..., 2 * half:]], -1)

        keys = turned(st["key"], KV, st["k_norm"])
        for b, (new, past) in enumerate(zip(s["new"], s["past"])):
            at, rows = slots(b, past, past + new), slice(starts_at[b], starts_at[b + 1])
            flat_k[at] = keys[rows]
            flat_v[at] = st["value"].double().view(-1, KV, D)[rows]
        return turned(st["query"], H, st["q_norm"]).view(-1, H * D), kc, vc
    lo, hi = _ranges(case, s)
    out = torch.zeros(st["tokens"], H, D, dtype=torch.float64, device=DEVICE)
    q = st["query"].double().view(-1, H, D)
    for b, (new, past) in enumerate(zip(s["new"], s["past"])):
        at = slots(b, 0, past + new)
        j = torch.arange(past + new, device=DEVICE)
        for t0 in range(starts_at[b], starts_at[b + 1], 1024):
            t1 = min(t0 + 1024, starts_at[b + 1])
            first = torch.tensor(lo[t0:t1], device=DEVICE)[:, None]
            end = torch.tensor(hi[t0:t1], device=DEVICE)[:, None]
            hidden = ~((j >= first) & (j < end))
            pos = past + torch.arange(t0 - starts_at[b], t1 - starts_at[b], device=DEVICE)
            for h in range(H):
                kh = h // (H // KV)
                x = q[t0:t1, h] @ flat_k[at, kh].T * D ** -0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if case["op"] == "masked" and case["slopes"]:
                    x = x - 2.0 ** (-8.0 * (h + 1) / H) * (pos[:, None] - j).abs()
                x = x.masked_fill(hidden, -math.inf)
                if st["sink"] is not None:
                    x = torch.cat([x, st["sink"][h].double().expand(t1 - t0, 1)], 1)
                p = torch.softmax(x, 1)[:, :past + new].nan_to_num(0.0)
                out[t0:t1, h] = p @ flat_v[at, kh]
    return out.view(-1, H * D)
