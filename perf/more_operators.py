"""Operators that keep a paged cache at work: drafted trees and what is accepted of them, attention that
keeps account of what its keys weigh, and the eviction that goes by that account.

  tree     attention of the nodes of drafted trees, each over the cached keys and its own ancestors
  accept   the path of a drafted tree that the model agrees with, and its rows moved to where the
           cached sequence goes on
  weigh    attention over the pages that adds what every key weighed to an account beside the pages
  evict    the keys of every head that stay by that account, written to pages of their own

Where `own` is false, run() computes them from elementary torch operations in 32 bits on padded
batches; where it is true it makes the library's calls.  A case holds sizes and options only.
`layout` seeds the ragged lengths and the trees (so work() can count them); the seed of prepare()
makes the tensors and the order of the pages.
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
DEEPEST = 40  # nodes of a drafted path, at most
VOCABULARY = 32000


# ---------------------------------------------------------------------------------------- cases

_BASE = dict(dtype="bf16", heads=32, kv=8, head=128, block=16, seqs=1, past_min=0, past_max=0, layout=1)


def _case(name, **kw):
    return kw if name is None else dict(name=name, **kw)


def _tree(name=None, **kw):
    # seqs sequences with trees of nodes_min..nodes_max drafted tokens after past_min..past_max keys;
    # chain: share of the nodes that follow the node before them, the others hang on any earlier one.
    return _case(name, **{**dict(op="tree", **_BASE, nodes_min=1, nodes_max=1, chain=0.4, window=-1,
                                 softcap=0.0, sink=False), **kw})


def _accept(name=None, **kw):
    # the same trees; about `agree` of the steps down a path are the model's own choice, too.
    return _case(name, **{**dict(op="accept", **_BASE, nodes_min=1, nodes_max=1, chain=0.4, agree=0.8), **kw})


def _weigh(name=None, **kw):
    # new_min..new_max new tokens, the last `observed` of which count (0: all of them).
    return _case(name, **{**dict(op="weigh", **_BASE, new_min=1, new_max=1, observed=0, window=-1,
                                 softcap=0.0, sink=False), **kw})


def _evict(name=None, **kw):
    # past_min..past_max keys of which `budget` stay: the first `sinks`, the last `recent` and the
    # heaviest of the others.
    return _case(name, **{**dict(op="evict", **_BASE, budget=1, sinks=0, recent=0), **kw})


def listed():
    return [
        # One user's chat, a small tree of drafts: launch latency is most of it.
        _tree("tree_one_user", nodes_min=26, nodes_max=26, past_min=700, past_max=700),
        # A server's step that checks everybody's drafts.
        _tree("tree_step_16", heads=28, kv=4, seqs=16, nodes_min=40, nodes_max=64, past_min=500,
              past_max=6000, layout=3),
        # Smaller trees of a model with sliding windows and sinks at head 64.
        _tree("tree_window", dtype="f16", heads=64, kv=8, head=64, block=32, seqs=24, nodes_min=9,
              nodes_max=33, past_min=200, past_max=4000, window=1000, sink=True, layout=5),
        # A wide tree over one long document.
        _tree("tree_long_document", nodes_min=257, nodes_max=257, past_min=60001, past_max=60001,
              chain=0.2, layout=7),
        # What one user's tree leaves: latency alone.
        _accept("accept_one_user", nodes_min=26, nodes_max=26, past_min=700, past_max=700),
        # What a server's step leaves: many trees at odd lengths.
        _accept("accept_step_64", heads=24, kv=4, head=256, block=64, seqs=64, nodes_min=30,
                nodes_max=64, past_min=100, past_max=6000, chain=0.7, agree=0.9, layout=3),
        # One token of a small model whose cache is kept to a budget.
        _weigh("weigh_one_token", dtype="f16", heads=8, kv=2, head=64, past_min=300, past_max=300),
        # A loaded server's step, every key's weight kept.
        _weigh("weigh_step_48", seqs=48, past_min=511, past_max=8190, layout=3),
        # Prompts of which the last rows say what stays.
        _weigh("weigh_prompt_last_32", heads=28, kv=4, seqs=2, new_min=3001, new_max=5001, observed=32,
               layout=2),
        # A prompt all of whose rows count; softcap.
        _weigh("weigh_prompt_all", dtype="f16", heads=24, kv=4, head=256, block=32, new_min=4095,
               new_max=4095, past_min=600, past_max=600, softcap=50.0),
        # A small model's cache cut once.
        _evict("evict_one", dtype="f16", heads=8, kv=2, head=64, past_min=1201, past_max=1201, budget=500,
               sinks=4, recent=64),
        # Long prompts cut to a fraction before they are decoded.
        _evict("evict_prompts_16", seqs=16, past_min=4001, past_max=9000, budget=2048, sinks=4,
               recent=255, layout=3),
    ]


HEADS = ((32, 8, 128), (28, 4, 128), (8, 2, 64), (64, 8, 64), (24, 8, 96), (8, 1, 256), (24, 4, 256))


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST_BYTES, MOST_FLOPS, MOST_SCORES = 8.0e8, 2.4e11, 1.4e9


def _scores(case):
    """Scores of the padded plain form."""
    if case["op"] not in ("tree", "weigh"):
        return 0
    s = _lengths(case)
    return (len(s["new"]) * max(s["new"]) * case["heads"] *
            max(p + n for p, n in zip(s["past"], s["new"])))


def _draw_once(rng):
    op = rng.choices(("tree", "accept", "weigh", "evict"), (0.35, 0.15, 0.3, 0.2))[0]
    heads, kv, head = rng.choice(HEADS)
    longest = _logint(rng, 20, 16000)
    base = dict(dtype=rng.choice(("bf16", "f16")), heads=heads, kv=kv, head=head,
                block=rng.choice((16, 16, 32, 64, 256)), seqs=_logint(rng, 1, 64),
                past_min=longest // 4, past_max=longest, layout=rng.randrange(1 << 20))
    if op in ("tree", "accept"):
        most = _logint(rng, 1, 200)
        base.update(nodes_min=max(1, most // 2), nodes_max=most, chain=rng.uniform(0.0, 0.9))
        if op == "accept":
            return _accept(**base, agree=rng.uniform(0.3, 1.0))
    if op == "evict":
        budget = _logint(rng, 8, longest)
        sinks = rng.choice((0, min(4, budget // 4)))
        return _evict(**base, budget=budget, sinks=sinks, recent=rng.choice((0, budget // 8, budget // 2)))
    forms = dict(window=rng.choice((-1, -1, -1, _logint(rng, 16, 2000))),
                 softcap=rng.choice((0.0, 0.0, 0.0, 50.0)), sink=rng.random() < 0.2)
    if op == "tree":
        return _tree(**base, **forms)
    if rng.random() < 0.5:  # a step of a token or a few
        return _weigh(**base, **forms, new_max=rng.choice((1, 1, 1, 3)))
    most = _logint(rng, 17, 5000)
    base.update(seqs=_logint(rng, 1, 8), past_min=0, past_max=rng.choice((0, _logint(rng, 1, 2000))))
    return _weigh(**base, **forms, new_min=max(1, most // 3), new_max=most,
                  observed=rng.choice((0, 1, 32, 64)))


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and _scores(case) <= MOST_SCORES:
            return case


# -------------------------------------------------------------------------------------- lengths

def _drafted(rng, nodes, chain):
    """Parents of a tree of drafted tokens, row 0 its root, and every node's depth."""
    parents, depth = [-1], [0]
    for r in range(1, nodes):
        p = r - 1 if rng.random() < chain else rng.randrange(r)
        while depth[p] >= DEEPEST - 1:
            p = parents[p]
        parents.append(p)
        depth.append(depth[p] + 1)
    return parents, depth


def _lengths(case):
    """New tokens and cached keys, the trees, and how far down each tree the model agrees."""
    rng = random.Random(case["layout"])
    out = dict(new=[], past=[], parents=[], depth=[], agreed=[])
    for _ in range(case["seqs"]):
        out["past"].append(rng.randint(case["past_min"], case["past_max"]))
        if case["op"] in ("tree", "accept"):
            parents, depth = _drafted(rng, rng.randint(case["nodes_min"], case["nodes_max"]), case["chain"])
            out["new"].append(len(parents))
            out["parents"].append(parents)
            out["depth"].append(depth)
            if case["op"] == "accept":
                node, path = max(range(len(depth)), key=lambda r: (depth[r], rng.random())), []
                while node >= 0:
                    path.append(node)
                    node = parents[node]
                path, n = path[::-1], 1
                while n < len(path) and rng.random() < case["agree"]:
                    n += 1
                out["agreed"].append(path[:n])
        else:
            out["new"].append(rng.randint(case["new_min"], case["new_max"]) if case["op"] == "weigh" else 0)
    return out


def work(case):
    s = _lengths(case)
    H, KV, D, window = case["heads"], case["kv"], case["head"], case.get("window", -1)
    row = KV * D * 2 * 2  # a token's keys and values
    if case["op"] == "accept":
        # the trees with their tokens, and every accepted row that moves: read and written
        moved = sum(r != i for path in s["agreed"] for i, r in enumerate(path))
        return {"bytes": float(2 * moved * row + sum(s["new"]) * (4 + 8 + 8)), "flops": float(sum(s["new"]))}
    if case["op"] == "evict":
        kept = sum(min(case["budget"], n) for n in s["past"])
        return {"bytes": float(2 * kept * row + KV * 4 * (sum(s["past"]) + 3 * kept)),
                "flops": float(sum(s["past"]) * KV)}
    pairs = keys = 0
    for b, (new, past) in enumerate(zip(s["new"], s["past"])):
        near = window if window > 0 else past + new
        if case["op"] == "tree":
            depth = s["depth"][b]
            pairs += sum(min(past + d + 1, near) for d in depth)
        else:
            pairs += sum(min(past + i + 1, near) for i in range(new))
        keys += min(past + new, near + new - 1)
    tokens = sum(s["new"])
    flops, moved = 4 * pairs * H * D, keys * row + 2 * tokens * H * D * 2
    if case["op"] == "weigh":
        moved += 2 * sum(p + n for p, n in zip(s["past"], s["new"])) * KV * 4
        flops += 2 * pairs * H
    return {"bytes": float(moved), "flops": float(flops)}


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
    # eviction writes what stays to pages of its own
    kept = [-(-min(t, case["budget"]) // bs) if case["op"] == "evict" else 0 for t in total]

    def normal(*shape, std=1.0):
        x = torch.empty(shape, dtype=dt, device=DEVICE)
        return x.normal_(0.0, std, generator=g)

    need, table = 0, []
    for t in total + [k * bs for k in kept]:
        table.append(list(range(need, need - (-t // bs))))
        need += len(table[-1])
    num_blocks = need + 3
    order = torch.randperm(num_blocks, device=DEVICE, generator=g).to(torch.int32)
    index = torch.tensor([row + [0] * (max_blocks - len(row)) for row in table], device=DEVICE)
    pages = order[index].contiguous()
    st = dict(case=case, tokens=T, key_cache=normal(num_blocks, bs, KV, D),
              value_cache=normal(num_blocks, bs, KV, D), past=_i32(s["past"]), block_table=pages[:B],
              cum=_i32([0] + torch.tensor(s["new"]).cumsum(0).tolist()), max_query_len=max(s["new"]),
              max_context_len=max(total))
    # where the plain form finds the packed tokens in a padded batch
    inside = torch.arange(max(s["new"]), device=DEVICE)[None, :] < _i32(s["new"])[:, None]
    st["rows"] = inside.flatten().nonzero().flatten()
    if case["op"] in ("weigh", "evict"):
        # what the keys weighed so far: a few much, most little
        w = torch.empty(num_blocks, KV, bs, device=DEVICE).normal_(0.0, 1.0, generator=g)
        st["key_weights"] = torch.exp(2.0 * w - 3.0)
    if case["op"] == "evict":
        st["block_table_out"] = pages[B:, :max(1, max(kept))].contiguous()
        return st
    if case["op"] in ("tree", "accept"):
        st["parents"] = _i32(sum(s["parents"], []))
    if case["op"] == "accept":
        # the model's choice at every node: the drafted token along the agreed path, else another one
        tokens = torch.randint(VOCABULARY, (T,), device=DEVICE, generator=g)
        targets = torch.randint(VOCABULARY, (T,), device=DEVICE, generator=g)
        at = [s0 + r for s0, path in zip(st["cum"].tolist(), s["agreed"]) for r in path[:-1]]
        to = [s0 + r for s0, path in zip(st["cum"].tolist(), s["agreed"]) for r in path[1:]]
        if at:
            targets[at] = tokens[to]
        st["draft_tokens"], st["target_tokens"] = tokens, targets
        return st
    # scores of a trained model spread wider than one
    st["query"] = normal(T, H * D) * 1.5
    st["output"] = torch.empty_like(st["query"])
    st["sink"] = normal(H) if case["sink"] else None
    return st


# ------------------------------------------------------------------------------------ plain form

def _pages(st, keys):
    """Places in the pages of the positions 0 .. keys - 1 of every sequence."""
    bs, table = st["case"]["block"], st["block_table"].long()
    pos = torch.arange(keys, device=DEVICE).clamp(max=table.shape[1] * bs - 1).expand(table.shape[0], -1)
    return table.gather(1, pos // bs), pos % bs


def _ancestors(st):
    """[B, per, per]: whether a node is another one or an ancestor of it; powers of (1 + parent) reach DEEPEST up."""
    per = st["max_query_len"]
    r = torch.arange(per, device=DEVICE)
    parent = torch.full((len(st["past"]) * per,), -1, device=DEVICE).index_put((st["rows"],), st["parents"].long())
    up = (parent.view(-1, per)[..., None] == r).float() + torch.eye(per, device=DEVICE)
    return torch.linalg.matrix_power(up, DEEPEST) > 0, parent.view(-1, per)


def _attend(st, seen):
    """Outputs and probabilities [B, KV, per, g, keys] of the rows under seen [B, per, keys]."""
    case = st["case"]
    H, KV, D, g = case["heads"], case["kv"], case["head"], case["heads"] // case["kv"]
    B, per, keys = seen.shape
    block, off = _pages(st, keys)
    k = st["key_cache"][block, off].float().permute(0, 2, 3, 1)
    v = st["value_cache"][block, off].float().transpose(1, 2)
    q = torch.zeros(B * per, H * D, device=DEVICE)
    q[st["rows"]] = st["query"].float()
    q = q.view(B, per, KV, g, D).transpose(1, 2).reshape(B, KV, per * g, D)
    x = q @ k / math.sqrt(D)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = torch.where(seen[:, None, :, None], x.view(B, KV, per, g, keys), -math.inf)
    m = x.amax(-1, keepdim=True)
    sink = None if st["sink"] is None else st["sink"].float().view(1, KV, 1, g, 1)
    m = m if sink is None else torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    den = p.sum(-1, keepdim=True)
    den = den if sink is None else den + torch.exp(sink - m)
    p = torch.where(den > 0, p / den, 0.0)
    used = seen.any(1)[:, None, :, None]  # (what no row sees may be anything)
    out = p.view(B, KV, per * g, keys) @ torch.where(used, v, 0.0)
    out = out.view(B, KV, per, g, D).transpose(1, 2).reshape(B * per, H * D)[st["rows"]]
    st["output"].copy_(out)
    return st["output"], p


def _plain_tree(st):
    per, keys, window = st["max_query_len"], st["max_context_len"], st["case"]["window"]
    past = st["past"].long()[:, None, None]
    above, _ = _ancestors(st)
    depth = above.sum(-1) - 1  # [B, per]
    j = torch.arange(keys, device=DEVICE)
    node = (j - past).clamp(0, per - 1).expand(-1, per, -1)
    seen = (j < past) | ((j < past + per) & above.gather(2, node))
    if window > 0:
        at = torch.where(j < past, j, past + depth[:, None].expand(-1, per, -1).gather(2, node))
        seen = seen & (at > past + depth[..., None] - window)
    return _attend(st, seen)[0]


def _plain_weigh(st):
    case = st["case"]
    per, keys, bs = st["max_query_len"], st["max_context_len"], case["block"]
    past, new = st["past"].long(), st["cum"].long().diff()
    j, r = torch.arange(keys, device=DEVICE), torch.arange(per, device=DEVICE)
    pos = past[:, None] + r
    seen = (j <= pos[..., None]) & (r < new[:, None])[..., None]
    if case["window"] > 0:
        seen = seen & (j > pos[..., None] - case["window"])
    out, p = _attend(st, seen)
    counts = r < new[:, None]
    if case["observed"]:
        counts = counts & (r >= (new - case["observed"])[:, None])
    p = torch.where(counts[:, None, :, None, None], p, 0.0).sum((2, 3))  # [B, KV, keys]
    block, off = _pages(st, keys)
    b, j = (j < (past + new)[:, None]).nonzero(as_tuple=True)
    block, off, w = block[b, j], off[b, j], p[b, :, j]
    old = torch.where((j < past[b])[:, None], st["key_weights"][block, :, off], 0.0)
    st["key_weights"][block, :, off] = old + w
    return out, st["key_weights"]


def _plain_accept(st):
    per, bs = st["max_query_len"], st["case"]["block"]
    past, new = st["past"].long(), st["cum"].long().diff()
    B, r = len(past), torch.arange(per, device=DEVICE)

    def padded(x):
        return torch.full((B * per,), -1, device=DEVICE).index_put((st["rows"],), x.long()).view(B, per)

    above, parent = _ancestors(st)
    tokens, targets = padded(st["draft_tokens"]), padded(st["target_tokens"])
    agree = (tokens == targets.gather(1, parent.clamp(min=0))) & (parent >= 0)
    # of several children with the model's token the first one
    earlier = (parent[:, :, None] == parent[:, None]) & agree[:, None] & (r < r[:, None])
    agree = (agree & ~earlier.any(-1)) | (r == 0)
    taken = (above.float() @ (~agree).float()[..., None])[..., 0] == 0
    taken = taken & (r < new[:, None])
    depth = above.sum(-1) - 1
    count = taken.sum(-1)
    path = torch.full((B, DEEPEST), -1, dtype=torch.int32, device=DEVICE)
    b, row = taken.nonzero(as_tuple=True)
    path[b, depth[b, row]] = row.to(torch.int32)
    last = path.gather(1, (count - 1).clamp(min=0)[:, None]).long()
    after = targets.gather(1, last)[:, 0]
    src, dst = past[b] + row, past[b] + depth[b, row]
    table = st["block_table"].long()
    for cache in (st["key_cache"], st["value_cache"]):
        cache[table[b, dst // bs], dst % bs] = cache[table[b, src // bs], src % bs]
    return path, count.to(torch.int32), after, st["key_cache"], st["value_cache"]


def _plain_evict(st):
    case = st["case"]
    budget, bs, keys = case["budget"], case["block"], st["max_context_len"]
    n = st["past"].long()[:, None]
    block, off = _pages(st, keys)
    j = torch.arange(keys, device=DEVICE)
    w = st["key_weights"][block, :, off].transpose(1, 2)  # [B, KV, keys]
    always = (j < case["sinks"]) | (j >= n - case["recent"])
    w = torch.where(always[:, None], math.inf, w)
    w = torch.where((j < n)[:, None], w, -math.inf)
    best = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :budget]
    best = torch.where(best < n[..., None], best, keys)
    kept = torch.sort(best, dim=-1)[0]
    kept = torch.where(kept < keys, kept, -1)
    if keys < budget:
        kept = torch.cat([kept, torch.full((*kept.shape[:2], budget - keys), -1, device=DEVICE)], -1)
    b, h, i = (kept >= 0).nonzero(as_tuple=True)
    at = kept[b, h, i]
    table, out = st["block_table"].long(), st["block_table_out"].long()
    sp, so, dp, do = table[b, at // bs], at % bs, out[b, i // bs], i % bs
    for cache in (st["key_cache"], st["value_cache"]):
        cache[dp, do, h] = cache[sp, so, h]
    st["key_weights"][dp, h, do] = st["key_weights"][sp, h, so]
    return (kept.to(torch.int32), n[:, 0].clamp(max=budget).to(torch.int32), st["key_cache"],
            st["value_cache"], st["key_weights"])


# ------------------------------------------------------------------------------------------ runs

def _library():
    place = str(Path(__file__).resolve().parent.parent / "onnxruntime-ep-mlx_amd")
    if place not in sys.path:
        sys.path.insert(0, place)
    import onnxruntime_ep_mlx_amd as ep
    return ep


def _own(st):
    ep, case = _library(), st["case"]
    caches = (st["key_cache"], st["value_cache"])
    if case["op"] == "evict":
        kept, lens = ep.evict_keys(*caches, st["key_weights"], st["past"], st["block_table"],
                                   budget=case["budget"], sinks=case["sinks"], recent=case["recent"],
                                   block_table_out=st["block_table_out"],
                                   max_context_len=st["max_context_len"])
        return kept, lens, *caches, st["key_weights"]
    if case["op"] == "accept":
        path, lens, after = ep.accept_drafts(*caches, st["cum"], st["past"], st["block_table"],
                                             st["parents"], st["draft_tokens"], st["target_tokens"],
                                             max_path=DEEPEST, max_query_len=st["max_query_len"])
        return path, lens, after, *caches
    args = (st["query"], *caches, st["cum"], st["past"], st["block_table"])
    kw = dict(num_heads=case["heads"], softcap=case["softcap"], local_window_size=case["window"],
              head_sink=st["sink"], max_query_len=st["max_query_len"],
              max_context_len=st["max_context_len"], out=st["output"])
    if case["op"] == "tree":
        return ep.tree_attention(*args, st["parents"], **kw)
    out = ep.accumulating_attention(*args, st["key_weights"], observed_rows=case["observed"], **kw)
    return out, st["key_weights"]


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "accept": _plain_accept, "weigh": _plain_weigh,
            "evict": _plain_evict}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """From the definitions, in 64 bits, one sequence at a time."""
    st = prepare(case, seed)
    s = _lengths(case)
    H, KV, D, bs = case["heads"], case["kv"], case["head"], case["block"]
    kc, vc = st["key_cache"].double(), st["value_cache"].double()
    flat_k, flat_v = kc.view(-1, KV, D), vc.view(-1, KV, D)

    def slots(b, positions, table="block_table"):
        p = torch.as_tensor(positions, device=DEVICE)
        return st[table][b].long()[p // bs] * bs + p % bs

    starts = [0]
    for n in s["new"]:
        starts.append(starts[-1] + n)
    if case["op"] == "accept":
        B = len(s["new"])
        path = torch.full((B, DEEPEST), -1, dtype=torch.int32)
        count, after = torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.int64)
        tokens, targets = st["draft_tokens"].tolist(), st["target_tokens"].tolist()
        for b, (new, past) in enumerate(zip(s["new"], s["past"])):
            node, rows = 0, [0]
            while True:
                want = targets[starts[b] + node]
                child = next((r for r in range(node + 1, new)
                              if s["parents"][b][r] == node and tokens[starts[b] + r] == want), None)
                if child is None:
                    break
                node = child
                rows.append(node)
            path[b, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
            count[b], after[b] = len(rows), targets[starts[b] + node]
            src = slots(b, [past + r for r in rows])
            dst = slots(b, list(range(past, past + len(rows))))
            for flat in (flat_k, flat_v):
                flat[dst] = flat[src].clone()
        return path.to(DEVICE), count.to(DEVICE), after.to(DEVICE), kc, vc
    if case["op"] == "evict":
        weights = st["key_weights"].double()
        flat_w = weights.transpose(1, 2).reshape(-1, KV)
        B, budget = len(s["past"]), case["budget"]
        kept = torch.full((B, KV, budget), -1, dtype=torch.int32)
        w_all = flat_w.cpu()
        for b, n in enumerate(s["past"]):
            at = slots(b, list(range(n)))
            lead, tail = min(case["sinks"], n), max(n - case["recent"], 0)
            for h in range(KV):
                w = w_all[at.cpu(), h].tolist()
                middle = sorted(range(lead, tail), key=lambda j: (-w[j], j)) if n > budget else []
                mine = sorted([*range(lead), *middle[:budget - case["sinks"] - case["recent"]],
                               *range(max(tail, lead), n)]) if n > budget else list(range(n))
                kept[b, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
                src, dst = slots(b, mine), slots(b, list(range(len(mine))), "block_table_out")
                for flat in (flat_k, flat_v, flat_w):
                    flat[dst, h] = flat[src, h]
        lens = torch.tensor([min(n, budget) for n in s["past"]], dtype=torch.int32)
        weights = flat_w.view(-1, bs, KV).transpose(1, 2).contiguous()
        return kept.to(DEVICE), lens.to(DEVICE), kc, vc, weights
    out = torch.zeros(st["tokens"], H, D, dtype=torch.float64, device=DEVICE)
    q = st["query"].double().view(-1, H, D)
    weights = st["key_weights"].double() if case["op"] == "weigh" else None
    for b, (new, past) in enumerate(zip(s["new"], s["past"])):
        at = slots(b, list(range(past + new)))
        j = torch.arange(past + new, device=DEVICE)
        place = j.clone()  # where the keys stand in their text
        above = None
        if case["op"] == "tree":
            place[past:] = past + torch.tensor(s["depth"][b], device=DEVICE)
            rows = []
            for r in range(new):
                line, node = [False] * new, r
                while node >= 0:
                    line[node], node = True, s["parents"][b][node]
                rows.append(line)
            above = torch.tensor(rows, device=DEVICE)
        added = torch.zeros(KV, past + new, dtype=torch.float64, device=DEVICE)
        for r0 in range(0, new, 1024):
            r1 = min(r0 + 1024, new)
            pos = place[past + r0:past + r1, None]
            hidden = place > pos
            if above is not None:
                hidden = torch.cat([hidden[:, :past], ~above[r0:r1]], 1)
            if case["window"] > 0:
                hidden = hidden | (place <= pos - case["window"])
            counted = torch.arange(r0, r1, device=DEVICE) >= (new - case.get("observed", 0) or 0)
            if not case.get("observed", 0):
                counted = torch.ones_like(counted)
            for h in range(H):
                kh = h // (H // KV)
                x = q[starts[b] + r0:starts[b] + r1, h] @ flat_k[at, kh].T * D ** -0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                x = x.masked_fill(hidden, -math.inf)
                if st["sink"] is not None:
                    x = torch.cat([x, st["sink"][h].double().expand(r1 - r0, 1)], 1)
                p = torch.softmax(x, 1)[:, :past + new].nan_to_num(0.0)
                out[starts[b] + r0:starts[b] + r1, h] = p @ flat_v[at, kh]
                added[kh] += p[counted].sum(0)
        if weights is not None:
            page, off = at // bs, at % bs
            old = torch.where((j < past)[:, None], weights[page, :, off], 0.0)
            weights[page, :, off] = old + added.T
    out = out.view(-1, H * D)
    return out if weights is None else (out, weights)
