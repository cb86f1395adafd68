"""pa_accept_drafts against its rule, to the bit: accepted paths and the rows that they move."""
from __future__ import annotations

import random

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from test_gpu_evict_keys import places, raw, recoded, setup
from upkeep_cases import accepted, packed, tree

pytestmark = pytest.mark.gpu


def drafts(nodes, seed=0, words=3, chain=0.4):
    """Trees whose few different tokens make siblings alike and paths long."""
    rng = random.Random(seed)
    parents = [tree(rng, n, chain) if n else [] for n in nodes]
    return parents, [[rng.randrange(words) for _ in p] for p in parents], [[rng.randrange(words) for _ in p] for p in parents]


def cum_of(nodes):
    return torch.tensor([0] + torch.tensor(nodes).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def i64(x):
    return torch.tensor(sum(x, []), dtype=torch.int64, device="cuda")


def moved(st, past, path, before):
    """Rows of the accepted paths where they should be, the rest of the pages as it was."""
    want = {s: before[s].clone() for s in ("kc", "vc")}
    spent = torch.zeros(st["kc"].shape[:2], dtype=torch.bool, device="cuda")
    for b, rows in enumerate(path):
        if not rows:
            continue
        src, dst = places(st, b, [past[b] + r for r in rows]), places(st, b, range(past[b], past[b] + len(rows)))
        for s in ("kc", "vc"):
            x = before[s][src]
            if st["kw"]:
                sc = st["kw"][s[0] + "_scale"]
                for h in range(st["KV"]):
                    want[s].view(torch.uint8)[dst[0], dst[1], h] = recoded(x[:, h], sc[src[0], h], sc[dst[0], h])
            else:
                want[s][dst] = x
        spent[dst] = True
    for s in ("kc", "vc"):
        assert torch.equal(raw(st[s]), raw(want[s]))


def verify(st, past, nodes, d, max_path=0, **kw):
    parents, tokens, targets = d
    before = {s: st[s].clone() for s in ("kc", "vc")}
    past_t = torch.tensor(past, dtype=torch.int32, device="cuda")
    path, lens, after = ep.accept_drafts(st["kc"], st["vc"], cum_of(nodes), past_t, st["table"], packed(parents),
                                         i64(tokens), i64(targets), max_path=max_path, **st["kw"], **kw)
    want = [accepted(*x)[:max_path or None] for x in zip(parents, tokens, targets)]
    for b, rows in enumerate(want):
        assert path[b].tolist() == rows + [-1] * (path.shape[1] - len(rows))
        assert int(lens[b]) == len(rows)
        assert int(after[b]) == (targets[b][rows[-1]] if rows else -1)
    moved(st, past, want, before)
    return want


@pytest.mark.parametrize("kind,D,block", [("bf16", 64, 16), ("f16", 128, 32), ("f32", 40, 7), ("bf16", 256, 256),
                                          ("f16", 3, 16), ("int8", 96, 16), ("int4", 65, 16), ("fp8", 64, 16),
                                          ("fp8", 30, 8)])
def test_rows(kind, D, block):
    nodes, past = [26, 0, 1, 64, 65, 200], [100, 9, 0, 16, 33, 5]
    st = setup([p + n for p, n in zip(past, nodes)], D=D, block=block, kind=kind, KV=3)
    verify(st, past, nodes, drafts(nodes))


def test_paths():
    """Chains agreed with to their ends, paths of one node, equal siblings, trees of several words of 64 rows."""
    nodes, past = [300, 40, 500, 129], [10, 0, 40, 1]
    chain = lambda n: list(range(-1, n - 1))  # noqa: E731
    for words, seed in ((1, 0), (2, 1), (50, 2)):
        st = setup([p + n for p, n in zip(past, nodes)], seed=seed)
        d = drafts(nodes, seed, words, chain=0.8)
        want = verify(st, past, nodes, d)
        if words == 1:  # every token is agreed with: first children all the way down
            assert max(map(len, want)) > 3
        st = setup([p + n for p, n in zip(past, nodes)], seed=seed)
        verify(st, past, nodes, ([chain(n) for n in nodes], d[1], d[2]))


def test_paths_end_at_their_bound():
    nodes, past = [100, 30], [10, 3]
    st = setup([110, 33])
    d = ([list(range(-1, n - 1)) for n in nodes], [[1] * n for n in nodes], [[1] * n for n in nodes])
    for most in (1, 7, 30, 31, 200):
        verify(setup([110, 33]), past, nodes, d, max_path=most)
    verify(st, past, nodes, d, max_query_len=100)


def test_odd_parents_are_never_taken():
    nodes = [6]
    parents = [[-1, 0, 7, 3, -9, 1]]
    verify(setup([20]), [10], nodes, (parents, [[5] * 6], [[5] * 6]))


def test_given_paths():
    nodes, past = [40, 20, 0, 9], [30, 0, 4, 700]
    st = setup([p + n for p, n in zip(past, nodes)], D=128, KV=8)
    paths = [[0, 3, 4, 5, 9, 22, 39], [], [], [4, 8]]
    path = torch.tensor([p + [-1] * (7 - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    lens = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
    before = {s: st[s].clone() for s in ("kc", "vc")}
    got = ep.accept_drafts(st["kc"], st["vc"], cum_of(nodes), torch.tensor(past, dtype=torch.int32, device="cuda"),
                           st["table"], path=path, path_lens=lens)
    assert got[0] is path and got[1] is lens and got[2] is None
    moved(st, past, paths, before)


def test_captured_and_replayed():
    nodes, past = [64, 30], [100, 7]
    st = setup([164, 37], D=128, KV=4)
    start = {s: st[s].clone() for s in ("kc", "vc")}
    d = drafts(nodes, 5, 2)
    held = packed(d[0]), i64(d[1]), i64(d[2])
    cum, past_t = cum_of(nodes), torch.tensor(past, dtype=torch.int32, device="cuda")

    def call():
        return ep.accept_drafts(st["kc"], st["vc"], cum, past_t, st["table"], *held, max_path=40)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fixed = call()
    for seed in range(3):
        d = drafts(nodes, seed, 2)
        for x, y in zip(held, (packed(d[0]), i64(d[1]), i64(d[2]))):
            x.copy_(y)
        seen = []
        for how in (call, None, None):
            for x in start:
                st[x].copy_(start[x])
            got = how() if how else (graph.replay(), fixed)[1]
            torch.cuda.synchronize()
            seen.append([x.clone() for x in (*got, st["kc"], st["vc"])])
        for other in seen[1:]:
            assert all(torch.equal(a, b) for a, b in zip(seen[0], other))
