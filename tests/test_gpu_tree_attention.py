"""pa_tree_attention against its definition in 64 bits: types, heads, pages, trees of every shape, windows by depth,
softcaps, sinks; siblings that hold NaN; captured, on two streams, in a workspace of the caller's."""
from __future__ import annotations

import random

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import check, make_batch
from upkeep_cases import attention64, lines, packed, tree, tree_seen, trees

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(st, parents, *, scale=0.0, softcap=0.0, window=-1, sink=None, **kw):
    kw = {"max_query_len": max(st["new"]), "max_context_len": max(st["total"]), **kw}
    pad = st["q"].shape[0] - sum(st["new"])
    return ep.tree_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"],
                             packed(parents, pad=pad), num_heads=st["H"], scale=scale, softcap=softcap,
                             local_window_size=window, head_sink=sink, k_scale=st["k_scale"],
                             v_scale=st["v_scale"], k_quant_type=st["quant"], v_quant_type=st["quant"], **kw)


def compare(st, parents, *, window=-1, call=None, **forms):
    got = run(st, parents, window=window, **forms, **(call or {}))
    seen = [tree_seen(p, past, window) for p, past in zip(parents, st["past"])]
    want, tol, _ = attention64(st, seen, **forms)
    check(got[:want.shape[0]], want, tol)
    return got


LAYOUTS = [(BF16, 8, 2, 128, 16), (F16, 8, 2, 128, 32), (F16, 8, 1, 64, 16), (BF16, 6, 3, 96, 16),
           (BF16, 4, 1, 256, 16), (F16, 4, 2, 256, 256), (BF16, 16, 2, 64, 64), (F16, 7, 1, 128, 8),
           (BF16, 4, 4, 128, 24), (F32, 4, 2, 64, 16), (BF16, 4, 2, 80, 16), (F16, 3, 1, 40, 7),
           (F32, 2, 1, 256, 16)]
BATCHES = {"single": ([1, 1, 1, 1], [0, 63, 64, 700]),
           "small": ([7, 0, 1, 9, 4], [9, 100, 31, 511, 1200]),
           "trees": ([33, 1, 64, 65, 0, 129], [0, 1, 17, 40, 9, 333]),
           "sixty_four": ([64, 33, 1, 63, 0], [70, 5, 0, 600, 8]),
           "wide": ([31, 32, 257], [65, 1000, 90])}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace("torch.", "") for y in x))
def test_layouts(layout, batch):
    dt, H, KV, D, block = layout
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, seed=1)
    compare(st, trees(st))
    compare(st, trees(st, chain=0.9, seed=1), window=5)


FORMS = {"window_one": dict(window=1), "window": dict(window=17), "window_past": dict(window=70),
         "softcap": dict(softcap=5.0), "softcap_large": dict(softcap=100.0), "softcap_window": dict(softcap=50.0, window=9),
         "sink": dict(sink=True), "scale": dict(scale=0.3), "negative_scale": dict(scale=-0.1)}


@pytest.mark.parametrize("batch", ["small", "sixty_four", "trees"])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_forms(dt, D, form, batch):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=2)
    f = dict(FORMS[form])
    if "sink" in f:
        f["sink"] = torch.linspace(-1, 2, 8).to(dt).cuda()
    compare(st, trees(st, chain=0.7, seed=3), **f)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 256), (F32, 64)])
def test_shapes_of_trees(dt, D):
    """Chains, stars, roots without a parent, parents that name no earlier row."""
    n = 100
    st = make_batch([n] * 4, [50, 0, 7, 130], H=4, KV=2, D=D, block=16, dtype=dt, seed=4)
    chain, star = list(range(-1, n - 1)), [-1] + [0] * (n - 1)
    odd = [(-5, r, r + 1, 1 << 30, -(1 << 31), 2)[r % 6] for r in range(n)]
    compare(st, [chain, star, [-1] * n, odd])
    compare(st, [chain, star, [-1] * n, odd], window=3)


def test_a_chain_is_causal_attention():
    st = make_batch([40, 3], [100, 600], H=8, KV=2, D=128, block=16, dtype=BF16, seed=5)
    for window in (-1, 25):
        got = run(st, [list(range(-1, n - 1)) for n in st["new"]], window=window)
        assert torch.equal(got, ep.masked_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"],
                                                    num_heads=8, local_window_size=window, max_query_len=40,
                                                    max_context_len=603))


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 64)])
def test_other_branches_may_hold_anything(dt, D):
    """NaN and infinities in keys and values change the rows that descend from them alone."""
    st = make_batch([70, 5], [30, 300], H=4, KV=1, D=D, block=16, dtype=dt, seed=6)
    parents = trees(st, chain=0.5, seed=2)
    above, _ = lines(parents[0])
    leaf = next(r for r in range(69, 0, -1) if above[:, r].sum() == 1)
    inner = next(r for r in range(5, 70) if above[:, r].sum() in (2, 3, 4))
    for b, j, side, x in ((0, 30 + leaf, "v", float("inf")), (0, 30 + inner, "v", float("nan")),
                          (0, 30 + leaf, "k", float("nan")), (1, 302, "v", -float("inf"))):
        at = st["bt"][b, j // 16].long(), j % 16
        st[side + "c"][at[0], at[1], 0, 3] = x
        st[side + "d"][at[0], at[1], 0, 3] = x
    got = run(st, parents)
    seen = [tree_seen(p, past) for p, past in zip(parents, st["past"])]
    want, tol, _ = attention64(st, seen)
    check(got, want, torch.where(torch.isfinite(want), tol, 1.0))


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8, torch.uint8])
def test_byte_coded_pages(kind):
    for dt in (BF16, F16):
        st = make_batch([20, 1, 35], [100, 0, 61], H=4, KV=2, D=64, block=16, dtype=dt, seed=8, cache_dtype=kind,
                        scales="NONE" if kind == torch.float8_e4m3fn else "PER_CHANNEL")
        if kind == torch.float8_e4m3fn:
            st["quant"] = "NONE"
        compare(st, trees(st), window=40)


def test_bounds_unknown_and_rows_behind_the_last_sequence():
    for dt, D in ((BF16, 128), (F32, 64)):
        st = make_batch([3, 40], [600, 3], H=8, KV=2, D=D, block=16, dtype=dt, seed=7, pad_tokens=5)
        parents = trees(st)
        out = torch.full_like(st["q"], 7.0)
        got = compare(st, parents, call=dict(max_query_len=0, max_context_len=0, out=out))
        assert got is out and bool((out[43:] == 7.0).all())


def test_large_trees_and_long_contexts():
    st = make_batch([1000], [20], H=4, KV=1, D=64, block=16, dtype=F16, seed=9)
    compare(st, trees(st, chain=0.95))
    compare(st, [list(range(-1, 999))], window=600)
    st = make_batch([70, 1], [20001, 9000], H=8, KV=2, D=128, block=16, dtype=BF16, seed=10)
    compare(st, trees(st))


def test_the_most_nodes():
    st = make_batch([4096], [3], H=2, KV=1, D=64, block=16, dtype=F16, seed=11)
    compare(st, [tree(random.Random(1), 4096, 0.3)])


def test_no_tokens():
    st = make_batch([0, 0], [4, 0], H=4, KV=2, D=64, block=16, dtype=F16, seed=6)
    assert run(st, [[], []], max_query_len=0).shape == (0, 256)


def test_captured_and_replayed():
    """Replays over other trees and contexts, eager calls between them, give the eager bits."""
    st = make_batch([26, 9, 40], [300, 2000, 100], H=8, KV=2, D=128, block=16, dtype=BF16, seed=14)
    held = packed(trees(st))
    out = torch.empty_like(st["q"])

    def call(out):
        return ep.tree_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], held, num_heads=8,
                                 local_window_size=500, max_query_len=40, max_context_len=2009, out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i, past in enumerate(([300, 2000, 100], [299, 1000, 20], [0, 1, 0])):
        st["past_t"].copy_(torch.tensor(past, dtype=torch.int32))
        held.copy_(packed(trees(st, seed=i)))
        for _ in range(2):
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call(torch.empty_like(out)))


def test_two_streams_at_once_and_own_workspaces():
    sts = [make_batch([20] * 4, [400 * (i + 1)] * 4, H=8, KV=2, D=128, block=16, dtype=BF16, seed=20 + i)
           for i in range(2)]
    want = [run(st, trees(st)) for st in sts]
    own = [torch.empty(64 << 20, dtype=torch.uint8, device="cuda") for _ in sts]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sts], [[], []]
    for k in range(12):
        for i, (st, s) in enumerate(zip(sts, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(st, trees(st), workspace=own[i] if k % 2 else None))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
