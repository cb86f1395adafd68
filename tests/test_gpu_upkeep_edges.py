"""Drafted trees, accounts, accepted rows and eviction where they can go wrong: heads beyond 256, coded pages under odd
heads, tensors at odd addresses, tables that name no page, pages that sequences share."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
import test_gpu_accumulating_attention as weigh
import test_gpu_tree_attention as tree
from masked_cases import check, make_batch
from test_gpu_accept_drafts import cum_of, drafts, i64
from test_gpu_evict_keys import places, raw, setup
from upkeep_cases import attention64, causal_seen, packed, trees

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEPS = [([1, 1, 2], [0, 70, 601]), ([9, 0, 40, 3], [33, 5, 0, 130])]


@pytest.mark.parametrize("new,past", STEPS, ids=["step", "rows"])
@pytest.mark.parametrize("dt,H,KV,D,block", [(BF16, 4, 2, 264, 16), (F32, 3, 1, 320, 7), (F16, 2, 2, 512, 32),
                                             (BF16, 6, 2, 640, 16), (F32, 4, 2, 257, 16)])
def test_heads_beyond_256(dt, H, KV, D, block, new, past):
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, seed=1)
    tree.compare(st, trees(st))
    tree.compare(st, trees(st, seed=1), window=4, softcap=8.0)
    weigh.compare(st)
    weigh.compare(st, observed=2, window=20, sink=torch.linspace(-1, 1, H).to(dt).cuda())


@pytest.mark.parametrize("new,past", STEPS, ids=["step", "rows"])
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 33), (F32, 200), (BF16, 320), (F32, 64)])
@pytest.mark.parametrize("kind,scales", [(torch.float8_e4m3fn, "NONE"), (torch.int8, "PER_TENSOR"), (torch.int8, "PER_CHANNEL"),
                                         (torch.uint8, "PER_TENSOR"), (torch.uint8, "PER_CHANNEL")],
                         ids=["fp8", "int8", "int8_channels", "int4", "int4_channels"])
def test_coded_pages(kind, scales, dt, D, new, past):
    st = make_batch(new, past, H=4, KV=2, D=D, block=16, dtype=dt, seed=2, cache_dtype=kind, scales=scales)
    tree.compare(st, trees(st))
    weigh.compare(st)


@pytest.mark.parametrize("dt,D,kind", [(F32, 64, None), (BF16, 80, None), (BF16, 128, torch.float8_e4m3fn), (F16, 256, torch.int8),
                                       (F32, 300, None)])
def test_prompts_of_other_types(dt, D, kind):
    """Rows that fill several chunks of sums, under a window, without causality, few of them observed."""
    st = make_batch([700, 1, 260], [30, 500, 0], H=4, KV=2, D=D, block=16, dtype=dt, seed=9, cache_dtype=kind)
    weigh.compare(st)
    weigh.compare(st, window=90, softcap=20.0)
    weigh.compare(st, causal=0, observed=600)
    tree.compare(st, trees(st), window=200)


def shifted(x, by=1):
    """The same values `by` elements behind an aligned address."""
    y = torch.empty(x.numel() + by, dtype=x.dtype, device=x.device)[by:].view(x.shape)
    return y.copy_(x)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 80)])
def test_odd_addresses(dt, D):
    for new, past in STEPS:
        st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=3)
        st["kc"], st["vc"] = shifted(st["kc"]), shifted(st["vc"], 3)
        tree.compare(st, trees(st))
        weigh.compare(st)


def test_accounts_at_odd_addresses():
    st = make_batch([1, 2, 30], [300, 5, 40], H=8, KV=2, D=128, block=16, dtype=BF16, seed=4)
    w = weigh.account(st)
    a, b = w.clone(), shifted(w)
    one, two = weigh.run(st, a), weigh.run(st, b)
    assert torch.equal(one, two) and torch.equal(a.view(torch.int32), b.view(torch.int32))
    e = setup([500, 90], seed=5)
    other = {x: e[x].clone() for x in ("kc", "vc", "w")}
    kept, _ = ep.evict_keys(e["kc"], e["vc"], e["w"], e["lens_t"], e["table"], budget=64, sinks=3, recent=5)
    moved = shifted(other["kc"], 1), shifted(other["vc"], 2), shifted(other["w"], 1)
    again, _ = ep.evict_keys(*moved, e["lens_t"], e["table"], budget=64, sinks=3, recent=5)
    assert torch.equal(kept, again) and all(torch.equal(e[x], y) for x, y in zip(("kc", "vc", "w"), moved))


def test_pages_that_sequences_share():
    """Outputs over a shared prefix are those of pages of one's own; its account is anybody's, the others' are not."""
    for new in ([1, 2, 1], [40, 3, 20]):
        st = make_batch(new, [96, 64, 70], H=8, KV=2, D=128, block=16, dtype=BF16, seed=6, shared=[64], group_cum=[0, 3])
        w = weigh.account(st)
        old = w.clone()
        got = weigh.run(st, w)
        want, tol, weights = attention64(st, [causal_seen(n, p) for n, p in zip(st["new"], st["past"])])
        check(got, want, tol)
        for b, (added, bound) in enumerate(weights):
            p = torch.arange(64, st["total"][b], device="cuda")
            at = st["bt"][b].long()[p // 16], slice(None), p % 16
            exact = torch.where((p < st["past"][b])[:, None], old[at].double(), 0.0) + added.T[64:]
            check(w[at], exact, bound.T[64:] + 2.0 ** -23 * exact + 1e-30)


@pytest.mark.parametrize("bad", [-1, 1 << 20, -(1 << 31)])
def test_tables_that_name_no_page(bad):
    """Entries within the lengths that are no page: nothing is written through them."""
    nodes, past = [40, 20], [90, 30]
    st = setup([p + n for p, n in zip(past, nodes)], seed=7)
    start = {x: st[x].clone() for x in ("kc", "vc", "w")}
    past_t = torch.tensor(past, dtype=torch.int32, device="cuda")
    parents, tokens, targets = drafts(nodes, words=1)
    alone = st["table"].clone()
    st["table"][0] = bad
    path, lens, _ = ep.accept_drafts(st["kc"], st["vc"], cum_of(nodes), past_t, st["table"], packed(parents), i64(tokens),
                                     i64(targets), key_weights=st["w"])
    assert int(lens[0]) > 1
    rows = torch.zeros(st["kc"].shape[:2], dtype=torch.bool, device="cuda")
    rows[places(st, 1, range(past[1], past[1] + nodes[1]))] = True
    for x in ("kc", "vc"):
        assert torch.equal(raw(st[x])[~rows], raw(start[x])[~rows])
    assert torch.equal(st["w"].transpose(1, 2)[~rows], start["w"].transpose(1, 2)[~rows])

    for out in (False, True):
        for x in start:
            st[x].copy_(start[x])
        st["table"].copy_(alone)
        (st["other"] if out else st["table"])[0] = bad
        ep.evict_keys(st["kc"], st["vc"], st["w"], st["lens_t"], st["table"], budget=24, sinks=1, recent=2,
                      block_table_out=st["other"] if out else None)
        rows[:] = False
        rows[places(st, 1, range(24 if out else sum(x[1] for x in (nodes, past))), "other" if out else "table")] = True
        for x in ("kc", "vc"):
            assert torch.equal(raw(st[x])[~rows], raw(start[x])[~rows])
        assert torch.equal(st["w"].transpose(1, 2)[~rows], start["w"].transpose(1, 2)[~rows])

    for new in ([1, 1], [40, 20]):
        b = make_batch(new, past, H=4, KV=2, D=64, block=16, dtype=BF16, seed=8)
        w = torch.rand(b["kc"].shape[0], 2, 16, device="cuda")
        old = w.clone()
        b["bt"][0] = bad
        weigh.run(b, w)
        p = torch.arange(b["total"][1], device="cuda")
        mine = torch.zeros(w.shape[0], 16, dtype=torch.bool, device="cuda")
        mine[b["bt"][1].long()[p // 16], p % 16] = True
        assert torch.equal(w.transpose(1, 2)[~mine], old.transpose(1, 2)[~mine])
        assert bool((w.transpose(1, 2)[mine] != old.transpose(1, 2)[mine]).any())
