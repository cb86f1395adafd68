"""Pages whose offsets pass 32 bits: the bits of the same pages at the start of a pool; and rows of odd sizes moved in
place over several rounds."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
import test_gpu_accumulating_attention as weigh
from masked_cases import make_batch
from test_gpu_accept_drafts import drafts, i64
from test_gpu_evict_keys import setup, verify
from upkeep_cases import packed, trees

pytestmark = pytest.mark.gpu

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def room():
    yield torch.empty((9 << 30) + 64, dtype=torch.uint8, device="cuda")
    torch.cuda.empty_cache()


def far(st, room):
    """The batch with its pages behind 4 GiB of each cache; only they and their scales are written."""
    nb = st["kc"].shape[0]
    page = st["kc"][0].numel() * st["kc"].element_size()
    first = (1 << 32) // page + 3
    out = dict(st, first=first)
    half = room.numel() // 2 // 16 * 16
    for i, s in enumerate(("kc", "vc")):
        pool = room[i * half:i * half + (first + nb) * page].view(st[s].dtype).view(first + nb, *st[s].shape[1:])
        pool[first:].view(torch.uint8).copy_(st[s].view(torch.uint8))
        out[s] = pool
        if st[s[0] + "_scale"] is not None:
            out[s[0] + "_scale"] = torch.cat([torch.ones(first, st["KV"], device="cuda"), st[s[0] + "_scale"]])
    out["bt"] = torch.where(st["bt"] >= 0, st["bt"] + first, st["bt"])
    return out


def at_far(x, first):
    return torch.cat([torch.zeros(first, *x.shape[1:], device="cuda"), x])


@pytest.mark.parametrize("new,past", [([1, 2], [300, 1000]), ([40, 3], [70, 600]), ([90, 1], [70, 600])],
                         ids=["step", "rows", "nodes"])
@pytest.mark.parametrize("dt,D,kind", [(BF16, 128, None), (F32, 64, None), (BF16, 128, FP8), (BF16, 320, None)])
def test_pages_beyond_32_bits(room, dt, D, kind, new, past):
    st = make_batch(new, past, H=8, KV=4, D=D, block=16, dtype=dt, seed=1, cache_dtype=kind)
    f = far(st, room)
    assert f["kc"].numel() * f["kc"].element_size() > 1 << 32
    w, got = weigh.account(st), []
    par = packed(trees(st))
    nodes, tokens, targets = drafts(new, words=1)
    for x in (st, f):
        at = (x["q"], x["kc"], x["vc"], x["cum"], x["past_t"], x["bt"])
        sc = dict(k_scale=x["k_scale"], v_scale=x["v_scale"])
        kw = dict(num_heads=8, max_query_len=max(new), max_context_len=max(st["total"]), **sc)
        acc = w.clone() if x is st else at_far(w, f["first"])
        outs = [ep.tree_attention(*at, par, **kw), ep.accumulating_attention(*at, acc, **kw)]
        outs += ep.accept_drafts(x["kc"], x["vc"], x["cum"], x["past_t"], x["bt"], packed(nodes), i64(tokens), i64(targets),
                                 key_weights=acc, **sc)
        outs += ep.evict_keys(x["kc"], x["vc"], acc, x["past_t"], x["bt"], budget=50, sinks=2, recent=5, **sc)
        lo = 0 if x is st else f["first"]
        got.append([y.contiguous().view(torch.uint8) for y in (*outs, x["kc"][lo:], x["vc"][lo:], acc[lo:])])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind,D", [("f16", 3), ("int4", 65), ("fp8", 30), ("fp8", 20), ("f32", 5), ("fp8", 64)])
def test_odd_rows_in_place_over_several_rounds(kind, D):
    verify(setup([3000, 700], D=D, kind=kind, KV=2, seed=7), 2500, 3, 90)
    verify(setup([3000, 700], D=D, kind=kind, KV=2, seed=8), 600, 0, 0)
